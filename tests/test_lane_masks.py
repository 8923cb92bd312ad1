"""Lane masks in inline assembly: on gfx950 a select may read a mask only two issue slots after a comparison wrote it.  The
compiler pads its own pairs with idle slots, and nothing that stands within one asm statement."""
import glob
import os
import re

import pytest

from mplayers_amd import _build

# (the probes' patterns are timed, and what they leave in the registers is not read)
SOURCES = sorted(path for path in glob.glob(os.path.join(_build.CSRC, "*.hip")) + glob.glob(os.path.join(_build.CSRC, "*.h"))
                 if os.path.splitext(os.path.basename(path))[0] not in _build.PROBE_UNITS)


def _instructions(text):
  """Of each statement of string literals in a source, its instructions (macros between them stay out)."""
  text = re.sub(r"//[^\n]*", "", text).replace("\\\n", "\n")
  for run in re.findall(r'(?:"(?:[^"\\]|\\.)*"\s*)+', text):
    lines = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', run)).replace("\\t", " ").split("\\n")
    yield [line.strip() for line in lines if line.strip()]


def _too_near(instructions):
  """Pairs of a comparison and a select of its mask with fewer than two issue slots between them."""
  for i, line in enumerate(instructions):
    wrote = re.match(r"v_cmp\w*\s+(vcc|%\d+|s\[[^\]]*\])", line)
    slots = 0
    for other in instructions[i + 1:] if wrote else ():
      if slots >= 2 or re.match(r"v_cmp\w*\s+" + re.escape(wrote.group(1)) + r"\b", other):
        break
      if other.startswith("v_cndmask") and other.replace(" ", "").endswith("," + wrote.group(1)):
        yield line, other
      idle = re.match(r"s_nop (\d+)", other)
      slots += int(idle.group(1)) + 1 if idle else 1


def test_the_search_itself():
  near, far = 'asm("v_cmp_u_f32 vcc, %1, %1\\n\\tv_cndmask_b32 %0, %1, %2, vcc");', \
      'asm("v_cmp_u_f32 vcc, %1, %1\\n\\t" "s_nop 1\\n\\tv_cndmask_b32 %0, %1, %2, vcc");'
  assert [len(list(_too_near(x))) for text in (near, far) for x in _instructions(text)] == [1, 0]
  between = 'asm("v_cmp_eq_f32 %3, %1, %1\\n\\tv_mov_b32 %4, 0\\n\\tv_cndmask_b32 %0, %1, %2, %3");'
  assert [len(list(_too_near(x))) for x in _instructions(between)] == [1]


@pytest.mark.parametrize("path", SOURCES, ids=[os.path.basename(p) for p in SOURCES])
def test_masks_are_not_read_before_they_are_there(path):
  with open(path) as f:
    pairs = [pair for instructions in _instructions(f.read()) for pair in _too_near(instructions)]
  assert not pairs, pairs
