// Global memory at a base that the wavefront shares and an offset of 32 bits of each lane's own: one instruction, with the base in
// scalar registers.  Left to itself the compiler adds the two before, with an addition of 64 bits and two vector registers to each
// access in flight.  For runs of costs with the labels last, 500 x 1000 pixels, that was: the gradient of distillation over 256
// labels 372 us, now 318; of layer norm over 32 labels 46, now 34; best of 96 labels 49, now 38; verification over 256 labels
// 478, now 252.  With the labels first the bases differ from row to row, and holding each in scalar registers is no gain (gradient
// over 192 labels 138 us as it was, 152 so).
#ifndef MPLAYERS_AMD_MP_OFFSETS_H_
#define MPLAYERS_AMD_MP_OFFSETS_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mpl {

template <typename T>
using GlobalMemory = __attribute__((address_space(1))) T;

// index * sizeof(T) below 2^32, base the same in all lanes
template <typename T>
__device__ __forceinline__ GlobalMemory<T>* at_offset(T* base, unsigned index) {
  uint64_t shared = reinterpret_cast<uint64_t>(base);
  asm("" : "+s"(shared));  // (as it is: nothing is added to it that could be added to the offset)
  return reinterpret_cast<GlobalMemory<T>*>(shared + (uint32_t)(index * (unsigned)sizeof(T)));
}
template <typename T>
__device__ __forceinline__ T load_at(const T* base, unsigned index) {
  return *at_offset(base, index);
}
template <typename T>
__device__ __forceinline__ void store_at(T* base, unsigned index, T value) {
  *at_offset(base, index) = value;
}

// Four side by side, aligned to all of them; index: of the four.
template <typename T>
using QuadWords = uint32_t __attribute__((ext_vector_type(sizeof(T))));
template <typename T>
__device__ __forceinline__ void load_quad(const T* base, unsigned index, T (&x)[4]) {
  const QuadWords<T> words = *at_offset(reinterpret_cast<const QuadWords<T>*>(base), index);
  __builtin_memcpy(x, &words, sizeof(words));
}
template <typename T>
__device__ __forceinline__ void store_quad(T* base, unsigned index, T a, T b, T c, T d) {
  const T x[4] = {a, b, c, d};
  QuadWords<T> words;
  __builtin_memcpy(&words, x, sizeof(words));
  *at_offset(reinterpret_cast<QuadWords<T>*>(base), index) = words;
}

// How a run of costs with the labels last is moved: one by one, four side by side, or so in quads that are of one pixel.  Fours may be
// of two pixels or more.  us one by one -> four side by side, 40 M costs: best of 2 labels 134 -> 130, 3 106 -> 104, divergence and
// gradient 2 368 -> 365, 3 296 -> 292, verified 2 232 -> 209, 3 158 -> 141 (layer norm has a rule of its own for these); best of 21 52 ->
// 44, verified 5 136 -> 118.
enum { kEach, kFours, kQuads };
inline int run_mode(int n_disp, bool aligned) { return !aligned ? kEach : n_disp % 4 == 0 ? kQuads : kFours; }
// first: of the run, counted from what is aligned; a tile's pixels are whole fours, and its last one's costs need not be.
__device__ __forceinline__ int run_mode_of(int mode, int64_t first, unsigned total) {
  return mode == kFours && (((unsigned)first | total) & 3) != 0 ? (int)kEach : mode;
}

}  // namespace mpl

#endif  // MPLAYERS_AMD_MP_OFFSETS_H_
