// Dropout of the unary costs within the change to the layers' layout, for gfx950.
//
// x (items, labels, pixels), the network's layout, in fp32, fp16 or bf16  ->  y (items, pixels, labels) in fp32:
//   y[i, p, l] = keep(i, l, p) ? x[i, l, p] * scale : 0,   scale = 1 / (1 - rate)
// and its gradient, the same product back to x's layout and type.  keep is never stored: it is formed in either
// direction from a counter-based generator, the 4x32 multiply-and-xor rounds (ten of them) of Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (SC 2011).  The key is the seed, the counter is the number of
// a group of labels and the offset, both 64 bits; a label stays where its 32-bit word is at least rate * 2^32.
//
// Four labels of a pixel share a counter (its four words): a thread owns a quad of labels of one pixel, so the words
// it forms are all used (but for the last quad of a label count that is no multiple of four) wherever the pixel
// lies, and the number of pixels may be odd.

#include "mp_common.h"

using namespace mpl;

namespace {

constexpr int kPixels = 64;  // pixels of a tile: one wavefront along a label's row

enum Share { kElement = MPL_DROPOUT_ELEMENT, kPixel = MPL_DROPOUT_PIXEL, kLabel = MPL_DROPOUT_LABEL };

struct Dropout {
  const int64_t* state;  // seed, offset
  int64_t pixels, tiles;
  int labels;
  uint32_t bound;  // words from this on stay
  int nothing;     // rate 1
  float scale;
};

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words random_words(uint64_t group, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// which labels of quad q of a pixel stay, as factors
template <int SHARE>
__device__ __forceinline__ void factors(const Dropout& d, int64_t item, int64_t pixel, int q, int quads, uint64_t seed,
                                        uint64_t offset, bool keep[4]) {
  const uint64_t group = SHARE == kElement ? (uint64_t)(item * d.pixels + pixel) * (uint64_t)quads + (uint64_t)q
                         : SHARE == kPixel ? (uint64_t)(item * d.pixels + pixel)
                                           : (uint64_t)item * (uint64_t)quads + (uint64_t)q;
  const Words r = random_words(group, offset, seed);
#pragma unroll
  for (int j = 0; j < 4; ++j) keep[j] = r.w[SHARE == kPixel ? 0 : j] >= d.bound && !d.nothing;
}

// An fp32 product, rounded as such before a narrower type rounds it again: the compiler would make one instruction
// of both for fp16 (not for bf16), and the types would differ in how they round.
__device__ __forceinline__ float scaled(float x, float scale) {
  float y = x * scale;
  asm("" : "+v"(y));
  return y;
}

// One tile of kPixels pixels and all labels per workgroup of 64 x 4 threads.  LAST: into the label-innermost layout.
template <typename T, int SHARE, bool LAST>
__global__ void __launch_bounds__(256) dropout_kernel(Dropout d, const void* __restrict__ src, void* __restrict__ dst) {
  extern __shared__ float tile[];  // [pixel][labels | 1]
  const int64_t block = (int64_t)blockIdx.x;
  const int64_t item = block / d.tiles, p0 = (block - item * d.tiles) * kPixels;
  const int px = (int)threadIdx.x, ty = (int)threadIdx.y, tid = ty * kPixels + px;
  const int n = d.labels, stride = n | 1, quads = (n + 3) >> 2;
  const int count = (int)min((int64_t)kPixels, d.pixels - p0);
  const uint64_t seed = (uint64_t)d.state[0], offset = (uint64_t)d.state[1];
  const int64_t first = item * n * d.pixels;
  const float* last_in = (const float*)src + first + p0 * n;
  float* last_out = (float*)dst + first + p0 * n;
  const T* rows_in = (const T*)src + first + p0;
  T* rows_out = (T*)dst + first + p0;
  if (!LAST) {
    for (int i = tid; i < count * n; i += 256) tile[i / n * stride + i % n] = last_in[i];
    __syncthreads();
  }
  if (px < count) {
    for (int q = ty; q < quads; q += 4) {
      bool keep[4];
      factors<SHARE>(d, item, p0 + px, q, quads, seed, offset, keep);
      for (int j = 0; j < 4 && 4 * q + j < n; ++j) {
        const int l = 4 * q + j;
        if (LAST)
          tile[px * stride + l] = keep[j] ? (float)rows_in[l * d.pixels + px] * d.scale : 0.f;
        else
          rows_out[l * d.pixels + px] = (T)(keep[j] ? scaled(tile[px * stride + l], d.scale) : 0.f);
      }
    }
  }
  if (LAST) {
    __syncthreads();
    for (int i = tid; i < count * n; i += 256) last_out[i] = tile[i / n * stride + i % n];
  }
}

template <typename T, bool LAST>
void launch(int share, const Dropout& d, const void* src, void* dst, unsigned blocks, hipStream_t st) {
  const dim3 block(kPixels, 4);
  const size_t lds = (size_t)kPixels * (size_t)(d.labels | 1) * sizeof(float);
  if (share == kElement)
    dropout_kernel<T, kElement, LAST><<<blocks, block, lds, st>>>(d, src, dst);
  else if (share == kPixel)
    dropout_kernel<T, kPixel, LAST><<<blocks, block, lds, st>>>(d, src, dst);
  else
    dropout_kernel<T, kLabel, LAST><<<blocks, block, lds, st>>>(d, src, dst);
}

template <bool LAST>
int run(const char* what, int dtype, int share, double rate, const int64_t* state, const void* src, void* dst, int batch,
        int n_disp, int64_t pixels, void* stream) {
  if (state == nullptr || src == nullptr || dst == nullptr) return fail(MPL_EINVAL, "%s: null pointer", what);
  if (dtype < 0 || dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d", what, dtype);
  if (share < 0 || share > kLabel) return fail(MPL_EINVAL, "%s: unknown share %d", what, share);
  if (!(rate >= 0 && rate <= 1)) return fail(MPL_EINVAL, "%s: the rate must be in [0, 1]", what);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "%s: n_disp must be in [1, %d], got %d", what, kMaxL, n_disp);
  if (batch < 0 || pixels < 0) return fail(MPL_EINVAL, "%s: negative size", what);
  if (batch == 0 || pixels == 0) return MPL_OK;
  Dropout d;
  d.state = state;
  d.pixels = pixels;
  d.tiles = (pixels + kPixels - 1) / kPixels;
  d.labels = n_disp;
  if (pixels > ((int64_t)1 << 40) || d.tiles * batch > 0x7fffffff) return fail(MPL_EINVAL, "%s: too many pixels", what);
  d.nothing = rate >= 1;
  d.bound = d.nothing ? 0u : (uint32_t)(rate * 4294967296.0);
  d.scale = d.nothing ? 0.f : (float)(1.0 / (1.0 - rate));
  const unsigned blocks = (unsigned)(d.tiles * batch);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == MPL_F32)
    launch<float, LAST>(share, d, src, dst, blocks, st);
  else if (dtype == MPL_F16)
    launch<_Float16, LAST>(share, d, src, dst, blocks, st);
  else
    launch<__bf16, LAST>(share, d, src, dst, blocks, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int mpl_dropout_labels_last(int dtype, int share, double rate, const int64_t* state, const void* src, float* dst,
                            int batch, int n_disp, int64_t pixels, void* stream) {
  return run<true>("dropout_labels_last", dtype, share, rate, state, src, dst, batch, n_disp, pixels, stream);
}

int mpl_dropout_labels_first(int dtype, int share, double rate, const int64_t* state, const float* src, void* dst,
                             int batch, int n_disp, int64_t pixels, void* stream) {
  return run<false>("dropout_labels_first", dtype, share, rate, state, src, dst, batch, n_disp, pixels, stream);
}

}  // extern "C"
