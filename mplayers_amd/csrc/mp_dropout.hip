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
//
// Bound by HBM: the mask costs no traffic and the change of layout is one the layer makes anyway.  us, forward /
// backward: fp32, 192 labels 1500x2000 883 / 885 (5.2 TB/s; the change of layout alone, mpl_transpose, 1019); fp16, 128
// labels 375x1242, whole pixels 74 / 80 (4.8 and 4.5 TB/s; in turn, one in the cache that the other filled, 62 / 95);
// bf16, 21 labels 12x129x129 9.7 / 8.7 (2.5 and 2.8 TB/s; what bounds it is not shown: vector issue is 0.3 of it, so not
// the generator; its accesses are 2 bytes to a lane, 4 on the operators' side, as its labels are no multiple of four).
// The generator takes 20 wide products and 20 exclusive ors for four labels, 420 vector instructions to a wavefront of
// the first case in all.

#include "mp_common.h"

using namespace mpl;

namespace {


constexpr int64_t kFewTiles = 4096;  // of 64 pixels, see launch_share

enum Share { kElement = MPL_DROPOUT_ELEMENT, kPixel = MPL_DROPOUT_PIXEL, kLabel = MPL_DROPOUT_LABEL };

struct Dropout {
  const int64_t* state;  // seed, offset
  int64_t pixels;
  int tiles, labels;
  uint32_t bound;  // words from this on stay
  int nothing;     // rate 1
  float scale;
  uint32_t reciprocal;  // 2^32 / labels, rounded up
  int whole_quads;      // the label-innermost side: labels in fours, all aligned
  int xcd_group;        // tiles beside each other that go to one die (xcd_block)
};

struct Words {
  uint32_t w[4];
};

// one instruction (0x96: the truth table of a ^ b ^ c)
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return (uint32_t)__builtin_amdgcn_bitop3_b32((int)a, (int)b, (int)c, 0x96);
}

__device__ __forceinline__ Words random_words(uint64_t group, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// Bits 0 to 3: which labels of quad q of a pixel stay.
template <int SHARE>
__device__ __forceinline__ int stays(const Dropout& d, int64_t item, int64_t pixel, int q, int quads, uint64_t seed,
                                     uint64_t offset) {
  const uint64_t group = SHARE == kElement ? (uint64_t)(item * d.pixels + pixel) * (uint64_t)quads + (uint64_t)q
                         : SHARE == kPixel ? (uint64_t)(item * d.pixels + pixel)
                                           : (uint64_t)item * (uint64_t)quads + (uint64_t)q;
  const Words r = random_words(group, offset, seed);
  if (SHARE == kPixel) return r.w[0] >= d.bound && !d.nothing ? 15 : 0;
  int bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) bits |= r.w[j] >= d.bound && !d.nothing ? 1 << j : 0;
  return bits;
}

// An fp32 product, rounded as such before a narrower type rounds it again: the compiler would make one instruction
// of both for fp16 (not for bf16), and the types would differ in how they round.
__device__ __forceinline__ float scaled(float x, float scale) {
  float y = x * scale;
  asm("" : "+v"(y));
  return y;
}

// One tile of P pixels (P / 64 wavefronts beside each other) and all labels per workgroup of W times as many, so that the
// label-innermost side is one run of memory whatever the number of labels.  Those of wavefront w of W take the quads
// w + i * W, i < J, with a lane per pixel: 256 contiguous bytes of a label's row (fp32) to an instruction.  The tile lies in LDS with the labels of a pixel side by
// side, an odd number of quads apart, which keeps the 16-byte accesses of either side off each other's banks.
//
// The random words are formed between the loads and their first use.  What lies behind the last label or pixel is
// loaded from the last's place, so that there is no branch between the loads.
//
// LAST: into the label-innermost layout, else its gradient back.
template <typename T, int SHARE, bool LAST, int W, int J, int P>
__global__ void __launch_bounds__(P* W) dropout_kernel(Dropout d, const void* __restrict__ src,
                                                             void* __restrict__ dst) {
  constexpr int kStride = 4 * (W * J | 1);
  __shared__ __align__(16) float tile[P * kStride];
  const unsigned block = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, d.xcd_group);
  const unsigned of_item = block / (unsigned)d.tiles;
  const int64_t item = of_item, p0 = (int64_t)(block - of_item * (unsigned)d.tiles) * P;
  const int tid = (int)threadIdx.x, px = tid % P, wave = uniform_i(tid / P);
  const int n = d.labels, quads = (n + 3) >> 2;
  const int count = (int)min((int64_t)P, d.pixels - p0);
  const unsigned total = (unsigned)(count * n);
  const int64_t first = item * n * d.pixels;
  const uint64_t seed = (uint64_t)d.state[0], offset = (uint64_t)d.state[1];
  const int of = min(px, count - 1);
  const auto place = [&](unsigned i) {  // of entry i of the label-innermost run
    const unsigned p = n == 1 ? i : __umulhi(i, d.reciprocal);
    return p * kStride + (i - p * (unsigned)n);
  };
  int keep[J];
  const auto form_masks = [&]() {
    const int all = SHARE == kPixel ? stays<SHARE>(d, item, p0 + of, 0, quads, seed, offset) : 0;
#pragma unroll
    for (int i = 0; i < J; ++i)
      keep[i] = SHARE == kPixel ? all : stays<SHARE>(d, item, p0 + of, wave + i * W, quads, seed, offset);
  };
  if (LAST) {
    const T* from = (const T*)src + first + p0;
    T x[J][4];
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] = from[(int64_t)min(4 * (wave + i * W) + j, n - 1) * d.pixels + of];
    form_masks();
#pragma unroll
    for (int i = 0; i < J; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = keep[i] >> j & 1 ? (float)x[i][j] * d.scale : 0.f;
      *reinterpret_cast<float4*>(&tile[px * kStride + 4 * (wave + i * W)]) = float4{y[0], y[1], y[2], y[3]};
    }
    __syncthreads();
    float* to = (float*)dst + first + p0 * n;
    if (d.whole_quads) {
      for (unsigned i = (unsigned)tid * 4; i < total; i += P * W * 4)
        *reinterpret_cast<float4*>(to + i) = *reinterpret_cast<const float4*>(&tile[place(i)]);
    } else {
      for (unsigned i = (unsigned)tid; i < total; i += P * W) to[i] = tile[place(i)];
    }
  } else {
    const float* from = (const float*)src + first + p0 * n;
    if (d.whole_quads) {
      float4 x[J];
#pragma unroll
      for (int k = 0; k < J; ++k)
        x[k] = *reinterpret_cast<const float4*>(from + min((unsigned)(tid + k * P * W) * 4, total - 4));
      form_masks();
#pragma unroll
      for (int k = 0; k < J; ++k)
        *reinterpret_cast<float4*>(&tile[place(min((unsigned)(tid + k * P * W) * 4, total - 4))]) = x[k];
    } else {
      float x[4 * J];
#pragma unroll
      for (int k = 0; k < 4 * J; ++k) x[k] = from[min((unsigned)(tid + k * P * W), total - 1)];
      form_masks();
#pragma unroll
      for (int k = 0; k < 4 * J; ++k) tile[place(min((unsigned)(tid + k * P * W), total - 1))] = x[k];
    }
    __syncthreads();
    if (px >= count) return;
    T* to = (T*)dst + first + p0 + px;
#pragma unroll
    for (int i = 0; i < J; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(&tile[px * kStride + 4 * (wave + i * W)]);
      const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int l = 4 * (wave + i * W) + j;
        if (l < n) to[(int64_t)l * d.pixels] = (T)(keep[i] >> j & 1 ? scaled(y[j], d.scale) : 0.f);
      }
    }
  }
}

// Wavefronts W and quads J to a wavefront, pixels P of a tile.  Small launches do not fill the chip: up to eight wavefronts
// share a tile before one takes a third quad.  us forward / backward with one to four wavefronts of six quads -> this: 16
// labels 64x96 3.2 / 3.6 -> 2.4 / 2.5, 21 labels 129x129 4.7 / 4.6 -> 3.5 / 3.4, 64 labels 375x450 16.7 / 20.8 -> 15.4 / 15.9,
// 96 labels 384x1248 70.1 / 72.5 -> 70.2 / 70.9; a wavefront to every quad: 64 labels 15.6 / 16.9, 21 labels 600x800 17.8 /
// 16.4 (14.9 / 14.7 this).  Large launches of few labels are bound by the workgroups that start: wider tiles, from kFewTiles
// on, with 64 pixels -> this: bf16 2 labels 7x1217x1930 158 / 140 -> 89 / 81, 5 labels 182 / 153 -> 128 / 115, 13 labels
// 4x387x672 25.5 / 22.6 -> 20.0 / 18.1, fp32 4 labels 173 / 151 -> 99 / 93, 8 labels 191 / 186 -> 188 / 186.
template <typename T, int SHARE, bool LAST>
int launch_share(const char* what, Dropout& d, int batch, const void* src, void* dst, hipStream_t st) {
  const auto run = [&](auto kernel, int waves, int pixels) {
    const int64_t tiles = (d.pixels + pixels - 1) / pixels;
    // (a launch has less than 2^32 threads)
    if (tiles > (int64_t)0xffffffff / (pixels * waves) / batch) return fail(MPL_EINVAL, "%s: too many pixels", what);
    d.tiles = (int)tiles;
    kernel<<<(unsigned)(tiles * batch), pixels * waves, 0, st>>>(d, src, dst);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
  };
  const int n = d.labels;
  const bool few = d.pixels / 64 * batch <= kFewTiles;
  if (n <= 4)
    return few ? run(dropout_kernel<T, SHARE, LAST, 1, 1, 64>, 1, 64) : run(dropout_kernel<T, SHARE, LAST, 1, 1, 512>, 1, 512);
  if (n <= 8)
    return few ? run(dropout_kernel<T, SHARE, LAST, 2, 1, 64>, 2, 64) : run(dropout_kernel<T, SHARE, LAST, 1, 2, 256>, 1, 256);
  if (n <= 16)
    return few ? run(dropout_kernel<T, SHARE, LAST, 4, 1, 64>, 4, 64) : run(dropout_kernel<T, SHARE, LAST, 2, 2, 128>, 2, 128);
  if (n <= 24) return run(dropout_kernel<T, SHARE, LAST, 3, 2, 64>, 3, 64);
  if (n <= 32) return run(dropout_kernel<T, SHARE, LAST, 4, 2, 64>, 4, 64);
  if (n <= 48) return run(dropout_kernel<T, SHARE, LAST, 6, 2, 64>, 6, 64);
  if (n <= 64) return run(dropout_kernel<T, SHARE, LAST, 8, 2, 64>, 8, 64);
  if (n <= 96) return run(dropout_kernel<T, SHARE, LAST, 8, 3, 64>, 8, 64);
  if (n <= 128) return run(dropout_kernel<T, SHARE, LAST, 8, 4, 64>, 8, 64);
  if (n <= 192) return run(dropout_kernel<T, SHARE, LAST, 8, 6, 64>, 8, 64);
  return run(dropout_kernel<T, SHARE, LAST, 8, 8, 64>, 8, 64);
}
template <typename T, bool LAST>
int launch(const char* what, int share, Dropout& d, int batch, const void* src, void* dst, hipStream_t st) {
  return share == kElement ? launch_share<T, kElement, LAST>(what, d, batch, src, dst, st)
         : share == kPixel ? launch_share<T, kPixel, LAST>(what, d, batch, src, dst, st)
                           : launch_share<T, kLabel, LAST>(what, d, batch, src, dst, st);
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
  if (pixels > ((int64_t)1 << 40)) return fail(MPL_EINVAL, "%s: too many pixels", what);
  Dropout d;
  d.state = state;
  d.pixels = pixels;
  d.labels = n_disp;
  d.reciprocal = n_disp > 1 ? (uint32_t)((((uint64_t)1 << 32) + (uint64_t)n_disp - 1) / (uint64_t)n_disp) : 0u;
  d.whole_quads = n_disp % 4 == 0 && ((uintptr_t)(LAST ? dst : src) & 15) == 0;
  // Where rows are not whole cache lines the tiles beside each other share lines, which one die's L2 can join.  us forward
  // / backward, tiles dealt out one by one -> groups of 8 -> 16: fp32 192 labels 377x501 57.5 / 64.2 -> 52.2 / 59.4 -> 51.1 /
  // 58.3, 97 labels 301x803 40.6 / 38.5 -> 34.7 / 36.3 -> 34.4 / 35.3, fp16 128 labels 375x1242 77.7 / 82.6 -> 74.9 / 73.7 ->
  // 74.9 / 73.9, bf16 21 labels 12x129x129 9.2 / 8.8 -> 9.7 / 8.9 -> 9.7 / 8.8.
  d.xcd_group = pixels * (dtype == MPL_F32 ? 4 : 2) % kLineBytes != 0 ? 16 : 0;
  d.nothing = rate >= 1;
  d.bound = d.nothing ? 0u : (uint32_t)(rate * 4294967296.0);
  d.scale = d.nothing ? 0.f : (float)(1.0 / (1.0 - rate));
  const hipStream_t st = (hipStream_t)stream;
  return dtype == MPL_F32   ? launch<float, LAST>(what, share, d, batch, src, dst, st)
         : dtype == MPL_F16 ? launch<_Float16, LAST>(what, share, d, batch, src, dst, st)
                            : launch<__bf16, LAST>(what, share, d, batch, src, dst, st);
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
