// Layer norm of the unary costs over the labels of a pixel, within the change to the layers' layout, for gfx950.
//
// x in the network's layout (items, labels, pixels) or in the operators' (items, pixels, labels), fp32, fp16 or bf16
//   ->  y (items, pixels, labels) fp32:   y[l] = xhat[l] * weight[l] + bias[l],   xhat[l] = (x[l] - mean) * r,
//   r = 1 / sqrt(var + eps), mean and var over the labels of the pixel; and its gradient, with g[l] = dy[l] * weight[l]:
//   dx[l] = r * (g[l] - mean(g) - xhat[l] * mean(g * xhat)),   dweight[l] = sum over pixels of dy[l] * xhat[l],
//   dbias[l] = sum over pixels of dy[l].
//
// The mean is that of the differences from a first label, so that it is exact where the labels have one cost, and the variance that
// of the differences from the mean, in registers: each wavefront's own labels first, and those of the W wavefronts of a tile
// joined as sum(M2_w + n_w * (mean_w - mean)^2).  Where squares do not fit fp32 (costs 2^64 apart, a mask of the type's largest
// number) the pixel's costs are taken 2^-70 as large, and 2^100 times where they and eps are too small for it (costs 2^-50 apart
// without eps), which leaves xhat as it is.  Mean and r are kept for the gradient, 8 bytes a
// pixel, from 17 labels on; of fewer it forms them again from x, which it reads in any case.
//
// Bound by HBM: a pixel's labels are read once, and the change of layout is one that the layer makes anyway.  The sums over
// pixels stay in registers while a workgroup goes from tile to tile: a fp32 sum for each lane and label, then over the 64
// lanes, and the workgroups' sums in 64 bits and in their order by a second kernel, so that the same call gives the same bits.
// (The first of these in 32 bits is a choice: they take two registers a label, as it is what the shapes of the gradient go by, and
// a lane adds one term to its sum per tile.  Of N tiles to a workgroup a sum is off by at most (N + 16) 2^-24 of the sum of the
// terms' sizes, and of 100 tiles, with terms of one sign, was by 4e-8.)
// us, forward / gradient with all sums: fp32, 192 labels 1500x2000 858 / 1364 (5.4 and 5.1 TB/s, where a large copy moves
// 4.7); bf16, 21 labels 12x129x129 10.4 / 16.2; 97 labels 301x803 in the operators' layout 40 / 64.

#include <algorithm>

#include "mp_pixels.h"

using namespace mpl;

namespace {

// Labels up to which the gradient forms mean and r again.  us for 40 M costs, forward / gradient, kept -> formed again: 2 labels
// 129 / 123 -> 114 / 114, 4: 73 / 115 -> 66 / 99, 8: 68 / 105 -> 62 / 97, 16: 64 / 107 -> 60 / 102; 21: 66 / 117 -> 62 / 115, labels last
// 67 / 107 -> 63 / 116, bf16 44 / 76 -> 43 / 84, 4.2 M bf16 costs 8.4 / 14.7 -> 8.3 / 17.6 (registers and instructions).
constexpr int kFormedAgain = 16;
constexpr unsigned kSumRows = 2048;  // workgroups of a gradient, at most

struct Norm {
  Tiles t;
  const void* x;
  const float* weight;  // or nullptr: 1
  const float* bias;    // or nullptr: 0
  float* y;
  float* stats;  // mean and r of each pixel, or nullptr
  const float* dy;
  void* dx;      // or nullptr
  float* sums;   // of each workgroup: dweight, dbias
  float eps;
  int x_mode, y_mode;  // of runs in the operators' layout
};

// Up to four labels no run is one of fours (mode_of).
template <int W, int I>
constexpr bool kFoursToo = W * I > 1;
template <int W, int I>
__device__ __forceinline__ int run_mode_here(int mode, int64_t first, unsigned total) {
  return kFoursToo<W, I> ? run_mode_of(mode, first, total) : mode;
}

// labels that wavefront w of W has
template <int W, int I>
__device__ __forceinline__ int labels_of(int w, int n) {
  int count = 0;
#pragma unroll
  for (int i = 0; i < I; ++i) count += min(max(n - 4 * (w + i * W), 0), 4);
  return count;
}

// Mean and squared differences from it of this wavefront's labels of a pixel,
template <int W, int I>
__device__ __forceinline__ float2 own_moments(const float (&x)[I][4], int w, int n) {
  const auto is = [&](int i, int j) { return 4 * (w + i * W) + j < n; };
  float sum = 0, m2 = 0;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += is(i, j) ? x[i][j] - x[0][0] : 0.f;
  const int here = labels_of<W, I>(w, n);
  const float mean = here > 0 ? x[0][0] + sum / (float)here : 0.f;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = is(i, j) ? x[i][j] - mean : 0.f;
      m2 += d * d;
    }
  return float2{mean, m2};
}
// and the mean and variance + eps of the pixel from those of all W.
template <int W, int I>
__device__ __forceinline__ float2 join_moments(const float2 (*part)[kTilePixels], int lane, int n, float eps) {
  const float labels = (float)n;
  float2 of_wave[W];
  float sum = 0, m2 = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    of_wave[k] = part[k][lane];
    sum += (of_wave[k].x - of_wave[0].x) * (float)labels_of<W, I>(k, n);
  }
  const float mean = W > 1 ? of_wave[0].x + sum / labels : of_wave[0].x;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    const float d = of_wave[k].x - mean;
    m2 += W > 1 ? of_wave[k].y + (float)labels_of<W, I>(k, n) * d * d : of_wave[k].y;
  }
  return float2{mean, m2 / labels + eps};
}

constexpr float kFar = 0x1p-70f, kClose = 0x1p100f;

// r as it is kept: negative where the costs and the mean are kFar as large, and r is of those (2^-59 to 2^6 then: a variance beyond
// 2^128 becomes one of 2^-12 to 2^118); below kCloseMark where they are kClose times as large (r is 2^-50 to 2^53, kept
// 2^60 times as large).
constexpr float kCloseMark = -0x1p8f;
__device__ __forceinline__ bool is_close(float kept) { return kept < kCloseMark; }
__device__ __forceinline__ float r_of(float kept) { return is_close(kept) ? kept * -0x1p-60f : fabsf(kept); }
__device__ __forceinline__ float scale_of(float kept) { return is_close(kept) ? kClose : kept < 0 ? kFar : 1.f; }

// Mean and r of the lane's pixel, r as it is kept, and the costs as large as it says.  All wavefronts of a tile come to the
// same.  part: of the W wavefronts that share the tile.
template <int W, int I>
__device__ __forceinline__ float2 moments(float (&x)[I][4], float2 (*part)[kTilePixels], int w, int lane, int n, float eps) {
  part[w][lane] = own_moments<W, I>(x, w, n);
  if (W > 1) tile_sync<W>();
  float2 of = join_moments<W, I>(part, lane, n, eps);
  float mark = 1;
  if (__builtin_amdgcn_ballot_w64(!(of.y >= 0x1p-100f && of.y < __builtin_huge_valf())) != 0) {
    if (W > 1) tile_sync<W>();  // (the parts are read)
    // (costs of 2^-10 or more are further apart than 2^-50, or all the same)
    const bool far = !(of.y < __builtin_huge_valf()), close = of.y < 0x1p-100f && fabsf(of.x) < 0x1p-10f;
    const float scale = far ? kFar : close ? kClose : 1.f;
    mark = far ? -1.f : close ? -0x1p60f : 1.f;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][j] *= scale;
    part[w][lane] = own_moments<W, I>(x, w, n);
    if (W > 1) tile_sync<W>();
    of = join_moments<W, I>(part, lane, n, eps * scale * scale);
  }
  return float2{of.x, 1.f / sqrtf(of.y) * mark};
}

template <typename T, bool FIRST, int W, int I, int G>
__global__ void __launch_bounds__(64 * W * G) norm_kernel(Norm p) {
  constexpr int kStride = tile_stride(W * I);
  __shared__ __align__(16) float tiles[G * kTilePixels * kStride];
  __shared__ __align__(16) float affine[2][4 * W * I];
  __shared__ float2 part[W * G][kTilePixels];
  const int tid = (int)threadIdx.x % (64 * W), group = uniform_i((int)threadIdx.x / (64 * W));
  const int lane = tid % 64, w = uniform_i(tid / 64), n = p.t.labels;
  const unsigned at = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group) * G + group;
  const bool work = at < p.t.total;
  const unsigned item = at / p.t.per_item;
  const int64_t p0 = (int64_t)(at - item * p.t.per_item) * kTilePixels;
  const int count = work ? (int)min((int64_t)kTilePixels, p.t.pixels - p0) : 0;
  const unsigned total = (unsigned)(count * n);
  const int of = min(lane, count - 1);
  const int64_t first = (int64_t)item * n * p.t.pixels, run = first + p0 * n;
  float* const tile = tiles + group * kTilePixels * kStride;
  float* const mine = tile + lane * kStride;
  float x[I][4];
  if (work) {
    if (FIRST) {
      load_rows<W, I>((const T*)p.x + first + p0, p.t, w, of, x);
    } else {
      Run<I, T> r;
      const int mode = run_mode_here<W, I>(p.x_mode, first, total);
      load_run<W, I, kFoursToo<W, I>>((const T*)p.x + run, total, mode, tid, r);
      run_to_tile<W, I, kFoursToo<W, I>>(r, total, mode, tid, p.t, tile);
    }
  }
  for (int i = (int)threadIdx.x; i < 4 * W * I; i += 64 * W * G) {
    affine[0][i] = i >= n ? 0.f : p.weight != nullptr ? p.weight[i] : 1.f;
    affine[1][i] = i >= n || p.bias == nullptr ? 0.f : p.bias[i];
  }
  __syncthreads();
  if (!work) return;
  if (!FIRST) from_tile<W, I>(mine, w, x);
  const float2 of_pixel = moments<W, I>(x, part + group, w, lane, n, p.eps);
  float r = of_pixel.y;
  if (__builtin_amdgcn_ballot_w64(r < 0) != 0) r = r_of(r);
  if (p.stats != nullptr && w == 0 && lane < count)
    reinterpret_cast<float2*>(p.stats)[(int64_t)item * p.t.pixels + p0 + lane] = of_pixel;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int l = 4 * (w + i * W) + j;
      x[i][j] = (x[i][j] - of_pixel.x) * r * affine[0][l] + affine[1][l];
    }
  to_tile<W, I>(mine, w, x);
  tile_sync<W>();
  store_run<W, I, kFoursToo<W, I>>(p.y + run, total, run_mode_here<W, I>(p.y_mode, first, total), tid, p.t, tile);
}

// SUMS: with the sums over pixels that dweight and dbias are made of.
template <typename T, bool FIRST, bool SUMS, int W, int I, int G>
__global__ void __launch_bounds__(64 * W * G, I <= 4 ? 4 : 1) norm_grad_kernel(Norm p) {
  constexpr int kStride = tile_stride(W * I);
  __shared__ __align__(16) float tiles[G * kTilePixels * kStride];
  __shared__ __align__(16) float weight[4 * W * I];
  __shared__ float2 part[W * G][kTilePixels];
  constexpr bool kAgain = 4 * W * I <= kFormedAgain;
  __shared__ float2 part_again[kAgain ? W * G : 1][kTilePixels];
  const int tid = (int)threadIdx.x % (64 * W), group = uniform_i((int)threadIdx.x / (64 * W));
  const int lane = tid % 64, w = uniform_i(tid / 64), n = p.t.labels;
  float* const tile = tiles + group * kTilePixels * kStride;
  float* const mine = tile + lane * kStride;
  for (int i = (int)threadIdx.x; i < 4 * W * I; i += 64 * W * G)
    weight[i] = i >= n ? 0.f : p.weight != nullptr ? p.weight[i] : 1.f;
  __syncthreads();
  const float per_label = 1.f / (float)n;
  float dw[SUMS ? I : 1][4] = {}, db[SUMS ? I : 1][4] = {};
  for (unsigned at = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group) * G + group; at < p.t.total;
       at += gridDim.x * G) {
    const unsigned item = at / p.t.per_item;
    const int64_t p0 = (int64_t)(at - item * p.t.per_item) * kTilePixels;
    const int count = (int)min((int64_t)kTilePixels, p.t.pixels - p0);
    const unsigned total = (unsigned)(count * n);
    const int of = min(lane, count - 1);
    const int64_t first = (int64_t)item * n * p.t.pixels, run = first + p0 * n;
    float x[I][4], d[I][4];
    Run<I, float> dy;
    const int x_mode = run_mode_here<W, I>(p.x_mode, first, total), y_mode = run_mode_here<W, I>(p.y_mode, first, total);
    load_run<W, I, kFoursToo<W, I>>(p.dy + run, total, y_mode, tid, dy);
    float2 of_pixel;
    if (!kAgain) of_pixel = reinterpret_cast<const float2*>(p.stats)[(int64_t)item * p.t.pixels + p0 + of];
    if (FIRST) {
      load_rows<W, I>((const T*)p.x + first + p0, p.t, w, of, x);
    } else {
      Run<I, T> rx;
      load_run<W, I, kFoursToo<W, I>>((const T*)p.x + run, total, x_mode, tid, rx);
      run_to_tile<W, I, kFoursToo<W, I>>(rx, total, x_mode, tid, p.t, tile);
      tile_sync<W>();
      from_tile<W, I>(mine, w, x);
      tile_sync<W>();
    }
    run_to_tile<W, I, kFoursToo<W, I>>(dy, total, y_mode, tid, p.t, tile);
    if (kAgain) of_pixel = moments<W, I>(x, part_again + group, w, lane, n, p.eps);
    float r = of_pixel.y, r_of_x = r;
    const bool scaled = __builtin_amdgcn_ballot_w64(of_pixel.y < 0) != 0;
    if (scaled) {
      if (!kAgain) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] *= scale_of(of_pixel.y);
      }
      // (of close costs r * kClose may be beyond fp32 where the gradient is not: half of the scale here, half behind)
      r = r_of(of_pixel.y);
      r_of_x = is_close(of_pixel.y) ? r * 0x1p50f : r * scale_of(of_pixel.y);
    }
    if (!kAgain || W == 1) tile_sync<W>();
    from_tile<W, I>(mine, w, d);
    float s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int l = 4 * (w + i * W) + j;
        // (behind the last label or pixel of a tile in LDS lies an earlier one's, or no number at all)
        const bool in = l < n && lane < count;
        d[i][j] = in ? d[i][j] : 0.f;
        x[i][j] = in ? (x[i][j] - of_pixel.x) * r : 0.f;
        if (SUMS) {
          dw[i][j] += d[i][j] * x[i][j];
          db[i][j] += d[i][j];
        }
        d[i][j] *= weight[l];
        s1 += d[i][j];
        s2 += d[i][j] * x[i][j];
      }
    if (W > 1) {
      part[w][lane] = float2{s1, s2};
      tile_sync<W>();
      s1 = s2 = 0;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float2 of_wave = part[k][lane];
        s1 += of_wave.x;
        s2 += of_wave.y;
      }
    }
    if (p.dx != nullptr) {
      s1 *= per_label;
      s2 *= per_label;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = r_of_x * (d[i][j] - s1 - x[i][j] * s2);
      if (scaled) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] *= is_close(of_pixel.y) ? 0x1p50f : 1.f;
      }
      if (FIRST) {
        if (lane < count) store_rows<W, I>((T*)p.dx + first + p0, p.t, w, lane, x);
      } else {
        to_tile<W, I>(mine, w, x);
        tile_sync<W>();
        store_run<W, I, kFoursToo<W, I>>((T*)p.dx + run, total, x_mode, tid, p.t, tile);
      }
    }
    tile_sync<W>();  // (the next tile overwrites this one and its parts)
  }
  if (SUMS) {
    // over the lanes, and the G wavefronts that had tiles of their own
    __shared__ float ends[G][2][4 * W * I];
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = wave_sum(dw[i][j]), b = wave_sum(db[i][j]);
        if (lane == 0) {
          ends[group][0][4 * (w + i * W) + j] = a;
          ends[group][1][4 * (w + i * W) + j] = b;
        }
      }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < 2 * n; i += 64 * W * G) {
      float sum = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) sum += i < n ? ends[g][0][i] : ends[g][1][i - n];
      p.sums[(int64_t)blockIdx.x * 2 * n + i] = sum;
    }
  }
}

// The workgroups' rows of 2 * n sums, a column to every 16th thread, in 64 bits.
__global__ void __launch_bounds__(1024) norm_sums_kernel(const float* __restrict__ sums, int rows, int n, float* __restrict__ dweight,
                                                       float* __restrict__ dbias) {
  __shared__ double part[64][17];
  const int of = (int)threadIdx.x % 16, by = (int)threadIdx.x / 16, column = (int)blockIdx.x * 16 + of;
  double sum = 0;
  if (column < 2 * n) {
#pragma unroll 8
    for (int row = by; row < rows; row += 64) sum += (double)sums[(int64_t)row * 2 * n + column];
  }
  part[by][of] = sum;
  __syncthreads();
  if (by == 0 && column < 2 * n) {
    sum = 0;
#pragma unroll
    for (int k = 0; k < 64; ++k) sum += part[k][of];
    if (column < n) {
      if (dweight != nullptr) dweight[column] = (float)sum;
    } else if (dbias != nullptr) {
      dbias[column - n] = (float)sum;
    }
  }
}

int status(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// The gradient's shapes: fewer labels to a wavefront, whose sums over the pixels take two registers each.  us, with the shapes of
// the forward pass -> these: bf16, 21 labels 12x129x129 19.5 -> 12.3, 16 labels 64x96 6.8 -> 4.1; images of 64 M costs the same
// but for 21 labels (172 -> 179) and 8 (179 -> 165).  Up to 16 labels to a wavefront in 128 registers, so that two workgroups of
// eight share a compute unit: 97 labels 301x803 in the operators' layout 101 -> 71 when it was taken.
template <typename F>
void with_grad_shape(int n, F f) {
  if (n <= 4)
    f(TileShape<1, 1, 4>());
  else if (n <= 8)
    f(TileShape<2, 1, 1>());
  else if (n <= 16)
    f(TileShape<4, 1, 1>());
  else if (n <= 24)
    f(TileShape<3, 2, 1>());
  else if (n <= 32)
    f(TileShape<4, 2, 1>());
  else if (n <= 48)
    f(TileShape<6, 2, 1>());
  else if (n <= 64)
    f(TileShape<8, 2, 1>());
  else if (n <= 96)
    f(TileShape<8, 3, 1>());
  else if (n <= 128)
    f(TileShape<8, 4, 1>());
  else if (n <= 192)
    f(TileShape<8, 6, 1>());
  else
    f(TileShape<8, 8, 1>());
}

// Workgroups of a gradient, each with as many tiles as the others.  Those of eight wavefronts are a quarter as many: 192 labels
// 1500x2000 as fast with 512 as with 2048, the sum of their rows 12 -> 6 us.  Of four wavefronts seven are resident to a compute unit
// and not eight where they need more than 80 scalar registers (16 more are set aside for each), and what is left over
// makes a second round.  us with 2048 -> 1792, 40 M costs: 2 labels 142 -> 115, 3 120 -> 98, 4 108 -> 99, 12 130 -> 109, 16 118 ->
// 103; of two wavefronts 6 labels 112 -> 119, 8 97 -> 97, not taken.
unsigned grad_blocks(unsigned tiles, int waves, int per_block) {
  const unsigned most = waves >= 8 ? kSumRows / 4 : waves == 4 ? kSumRows / 8 * 7 : kSumRows, groups = (tiles + (unsigned)per_block - 1) / (unsigned)per_block;
  const unsigned rounds = (groups + most - 1) / most;
  return (groups + rounds - 1) / rounds;
}

template <typename T, bool FIRST>
void launch(const Norm& p, hipStream_t st) {
  with_shape(p.t.labels, [&](auto s) {
    constexpr int W = s.kW, I = s.kI, G = s.kG;
    norm_kernel<T, FIRST, W, I, G><<<(p.t.total + G - 1) / G, 64 * W * G, 0, st>>>(p);
  });
}
template <typename T, bool FIRST>
void launch_grad(const Norm& p, float* dweight, float* dbias, hipStream_t st) {
  with_grad_shape(p.t.labels, [&](auto s) {
    constexpr int W = s.kW, I = s.kI, G = s.kG;
    const unsigned blocks = grad_blocks(p.t.total, W * G, G);
    if (p.sums == nullptr) {
      norm_grad_kernel<T, FIRST, false, W, I, G><<<blocks, 64 * W * G, 0, st>>>(p);
      return;
    }
    norm_grad_kernel<T, FIRST, true, W, I, G><<<blocks, 64 * W * G, 0, st>>>(p);
    norm_sums_kernel<<<(2 * p.t.labels + 15) / 16, 1024, 0, st>>>(p.sums, (int)blocks, p.t.labels, dweight, dbias);
  });
}
template <typename F>
void with_type(int dtype, bool labels_first, F f) {
  const auto by_layout = [&](auto type) {
    labels_first ? f(type, std::true_type()) : f(type, std::false_type());
  };
  if (dtype == MPL_F32)
    by_layout(float());
  else if (dtype == MPL_F16)
    by_layout((_Float16)0);
  else
    by_layout((__bf16)0);
}

int prepare(const char* what, Norm& p, int dtype, bool labels_first, float eps, int batch, int n_disp, int64_t pixels) {
  if (dtype < 0 || dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d", what, dtype);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "%s: n_disp must be in [1, %d], got %d", what, kMaxL, n_disp);
  if (!(eps >= 0 && eps < __builtin_huge_valf())) return fail(MPL_EINVAL, "%s: eps must be finite and not below 0", what);
  if (batch < 0 || pixels < 0) return fail(MPL_EINVAL, "%s: negative size", what);
  if (batch > 0 && !make_tiles(p.t, batch, n_disp, pixels, labels_first, dtype == MPL_F32 ? 4 : 2))
    return fail(MPL_EINVAL, "%s: too many pixels", what);
  return MPL_OK;
}
// (Fours of up to three labels are of two pixels or more, and their kernels are without them.  us one by one -> four side by side, 40 M
// costs, forward and gradient: 2 labels 228 -> 223, labels last 243 -> 248, 3 184 -> 196 and 192 -> 191; 5 225 -> 209, 7 178 -> 172;
// labels last, 5 261 -> 241, 150 218 -> 195.)
int mode_of(const void* at, int n_disp, int dtype) {
  return n_disp < 4 ? (int)kEach : run_mode(n_disp, ((uintptr_t)at & (dtype == MPL_F32 ? 15 : 7)) == 0);
}

}  // namespace

extern "C" {

int64_t mpl_norm_workspace(int batch, int n_disp, int64_t pixels) {
  if (batch <= 0 || pixels <= 0 || n_disp < 1 || n_disp > kMaxL) return 0;
  const int64_t per_item = (pixels + kTilePixels - 1) / kTilePixels;
  const int64_t rows = per_item > (int64_t)kSumRows / batch ? (int64_t)kSumRows : per_item * batch;
  return rows * 2 * n_disp;
}

int mpl_norm_stats(int n_disp) { return n_disp > kFormedAgain ? 2 : 0; }

int mpl_norm_labels_last(int dtype, int labels_first, const void* src, const float* weight, const float* bias, float eps,
                         float* dst, float* stats, int batch, int n_disp, int64_t pixels, void* stream) {
  Norm p = {};
  const int rc = prepare("norm_labels_last", p, dtype, labels_first != 0, eps, batch, n_disp, pixels);
  if (rc != MPL_OK) return rc;
  if (batch == 0 || pixels == 0) return MPL_OK;
  if (src == nullptr || dst == nullptr) return fail(MPL_EINVAL, "norm_labels_last: null pointer");
  p.x = src;
  p.weight = weight;
  p.bias = bias;
  p.y = dst;
  p.stats = n_disp > kFormedAgain ? stats : nullptr;
  p.eps = eps;
  p.x_mode = mode_of(src, n_disp, dtype);
  p.y_mode = mode_of(dst, n_disp, MPL_F32);
  with_type(dtype, labels_first != 0, [&](auto type, auto first) { launch<decltype(type), first.value>(p, (hipStream_t)stream); });
  return status("norm_labels_last");
}

int mpl_norm_labels_last_grad(int dtype, int labels_first, const void* src, const float* weight, float eps,
                              const float* stats, const float* ddst, void* dsrc, float* dweight, float* dbias, float* workspace,
                              int batch, int n_disp, int64_t pixels, void* stream) {
  Norm p = {};
  const int rc = prepare("norm_labels_last_grad", p, dtype, labels_first != 0, eps, batch, n_disp, pixels);
  if (rc != MPL_OK) return rc;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (batch == 0 || pixels == 0) {
    // (a sum of nothing)
    if (sums) norm_sums_kernel<<<(2 * n_disp + 15) / 16, 1024, 0, (hipStream_t)stream>>>(nullptr, 0, n_disp, dweight, dbias);
    return sums ? status("norm_labels_last_grad") : MPL_OK;
  }
  if (src == nullptr || ddst == nullptr || (stats == nullptr && n_disp > kFormedAgain) || (sums && workspace == nullptr))
    return fail(MPL_EINVAL, "norm_labels_last_grad: null pointer");
  if (dsrc == nullptr && !sums) return MPL_OK;
  p.x = src;
  p.weight = weight;
  p.eps = eps;
  p.stats = const_cast<float*>(stats);
  p.dy = ddst;
  p.dx = dsrc;
  p.sums = sums ? workspace : nullptr;
  p.x_mode = std::min(mode_of(src, n_disp, dtype), mode_of(dsrc, n_disp, dtype));
  p.y_mode = mode_of(ddst, n_disp, MPL_F32);
  with_type(dtype, labels_first != 0,
            [&](auto type, auto first) { launch_grad<decltype(type), first.value>(p, dweight, dbias, (hipStream_t)stream); });
  return status("norm_labels_last_grad");
}

}  // extern "C"
