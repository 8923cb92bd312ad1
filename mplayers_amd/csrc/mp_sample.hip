// Labels drawn from the layers' costs, for gfx950.
//
// A pixel's costs c[l] are energies: label l has weight w[l] = exp((best - c[l]) / T).  Of the labels that top_k,
// top_p and min_p leave, in label order, the first one whose running sum exceeds u * (sum of all) is drawn, u given
// by the caller.  Costs of +inf and NaN are no candidates, T <= 0 is top_k = 1, equal costs order by label.
//
// All three filters keep the best labels down to a threshold (a cost, and how many of the labels that have exactly
// that cost): top_k the cost of the k-th best, top_p the least cost whose labels down to it weigh enough, min_p
// best + T * ln(1 / min_p).  So no sort: the threshold is found by halving the range of costs, each step moving an
// end to a cost that occurs.
//
// Which label is drawn must not depend on how the sums are formed, or two correct programs would disagree on the
// pixels whose target falls next to a border: weights and sums are held in 64 bits, which leaves borders of a
// relative width of 2^-52.

#include "mp_common.h"

using namespace mpl;

namespace {

constexpr int kPixels = 64;  // pixels of a workgroup

struct Sample {
  const float* cost;
  const float* uniforms;
  uint8_t* labels;
  const float* temperature;  // one per image, or nullptr for the number below
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t pixels, tiles, items_pixels;
  int n, n_cv, n_draws;
};

constexpr float kInf = __builtin_huge_valf();

// +inf for what is no candidate, and one zero: comparisons of the results are those of numbers.  By bits: the library
// is compiled for code without NaNs.
__device__ __forceinline__ float candidate(float c) {
  const int bits = __builtin_bit_cast(int, c);
  const float clean = (bits & 0x7fffffff) > 0x7f800000 ? kInf : c;
  return clean == 0.f ? 0.f : clean;
}
// x > 0 and a number, x >= 1 or no number
__device__ __forceinline__ bool positive(float x) {
  const int bits = __builtin_bit_cast(int, x);
  return bits > 0 && bits <= 0x7f800000;
}

// Reductions over the S lanes of a pixel, neighbours within a row of 16.
template <int CTRL>
__device__ __forceinline__ int move_i(int x) {
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float move(float x) {
  return __builtin_bit_cast(float, move_i<CTRL>(__builtin_bit_cast(int, x)));
}
template <int CTRL>
__device__ __forceinline__ int move(int x) {
  return move_i<CTRL>(x);
}
template <int CTRL>
__device__ __forceinline__ double move(double x) {
  const int64_t bits = __builtin_bit_cast(int64_t, x);
  const uint32_t lo = (uint32_t)move_i<CTRL>((int)(uint32_t)bits), hi = (uint32_t)move_i<CTRL>((int)(bits >> 32));
  return __builtin_bit_cast(double, (int64_t)(((uint64_t)hi << 32) | lo));
}
template <int S, typename V, typename F>
__device__ __forceinline__ V over_lanes(V x, F f) {
  if (S > 1) x = f(x, move<0xB1>(x));   // the other of a pair
  if (S > 2) x = f(x, move<0x4E>(x));   // the other pair of four
  if (S > 4) x = f(x, move<0x141>(x));  // the other four of eight
  if (S > 8) x = f(x, move<0x140>(x));  // the other eight
  return x;
}
template <int S>
__device__ __forceinline__ float lanes_min(float x) {
  return over_lanes<S>(x, [](float a, float b) { return b < a ? b : a; });
}
template <int S>
__device__ __forceinline__ float lanes_max(float x) {
  return over_lanes<S>(x, [](float a, float b) { return b > a ? b : a; });
}
template <int S, typename V>
__device__ __forceinline__ V lanes_sum(V x) {
  return over_lanes<S>(x, [](V a, V b) { return a + b; });
}
// sum of the lanes before this one, one after the other: a lane that adds nothing leaves the bits as they are
template <int S, typename V>
__device__ __forceinline__ V lanes_before(V x, int s) {
  V upto = x;
#pragma unroll
  for (int i = 1; i < S; ++i) {
    const V left = move<0x111>(upto);
    if (s == i) upto = left + x;
  }
  const V left = S > 1 ? move<0x111>(upto) : x;
  return s == 0 ? V(0) : left;
}

// The least cost t of the pixel's with sum(of labels with v <= t) >= target, from `from` (the best) on; `to` (the
// worst candidate) where no sum reaches it.
template <int NV, int S, typename V, typename SumUpTo>
__device__ __forceinline__ float threshold(const float (&v)[NV], float from, float to, V target, SumUpTo sum_up_to) {
  float lo = from, hi = to;
  for (int step = 0; __builtin_amdgcn_ballot_w64(lo < hi) != 0; ++step) {
    // Halves the costs, and after a while what lies between their bit patterns: costs that grow from one to the next
    // by factors would lose one a step.
    float mid = 0.5f * lo + 0.5f * hi;
    if (step >= 10) {
      const int a = float_key(__builtin_bit_cast(int, lo)), b = float_key(__builtin_bit_cast(int, hi));
      mid = __builtin_bit_cast(float, float_key((int)(((int64_t)a + b) >> 1)));
    }
    if (!(mid >= lo && mid < hi)) mid = lo;
    float below = lo, above = hi;
    V sum = V(0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = v[j] <= mid;
      if (in) below = v[j] > below ? v[j] : below;
      if (!in) above = v[j] < above ? v[j] : above;
      sum += in ? sum_up_to(j) : V(0);
    }
    sum = lanes_sum<S>(sum);
    below = lanes_max<S>(below);
    above = lanes_min<S>(above);
    if (lo < hi) {
      if (sum >= target)
        hi = below;
      else
        lo = above;
    }
  }
  return hi;
}

// S lanes per pixel, NV labels per lane: lane s owns labels s * NV ... s * NV + NV - 1.
template <int NV, int S, bool FILTER, bool LAST>
__global__ void __launch_bounds__(kPixels* S) sample_kernel(Sample p) {
  constexpr int kQuads = S * NV / 4, kJ = NV / 4;  // of four labels: in all, per lane
  constexpr int kStride = 4 * (kQuads | 1);
  __shared__ __align__(16) float tile[kPixels * kStride];
  const int64_t block = (int64_t)blockIdx.x;
  const int64_t item = block / p.tiles, p0 = (block - item * p.tiles) * kPixels;
  const int count = (int)min((int64_t)kPixels, p.pixels - p0);
  const int tid = (int)threadIdx.x;
  const float* cost = p.cost + item * p.n * p.pixels;
  // the quads of a pixel lie in the order in which its lanes read them: quad q, of lane q / kJ, at place q % kJ * S + q / kJ
  const auto place = [](int l) { return ((l >> 2) % kJ * S + (l >> 2) / kJ) * 4 + (l & 3); };
  if (LAST) {
    for (int i = tid; i < count * p.n; i += kPixels * S) tile[i / p.n * kStride + place(i % p.n)] = cost[p0 * p.n + i];
  } else {
    const int px = tid % kPixels;
    if (px < count)
      for (int l = tid / kPixels; l < p.n; l += S) tile[px * kStride + place(l)] = cost[l * p.pixels + p0 + px];
  }
  __syncthreads();
  const int px = tid / S, s = tid % S;
  if (px >= count) return;  // (whole pixels: the lanes of one stay or go together)
  float v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    v[j] = s * NV + j < p.n ? candidate(tile[px * kStride + ((j >> 2) * S + s) * 4 + (j & 3)]) : kInf;
  float best = v[0];
#pragma unroll
  for (int j = 1; j < NV; ++j) best = v[j] < best ? v[j] : best;
  best = lanes_min<S>(best);

  const int image = (int)(item / p.n_cv);
  const float t32 = p.temperature != nullptr ? p.temperature[image] : p.temperature_all;
  const bool warm = positive(t32);
  const double inv_t = warm ? 1.0 / (double)t32 : 0.0;
  double w[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const double e = exp(((double)best - (double)v[j]) * inv_t);
    w[j] = !(v[j] < kInf) ? 0.0 : v[j] == best ? 1.0 : best == -kInf ? 0.0 : e;
  }

  if (FILTER) {
    const auto worst = [&]() {
      float m = best;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (v[j] < kInf) m = v[j] > m ? v[j] : m;
      return lanes_max<S>(m);
    };
    // takes out what is worse than t, and of the labels at t those behind the first `ties`
    const auto cut = [&](float t, auto stays) {
      int at = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) at += v[j] == t ? 1 : 0;
      int rank = lanes_before<S>(at, s);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const bool tie = v[j] == t;
        if (v[j] > t || (tie && !stays(rank))) {
          v[j] = kInf;
          w[j] = 0.0;
        }
        rank += tie ? 1 : 0;
      }
    };
    int k = p.top_k != nullptr ? p.top_k[image] : p.top_k_all;
    if (k <= 0) k = p.n;
    if (!warm) k = 1;
    if (k < p.n) {
      const float t = threshold<NV, S, int>(v, best, worst(), k, [](int) { return 1; });
      int less = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) less += v[j] < t ? 1 : 0;
      less = lanes_sum<S>(less);
      cut(t, [&](int rank) { return less + rank < k; });
    }
    const float top_p = p.top_p != nullptr ? p.top_p[image] : p.top_p_all;
    if (top_p < 1.f) {
      double total = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) total += w[j];
      const double target = (double)top_p * lanes_sum<S>(total);
      const float t = threshold<NV, S, double>(v, best, worst(), target, [&](int j) { return w[j]; });
      double less = 0, at = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        less += v[j] < t ? w[j] : 0.0;
        if (v[j] == t) at = w[j];
      }
      less = lanes_sum<S>(less);
      at = over_lanes<S>(at, [](double a, double b) { return a > b ? a : b; });
      cut(t, [&](int rank) { return less + rank * at < target || (t == best && rank == 0); });
    }
    const float min_p = p.min_p != nullptr ? p.min_p[image] : p.min_p_all;
    if (positive(min_p)) {
      const double reach = min_p >= 1.f ? 0.0 : -(double)t32 * log((double)min_p);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (v[j] != best && (double)v[j] - (double)best > reach) w[j] = 0.0;
    }
  }

  int last = 0;
  double sum = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (w[j] > 0) last = s * NV + j;
    sum += w[j];
    w[j] = sum;
  }
  const double before = lanes_before<S>(sum, s);
  // (lanes_sum would add in another order)
  const double total = over_lanes<S>(before + sum, [](double a, double b) { return a > b ? a : b; });
  last = over_lanes<S>(last, [](int a, int b) { return a > b ? a : b; });
  const int64_t at = item * p.pixels + p0 + px;
  for (int d = 0; d < p.n_draws; ++d) {
    const float u = p.uniforms[d * p.items_pixels + at];
    const double target = (positive(u) ? (double)u : 0.0) * total;
    int label = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) label += before + w[j] <= target ? 1 : 0;
    label = lanes_sum<S>(label);
    if (s == 0) p.labels[d * p.items_pixels + at] = (uint8_t)(label < last ? label : last);
  }
}

template <int NV, int S>
void launch(const Sample& p, bool filter, bool labels_first, unsigned blocks, hipStream_t st) {
  const auto run = [&](auto kernel) { kernel<<<blocks, kPixels * S, 0, st>>>(p); };
  if (filter)
    labels_first ? run(sample_kernel<NV, S, true, false>) : run(sample_kernel<NV, S, true, true>);
  else
    labels_first ? run(sample_kernel<NV, S, false, false>) : run(sample_kernel<NV, S, false, true>);
}

}  // namespace

extern "C" {

int mpl_sample_labels(int labels_first, const float* cost, const float* uniforms, int batch, int n_cv, int n_disp,
                      int64_t pixels, int n_draws, const float* temperatures, float temperature, const int32_t* top_ks,
                      int top_k, const float* top_ps, float top_p, const float* min_ps, float min_p, uint8_t* labels,
                      void* stream) {
  if (batch < 0 || n_cv < 0 || pixels < 0 || n_draws < 0) return fail(MPL_EINVAL, "sample_labels: negative size");
  if (n_disp < 1 || n_disp > kMaxL)
    return fail(MPL_EINVAL, "sample_labels: n_disp must be in [1, %d], got %d", kMaxL, n_disp);
  if (batch == 0 || n_cv == 0 || pixels == 0 || n_draws == 0) return MPL_OK;
  if (cost == nullptr || uniforms == nullptr || labels == nullptr)
    return fail(MPL_EINVAL, "sample_labels: null pointer");
  const int64_t items = (int64_t)batch * n_cv;
  const int64_t tiles = (pixels + kPixels - 1) / kPixels;
  if (items > 0x7fffffff || pixels > ((int64_t)1 << 40) || tiles * items > 0x7fffffff)
    return fail(MPL_EINVAL, "sample_labels: too many pixels");
  Sample p;
  p.cost = cost;
  p.uniforms = uniforms;
  p.labels = labels;
  p.temperature = temperatures;
  p.top_k = top_ks;
  p.top_p = top_ps;
  p.min_p = min_ps;
  p.temperature_all = temperature;
  p.top_k_all = top_k;
  p.top_p_all = top_p;
  p.min_p_all = min_p;
  p.pixels = pixels;
  p.tiles = tiles;
  p.items_pixels = items * pixels;
  p.n = n_disp;
  p.n_cv = n_cv;
  p.n_draws = n_draws;
  const bool filter = temperatures != nullptr || !(temperature > 0) || top_ks != nullptr || (top_k > 0 && top_k < n_disp) ||
                      top_ps != nullptr || top_p < 1.f || min_ps != nullptr || min_p > 0.f;
  const unsigned blocks = (unsigned)(tiles * items);
  const hipStream_t st = (hipStream_t)stream;
  const bool lf = labels_first != 0;
  // 16 labels a lane at most, in fours
  if (n_disp <= 4)
    launch<4, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 8)
    launch<8, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 12)
    launch<12, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 16)
    launch<16, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 24)
    launch<12, 2>(p, filter, lf, blocks, st);
  else if (n_disp <= 32)
    launch<16, 2>(p, filter, lf, blocks, st);
  else if (n_disp <= 48)
    launch<12, 4>(p, filter, lf, blocks, st);
  else if (n_disp <= 64)
    launch<16, 4>(p, filter, lf, blocks, st);
  else if (n_disp <= 96)
    launch<12, 8>(p, filter, lf, blocks, st);
  else if (n_disp <= 128)
    launch<16, 8>(p, filter, lf, blocks, st);
  else if (n_disp <= 192)
    launch<12, 16>(p, filter, lf, blocks, st);
  else
    launch<16, 16>(p, filter, lf, blocks, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "sample_labels: %s", hipGetErrorString(e));
}

}  // extern "C"
