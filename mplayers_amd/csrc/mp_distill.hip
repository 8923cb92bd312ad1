// The divergence of a layer's costs from a teacher's, of whose labels a list is kept, and its gradient, for gfx950.
//
// A pixel's student q = softmax(-c / T) over its labels; the teacher's classes are the entries (label, cost t) of its list and,
// where its cost is given, the rest of the labels as one.  p = softmax(-t / T) over the classes that are there.
//   loss = sum p (log p - log q(class)),   q(rest) = the sum of q over the labels that the list does not name
//   dloss/dc[l] = (p[l] - q[l]) / T for a label of the list (p summed over its entries),
//                 (p(rest) q[l] / q(rest) - q[l]) / T for another one
// With M = min c, Z = sum exp((M - c) / T) and the same for the classes (m, z) and the others (M', Z'):
//   log p - log q = ((c - M) - (t - m)) / T + log Z - log z,   log q(rest) = ((M - M') / T + log Z' - log Z)
// so no large numbers are subtracted that the costs do not have between them already, and the others may be as far from the best
// label as fp32 goes.  The gradient forms all this anew from the costs, which it reads in any case: nothing but its inputs is kept.
//
// An entry is there where its cost is not +inf, its label exists and the student's cost of that label is not +inf; the rest
// where its cost is not +inf and a label is left.  NaN (and -inf) goes through to the loss and the gradients of its pixel.
//
// A tile of 64 pixels, a lane to each (mp_pixels.h); the costs lie in LDS too, where the entries find the student's cost of
// their label.  Every wavefront of a tile goes through the whole list: W times as many instructions as one alone, but no
// further meeting.  Bound by HBM.

#include "mp_pixels.h"

using namespace mpl;

namespace {

constexpr float kInf = __builtin_huge_valf();

struct Distill {
  Tiles t;
  const void* cost;
  const uint8_t* labels;
  const void* costs;
  const float* rest;  // or nullptr
  float* loss;
  const float* dloss;
  void* dcost;
  int k, kept;               // entries of a list, type of their costs
  float to_exponent, inv_t;  // log2(e) / T, 1 / T
  int quads;                 // whole and aligned quads in the operators' layout
};

__device__ __forceinline__ float kept_cost(const Distill& p, int64_t at) {
  return p.kept == MPL_F32   ? ((const float*)p.costs)[at]
         : p.kept == MPL_F16 ? (float)((const _Float16*)p.costs)[at]
                             : (float)((const __bf16*)p.costs)[at];
}

// The least of some costs and the sum of their weights relative to it, (+inf, 0) of none.
struct Mass {
  float least, sum;
};
__device__ __forceinline__ float weight(float least, float c, float to_exponent) {
  return c == kInf ? 0.f : __builtin_amdgcn_exp2f((least - c) * to_exponent);
}
// Those of the W wavefronts of a tile; part: two floats for each and lane.
template <int W>
__device__ __forceinline__ Mass join(Mass own, float2 (*part)[kTilePixels], int w, int lane, float to_exponent) {
  if (W == 1) return own;
  part[w][lane] = float2{own.least, own.sum};
  tile_sync<W>();
  float2 of_wave[W];
  Mass all = {kInf, 0.f};
#pragma unroll
  for (int k = 0; k < W; ++k) {
    of_wave[k] = part[k][lane];
    all.least = of_wave[k].x < all.least ? of_wave[k].x : all.least;
  }
#pragma unroll
  for (int k = 0; k < W; ++k) all.sum += of_wave[k].y * weight(all.least, of_wave[k].x, to_exponent);
  return all;
}

template <typename T, bool FIRST, bool GRAD, int W, int I, int G>
__global__ void __launch_bounds__(64 * W * G) distill_kernel(Distill p) {
  constexpr int kStride = tile_stride(W * I), kShift = W == 1 ? 0 : W == 2 ? 1 : W == 4 ? 2 : 3;
  __shared__ __align__(16) float tiles[G * kTilePixels * kStride];
  __shared__ float2 part[2][W > 1 ? W : 1][kTilePixels];
  const int tid = (int)threadIdx.x % (64 * W), group = uniform_i((int)threadIdx.x / (64 * W));
  const int lane = tid % 64, w = uniform_i(tid / 64), n = p.t.labels;
  const unsigned at = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group) * G + group;
  if (at >= p.t.total) return;  // (W = 1: nobody waits for it)
  const unsigned item = at / p.t.per_item;
  const int64_t p0 = (int64_t)(at - item * p.t.per_item) * kTilePixels;
  const int count = (int)min((int64_t)kTilePixels, p.t.pixels - p0);
  const unsigned total = (unsigned)(count * n);
  const int of = min(lane, count - 1);
  const int64_t first = (int64_t)item * n * p.t.pixels, run = first + p0 * n, pixel = (int64_t)item * p.t.pixels + p0 + of;
  // of entry e of the lane's list
  const int64_t entry = FIRST ? (int64_t)item * p.k * p.t.pixels + p0 + of : pixel * p.k, step = FIRST ? p.t.pixels : 1;
  float* const tile = tiles + group * kTilePixels * kStride;
  float* const mine = tile + lane * kStride;
  float c[I][4];
  if (FIRST) {
    load_rows<W, I>((const T*)p.cost + first + p0, p.t, w, of, c);
    to_tile<W, I>(mine, w, c);
  } else {
    Run<I, T> r;
    load_run<W, I>((const T*)p.cost + run, total, p.quads, tid, r);
    run_to_tile<W, I>(r, total, p.quads, tid, p.t, tile);
    tile_sync<W>();
    from_tile<W, I>(mine, w, c);
  }
  // (labels behind the last are no candidates)
  const auto mass_of = [&](auto leave_out) {
    Mass m = {kInf, 0.f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) m.least = c[i][j] < m.least && !leave_out(i, j) ? c[i][j] : m.least;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) m.sum += leave_out(i, j) ? 0.f : weight(m.least, c[i][j], p.to_exponent);
    return m;
  };
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 4 * (w + i * W) + j < n ? c[i][j] : kInf;
  const Mass student = join<W>(mass_of([](int, int) { return false; }), part[0], w, lane, p.to_exponent);

  // the list: its least cost, and which of this wavefront's labels it names
  const auto exists = [&](int label, float t) { return t != kInf && label < n; };
  const auto cost_at = [&](int label) { return mine[min(label, n - 1)]; };
  const auto place = [&](int label) { return (label >> 2 >> kShift) * 4 + (label & 3); };
  const auto is_mine = [&](int label) { return W == 1 || ((label >> 2) & (W - 1)) == w; };
  float least = kInf;
  uint32_t named = 0;
  for (int e = 0; e < p.k; ++e) {
    const int label = p.labels[entry + e * step];
    const float t = kept_cost(p, entry + e * step);
    const bool is = exists(label, t);
    if (is && is_mine(label)) named |= 1u << place(label);
    least = is && cost_at(label) != kInf && t < least ? t : least;
  }
  const auto is_named = [&](int i, int j) { return (named >> (4 * i + j) & 1) != 0; };
  Mass others = {kInf, 0.f};
  float rest = kInf;
  if (p.rest != nullptr) {
    others = join<W>(mass_of(is_named), part[1], w, lane, p.to_exponent);
    rest = others.sum == 0.f ? kInf : p.rest[pixel];
    least = rest < least ? rest : least;
  }
  // the sum of the classes' weights, and of weight * (log p - log q) but for the logarithms of the sums
  float sum = 0, far = 0;
  for (int e = 0; e < p.k; ++e) {
    const int label = p.labels[entry + e * step];
    const float t = kept_cost(p, entry + e * step), own = cost_at(label);
    const float a = exists(label, t) && own != kInf ? weight(least, t, p.to_exponent) : 0.f;
    sum += a;
    if (!GRAD) far += a > 0 ? a * ((own - student.least) - (t - least)) : 0.f;
  }
  const float rest_weight = weight(least, rest, p.to_exponent);
  sum += rest_weight;
  if (!GRAD) {
    far *= p.inv_t;
    if (rest_weight > 0)
      far += rest_weight * (((others.least - student.least) - (rest - least)) * p.inv_t - logf(others.sum));
    const float loss = far / sum + (logf(student.sum) - logf(sum));
    if (w == 0 && lane < count) p.loss[pixel] = sum == 0.f ? 0.f : loss;
  } else {
    // p of the list's labels: each wavefront adds up its own, entry by entry
    const float per_sum = 1.f / sum;
    if (W > 1) tile_sync<W>();  // (the costs in LDS are done with)
    const float none[I][4] = {};
    to_tile<W, I>(mine, w, none);
    for (int e = 0; e < p.k; ++e) {
      const int label = p.labels[entry + e * step];
      const float t = kept_cost(p, entry + e * step);
      if (exists(label, t) && is_mine(label)) mine[label] += weight(least, t, p.to_exponent) * per_sum;
    }
    float d[I][4];
    from_tile<W, I>(mine, w, d);
    const float scale = p.dloss[pixel] * p.inv_t, per_student = 1.f / student.sum;
    const float share = rest_weight > 0 ? rest_weight * per_sum / others.sum : 0.f;
    const float nan = sum - sum;  // 0, or NaN where the teacher has one
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float q = weight(student.least, c[i][j], p.to_exponent) * per_student;
        const float r = share > 0 && !is_named(i, j) ? share * weight(others.least, c[i][j], p.to_exponent) : 0.f;
        d[i][j] = c[i][j] == kInf || sum == 0.f ? 0.f : ((d[i][j] + r) - q + nan) * scale;
      }
    if (FIRST) {
      if (lane < count) store_rows<W, I>((T*)p.dcost + first + p0, p.t, w, lane, d);
    } else {
      to_tile<W, I>(mine, w, d);
      tile_sync<W>();
      store_run<W, I>((T*)p.dcost + run, total, p.quads, tid, p.t, tile);
    }
  }
}

template <typename T, bool FIRST, bool GRAD>
void launch(const Distill& p, hipStream_t st) {
  with_shape(p.t.labels, [&](auto s) {
    constexpr int W = s.kW, I = s.kI, G = s.kG;
    distill_kernel<T, FIRST, GRAD, W, I, G><<<(p.t.total + G - 1) / G, 64 * W * G, 0, st>>>(p);
  });
}
template <bool GRAD>
int run(const char* what, int dtype, int labels_first, Distill& p, int kept_dtype, int k, float temperature, int items, int n_disp,
        int64_t pixels, hipStream_t st) {
  if (dtype < 0 || dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d", what, dtype);
  if (kept_dtype < 0 || kept_dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d of the list", what, kept_dtype);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "%s: n_disp must be in [1, %d], got %d", what, kMaxL, n_disp);
  if (k < 1 || k > kMaxL) return fail(MPL_EINVAL, "%s: the list must have 1 to %d entries, got %d", what, kMaxL, k);
  if (!(temperature > 0 && temperature < kInf && 1.f / temperature < kInf))
    return fail(MPL_EINVAL, "%s: the temperature must be finite and above 0", what);
  if (items < 0 || pixels < 0) return fail(MPL_EINVAL, "%s: negative size", what);
  if (items == 0 || pixels == 0) return MPL_OK;
  if (p.cost == nullptr || p.labels == nullptr || p.costs == nullptr ||
      (GRAD ? p.dloss == nullptr || p.dcost == nullptr : p.loss == nullptr))
    return fail(MPL_EINVAL, "%s: null pointer", what);
  if (!make_tiles(p.t, items, n_disp, pixels)) return fail(MPL_EINVAL, "%s: too many pixels", what);
  p.k = k;
  p.kept = kept_dtype;
  p.to_exponent = (float)(1.4426950408889634 / (double)temperature);
  p.inv_t = 1.f / temperature;
  const uintptr_t aligned = dtype == MPL_F32 ? 15 : 7;
  p.quads = n_disp % 4 == 0 && (((uintptr_t)p.cost | (uintptr_t)p.dcost) & aligned) == 0;
  const auto by_type = [&](auto type) {
    using T = decltype(type);
    labels_first != 0 ? launch<T, true, GRAD>(p, st) : launch<T, false, GRAD>(p, st);
  };
  if (dtype == MPL_F32)
    by_type(float());
  else if (dtype == MPL_F16)
    by_type((_Float16)0);
  else
    by_type((__bf16)0);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int mpl_distill_costs(int dtype, int labels_first, const void* cost, int kept_dtype, const uint8_t* kept_labels,
                      const void* kept_costs, const float* rest, float temperature, float* loss, int items, int n_disp, int n_kept,
                      int64_t pixels, void* stream) {
  Distill p = {};
  p.cost = cost;
  p.labels = kept_labels;
  p.costs = kept_costs;
  p.rest = rest;
  p.loss = loss;
  return run<false>("distill_costs", dtype, labels_first, p, kept_dtype, n_kept, temperature, items, n_disp, pixels,
                    (hipStream_t)stream);
}

int mpl_distill_costs_grad(int dtype, int labels_first, const void* cost, int kept_dtype, const uint8_t* kept_labels,
                           const void* kept_costs, const float* rest, float temperature, const float* dloss, void* dcost,
                           int items, int n_disp, int n_kept, int64_t pixels, void* stream) {
  Distill p = {};
  p.cost = cost;
  p.labels = kept_labels;
  p.costs = kept_costs;
  p.rest = rest;
  p.dloss = dloss;
  p.dcost = dcost;
  return run<true>("distill_costs_grad", dtype, labels_first, p, kept_dtype, n_kept, temperature, items, n_disp, pixels,
                   (hipStream_t)stream);
}

}  // extern "C"
