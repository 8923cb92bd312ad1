// Labels drafted from other costs, kept or drawn anew so that they are distributed as a layer's costs say, for gfx950.
//
// p = softmax(-cost / T) and q = softmax(-draft_cost / T') over a pixel's labels (q: 1 at the drafted label where no costs of the
// draft are given).  The label d stays where u0 q[d] < p[d], so with probability min(1, p[d] / q[d]); else one is drawn with u1 from
// what the draft leaves, max(p - q, 0): the first whose running sum, in label order, exceeds u1 * (sum of all).  A label drawn from
// q then is one of p, and is the drafted one as often as any way of drawing it can have it.  Where q[d] is 0 or there is no
// label d nothing was drafted, and one is drawn from p.

#include "mp_lanes.h"

using namespace mpl;

namespace {

struct Verify {
  const float* cost;
  const float* draft_cost;  // or nullptr
  const uint8_t* draft;
  const float* uniforms;    // items_pixels * n_drafts for keeping, then as many for drawing
  uint8_t* labels;
  uint8_t* kept;
  const float* temperature;  // one per image, or nullptr for the number below
  const float* draft_temperature;
  float temperature_all, draft_temperature_all;
  int64_t pixels, items_pixels;
  int n, n_cv, n_drafts, labels_first;
};

__device__ __forceinline__ double inverse(float temperature) { return positive(temperature) ? 1.0 / (double)temperature : 0.0; }

// Of one pixel by a wavefront, four labels to a lane, in 64 bits: the weights of softmax(-c / T), the best one's 1, 0 where there
// is no candidate.  T that is not above 0 leaves the first of the best labels.
__device__ __forceinline__ void weights64(const float (&v)[4], float temperature, double (&w)[4]) {
  float best = kInf;
#pragma unroll
  for (int j = 0; j < 4; ++j) best = v[j] < best ? v[j] : best;
  best = lanes_min<64>(best);
  const double to_exponent = inverse(temperature) * 1.4426950408889634;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double e = exp2_64(((double)best - (double)v[j]) * to_exponent);
    w[j] = !(v[j] < kInf) ? 0.0 : v[j] == best ? 1.0 : best == -kInf ? 0.0 : e;
  }
  if (!positive(temperature)) {
    int first = 256;
#pragma unroll
    for (int j = 3; j >= 0; --j) first = v[j] == best && best < kInf ? 4 * (int)(threadIdx.x & 63) + j : first;
    first = lanes_min<64>(first);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = 4 * (int)(threadIdx.x & 63) + j == first ? 1.0 : 0.0;
  }
}
__device__ __forceinline__ double total64(const double (&w)[4]) { return lanes_sum<64>((w[0] + w[1]) + (w[2] + w[3])); }

// Running sums over the labels, and the last label that weighs.  Each lane adds up in an order of its own, so that a sum may
// fall by a rounding from one lane to the next, or rise over a lane whose labels weigh nothing: they are made to rise at lanes
// that weigh only.
struct Running {
  double before, total;
  int last;
};
__device__ __forceinline__ Running running64(const double (&w)[4]) {
  const double sum = ((w[0] + w[1]) + w[2]) + w[3];
  const double ragged = wave_upto(sum, [](double a, double b) { return a + b; });
  const double upto = wave_upto(sum > 0 ? ragged : 0.0, [](double a, double b) { return b > a ? b : a; });
  Running r;
  r.total = from_lane(upto, 63);
  r.before = move_or_0<0x138>(upto);
  r.last = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (w[j] > 0) r.last = 4 * (int)(threadIdx.x & 63) + j;
  r.last = lanes_max<64>(r.last);
  return r;
}
// The first label whose running sum exceeds u * total, or the last that weighs.
__device__ __forceinline__ int pick64(const double (&w)[4], const Running& r, float u) {
  const double target = positive(u) && u >= 1.f ? __builtin_huge_val() : (positive(u) ? (double)u : 0.0) * r.total;
  int label = r.last;
  bool found = false;
  double run = r.before;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    run += w[j];
    if (!found && w[j] > 0) {
      label = 4 * (int)(threadIdx.x & 63) + j;
      found = run > target;
    }
  }
  const uint64_t past = __builtin_amdgcn_ballot_w64(r.before > target) >> 1 | (uint64_t)(r.total > target) << 63;
  return past != 0 ? from_lane(label, __builtin_ctzll(past)) : r.last;
}
__device__ __forceinline__ double of_label(const double (&w)[4], int label) {
  const double x = (label & 3) == 0 ? w[0] : (label & 3) == 1 ? w[1] : (label & 3) == 2 ? w[2] : w[3];
  return from_lane(x, label >> 2);
}

// One pixel by a wavefront: cost(l) and draft_cost(l) give its costs, at is its place in the drafts.
template <bool COSTS, typename Cost, typename DraftCost>
__device__ void verify_exactly(const Verify& p, int image, int64_t at, Cost cost, DraftCost draft_cost) {
  const int lane = (int)(threadIdx.x & 63);
  float v[4];
  double a[4], b[4] = {}, left[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = 4 * lane + j < p.n ? candidate(cost(4 * lane + j)) : kInf;
  weights64(v, p.temperature != nullptr ? p.temperature[image] : p.temperature_all, a);
  const double total = total64(a), total_or_1 = total > 0 ? total : 1.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] /= total_or_1;
  const Running all = running64(a);
  Running rest = all;
  if (COSTS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 4 * lane + j < p.n ? candidate(draft_cost(4 * lane + j)) : kInf;
    weights64(v, p.draft_temperature != nullptr ? p.draft_temperature[image] : p.draft_temperature_all, b);
    const double of_draft = total64(b), of_draft_or_1 = of_draft > 0 ? of_draft : 1.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] /= of_draft_or_1;
      left[j] = a[j] > b[j] ? a[j] - b[j] : 0.0;
    }
    rest = running64(left);
  }
  const int64_t drafts = p.items_pixels * p.n_drafts;
  for (int k = 0; k < p.n_drafts; ++k) {
    const int64_t place = k * p.items_pixels + at;
    const int d = uniform_i(p.draft[place]);
    const float u0 = uniform_f(p.uniforms[place]), u1 = uniform_f(p.uniforms[drafts + place]);
    const bool exists = d < p.n;
    const double p_d = of_label(a, exists ? d : 0), q_d = !exists ? 0.0 : COSTS ? of_label(b, d) : 1.0;
    const bool stays = total > 0 && exists && q_d > 0 && (positive(u0) ? (double)u0 : 0.0) * q_d < p_d;
    int label = d;
    if (!stays) {
      if (!COSTS && exists) {
#pragma unroll
        for (int j = 0; j < 4; ++j) left[j] = 4 * lane + j == d ? 0.0 : a[j];
        rest = running64(left);
      }
      const bool drafted = exists && q_d > 0 && rest.total > 0;
      label = drafted ? pick64(left, rest, u1) : pick64(a, all, u1);
    }
    if (lane == 0) {
      p.labels[place] = (uint8_t)(total > 0 ? label : 0);
      p.kept[place] = stays ? 1 : 0;
    }
  }
}

template <bool COSTS>
__global__ void __launch_bounds__(256) verify_kernel(Verify p) {
  for (int64_t at = (int64_t)blockIdx.x * 4 + uniform_i((int)threadIdx.x / 64); at < p.items_pixels; at += (int64_t)gridDim.x * 4) {
    const int64_t item = at / p.pixels, pixel = at - item * p.pixels;
    const int64_t first = item * p.n * p.pixels + (p.labels_first ? pixel : pixel * p.n), step = p.labels_first ? p.pixels : 1;
    verify_exactly<COSTS>(
        p, (int)(item / p.n_cv), at, [&](int l) { return p.cost[first + l * step]; },
        [&](int l) { return p.draft_cost[first + l * step]; });
  }
}

}  // namespace

extern "C" int mpl_verify_labels(int labels_first, const float* cost, const uint8_t* draft, const float* draft_cost,
                                 const float* uniforms, int batch, int n_cv, int n_disp, int64_t pixels, int n_drafts,
                                 const float* temperatures, float temperature, const float* draft_temperatures,
                                 float draft_temperature, uint8_t* labels, uint8_t* kept, void* stream) {
  if (batch < 0 || n_cv < 0 || pixels < 0 || n_drafts < 0) return fail(MPL_EINVAL, "verify_labels: negative size");
  if (n_disp < 1 || n_disp > kMaxL)
    return fail(MPL_EINVAL, "verify_labels: n_disp must be in [1, %d], got %d", kMaxL, n_disp);
  if (batch == 0 || n_cv == 0 || pixels == 0 || n_drafts == 0) return MPL_OK;
  if (cost == nullptr || draft == nullptr || uniforms == nullptr || labels == nullptr || kept == nullptr)
    return fail(MPL_EINVAL, "verify_labels: null pointer");
  LaneTiles t;
  if (!make_lane_tiles(t, (int64_t)batch * n_cv, n_disp, pixels)) return fail(MPL_EINVAL, "verify_labels: too many pixels");
  Verify p;
  p.cost = cost;
  p.draft_cost = draft_cost;
  p.draft = draft;
  p.uniforms = uniforms;
  p.labels = labels;
  p.kept = kept;
  p.temperature = temperatures;
  p.draft_temperature = draft_temperatures;
  p.temperature_all = temperature;
  p.draft_temperature_all = draft_temperature;
  p.pixels = pixels;
  p.items_pixels = (int64_t)batch * n_cv * pixels;
  p.n = n_disp;
  p.n_cv = n_cv;
  p.n_drafts = n_drafts;
  p.labels_first = labels_first != 0;
  const unsigned blocks = (unsigned)(p.items_pixels < (4 << 16) ? (p.items_pixels + 3) / 4 : 1 << 16);
  if (draft_cost != nullptr)
    verify_kernel<true><<<blocks, 256, 0, (hipStream_t)stream>>>(p);
  else
    verify_kernel<false><<<blocks, 256, 0, (hipStream_t)stream>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "verify_labels: %s", hipGetErrorString(e));
}
