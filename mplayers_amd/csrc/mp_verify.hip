// Labels drafted from other costs, kept or drawn anew so that they are distributed as a layer's costs say, for gfx950.
//
// p = softmax(-cost / T) and q = softmax(-draft_cost / T') over a pixel's labels (q: 1 at the drafted label where no costs of the
// draft are given).  The label d stays where u0 q[d] < p[d], so with probability min(1, p[d] / q[d]); else one is drawn with u1 from
// what the draft leaves, max(p - q, 0): the first whose running sum, in label order, exceeds u1 * (sum of all).  A label drawn from
// q then is one of p, and is the drafted one as often as any way of drawing it can have it.  Where q[d] is 0 or there is no
// label d nothing was drafted, and one is drawn from p.
//
// Either volume is read once: a pixel's labels lie in the registers of one to eight lanes (mp_lanes.h), p and q are formed there, and
// the running sums go to LDS only in wavefronts where a label is drawn anew.  Results are those of 64 bits, which 32 bits give but
// for drafts next to a border (see verify_kernel).  Bound by HBM for one draft: us, 192 labels 1500x2000 1015 to 1075 (4.3 to 4.6 TB/s; with 64
// bits throughout 15 300, without the drafts that do go there 945), 60 labels 1000x2000 184 to 192 (5.3 TB/s); 60 labels 375x450 in the
// operators' layout, 8 drafts, 32 by the instructions (910 to a wavefront of 16 pixels, half of the time) and the last wavefronts,
// which have the drafts that go to 64 bits: 28 without those.  Without the draft's costs 192 labels 1500x2000 528 to 562 (4.1 to 4.4
// TB/s), 60 labels 375x450, 8 drafts, 24.

#include "mp_lanes.h"

using namespace mpl;

namespace {

struct Verify {
  LaneTiles t;
  const float* cost;
  const float* draft_cost;  // or nullptr
  const uint8_t* draft;
  const float* uniforms;    // items_pixels * n_drafts for keeping, then as many for drawing
  uint8_t* labels;
  uint8_t* kept;
  const float* temperature;  // one per image, or nullptr for the number below
  const float* draft_temperature;
  float temperature_all, draft_temperature_all;
  int64_t items_pixels;
  int n_cv, n_drafts;
  int mode;  // of runs of both volumes
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

// One pixel by a wavefront: cost(l) and draft_cost(l) give its costs, at is its place in the drafts, of which those k whose bit
// k % 32 is set are asked for.
template <bool COSTS, typename Cost, typename DraftCost>
__device__ void verify_exactly(const Verify& p, int image, int64_t at, uint32_t asked, Cost cost, DraftCost draft_cost) {
  const int lane = (int)(threadIdx.x & 63);
  const int64_t drafts = p.items_pixels * p.n_drafts;
  // a draft to a lane, for the next 64
  int d_of_lane = 0;
  float u0_of_lane = 0, u1_of_lane = 0;
  const auto fetch = [&](int k) {
    const int64_t mine = min(k + lane, p.n_drafts - 1) * p.items_pixels + at;
    d_of_lane = p.draft[mine];
    u0_of_lane = p.uniforms[mine];
    u1_of_lane = p.uniforms[drafts + mine];
  };
  fetch(0);
  // (all that comes from memory is on its way before the first of it is waited for)
  float v[4], y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = cost(min(4 * lane + j, p.t.n - 1));
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = COSTS ? draft_cost(min(4 * lane + j, p.t.n - 1)) : 0.f;
  double a[4], b[4] = {}, left[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = 4 * lane + j < p.t.n ? candidate(v[j]) : kInf;
  weights64(v, p.temperature != nullptr ? p.temperature[image] : p.temperature_all, a);
  const double total = total64(a), total_or_1 = total > 0 ? total : 1.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] /= total_or_1;
  const Running all = running64(a);
  Running rest = all;
  if (COSTS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = 4 * lane + j < p.t.n ? candidate(y[j]) : kInf;
    weights64(y, p.draft_temperature != nullptr ? p.draft_temperature[image] : p.draft_temperature_all, b);
    const double of_draft = total64(b), of_draft_or_1 = of_draft > 0 ? of_draft : 1.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] /= of_draft_or_1;
      left[j] = a[j] > b[j] ? a[j] - b[j] : 0.0;
    }
    rest = running64(left);
  }
  for (int k = 0; k < p.n_drafts; ++k) {
    if (k > 0 && k % 64 == 0) fetch(k);
    if ((asked >> (k % 32) & 1) == 0) continue;
    const int64_t place = k * p.items_pixels + at;
    const int d = from_lane(d_of_lane, k % 64);
    const float u0 = from_lane(u0_of_lane, k % 64), u1 = from_lane(u1_of_lane, k % 64);
    const bool exists = d < p.t.n;
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

// A temperature as 32 bits use it.
struct Scale {
  float to_exponent;      // log2(e) / T
  bool cold, flat, far;  // T not above 0; infinite; beyond what fp32 exponents are sure of
};
__device__ __forceinline__ Scale scale_of(const float* each, float all, int image) {
  const float t = each != nullptr ? each[image] : all;
  Scale s;
  s.cold = !positive(t);
  s.flat = t == kInf;
  s.far = !s.cold && !s.flat && !(t > 1e-30f && t < 1e30f);
  s.to_exponent = s.cold || s.flat ? 0.f : (float)(inverse(t) * 1.4426950408889634);
  return s;
}

// The sum of a lane's numbers, fours first: of NV / 4 + 1 additions on the way of any of them.
template <int NV>
__device__ __forceinline__ float tree_sum(const float (&v)[NV]) {
  float sum = 0;
#pragma unroll
  for (int j = 0; j < NV; j += 4) {
    const float four = (v[j] + v[j + 1]) + (v[j + 2] + v[j + 3]);
    sum = j == 0 ? four : sum + four;
  }
  return sum;
}

// The weights of a pixel's labels in its S lanes, in place of the costs.
struct Weights {
  float best, total;  // the least cost, +inf where there is no candidate
  int first;          // cold: the first label that has it, the only one that weighs
};
template <int NV, int S>
__device__ __forceinline__ Weights weights32(float (&v)[NV], const Scale& scale, int s) {
  Weights w = {v[0], 0.f, S * NV};
#pragma unroll
  for (int j = 1; j < NV; ++j) w.best = v[j] < w.best ? v[j] : w.best;
  w.best = lanes_min<S>(w.best);
  if (scale.cold) {
#pragma unroll
    for (int j = NV - 1; j >= 0; --j) w.first = v[j] == w.best && w.best < kInf ? s * NV + j : w.first;
    w.first = lanes_min<S>(w.first);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = s * NV + j == w.first ? 1.f : 0.f;
    w.total = 1.f;
    return w;
  }
  if (scale.flat) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = v[j] < kInf ? 1.f : 0.f;
    w.total = lanes_sum<S>(tree_sum(v));
    return w;
  }
  const float best = w.best < kInf ? w.best : 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = __builtin_amdgcn_exp2f((best - v[j]) * scale.to_exponent);  // (0 of +inf)
  w.total = lanes_sum<S>(tree_sum(v));
  return w;
}

// S lanes per pixel, NV labels per lane.  The weights stay as they are, those of the draft are brought to the target's scale: p is
// a[l] / A and q is b[l] / B, so b[l] * (A / B) stands beside a[l].  They are formed in 32 bits, with a bound on how far they
// may be off, all relative to A and u = 2^-24:
//   weights   3 roundings of an exponent x (3 u x w, and sum(x w) <= ln(n) sum(w): the entropy of n labels) and an ulp of the
//             exponential: (2 + 3 ln 256) u < 19 u of their sum
//   b A / B   those, of A and B as much and their own additions, H u each with H = NV / 4 + 4 + S, a quotient and a product:
//             (59 + 2 H) u over all labels
//   a running sum of max(a - b A / B, 0): both of these, a rounding each, the additions of what lies before the lane and of the
//             lane's fours to it: (79 + 2 H + NV / 2 + 3 + S) u
// and as much for a target, which is a product with such a sum.  Where a target is as close to a sum as both (kNear), 32 bits
// do not tell, and verify_exactly() takes the draft: with costs as a layer gives them and a draft of which a sixth is rejected one
// draft in 490 of 192 labels, in 1300 of 60, in 3700 of 21.  So it does where u0 q[d] is as close to p[d] as (3 x + 64 + 2 H) u of
// either, x being their exponents.
template <int NV, int S, bool COSTS, bool LAST>
__global__ void __launch_bounds__(kLanePixels* S) verify_kernel(Verify p) {
  using Tile = LaneTile<NV, S>;
  constexpr int kSteps = NV / 4 + 4 + S;
  constexpr float kU = 0x1p-24f, kNear = 2 * (80 + 2 * kSteps + NV / 2 + 3 + S) * kU;
  constexpr float kLeast = 1e-30f;  // below it fp32 is not what the bounds say
  __shared__ __align__(16) float tile[kLanePixels * Tile::kStride];
  __shared__ uint32_t left_over[2];           // pixels for verify_exactly(),
  __shared__ uint32_t asked[kLanePixels];     // and their drafts
  const unsigned block = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group), tiles = (unsigned)p.t.tiles;
  const int64_t item = block / tiles, p0 = (int64_t)(block - (unsigned)item * tiles) * kLanePixels;
  const int count = (int)min((int64_t)kLanePixels, p.t.pixels - p0), n = p.t.n;
  const int tid = (int)threadIdx.x, px = tid / S, s = tid % S, of = min(px, count - 1);
  const int64_t first = item * n * p.t.pixels, at = item * p.t.pixels + p0 + of, drafts = p.items_pixels * p.n_drafts;
  const int64_t pixel = first + (LAST ? (p0 + of) * n : p0 + of), step = LAST ? 1 : p.t.pixels;
  if (tid < 2) left_over[tid] = 0;
  if (s == 0) asked[px] = 0;
  // A draft to a lane: its label and uniform numbers, and the costs of that label.
  struct Drafted {
    int64_t place;
    int label;
    float u0, u1, cost, draft_cost;
  };
  const auto fetch_label = [&](int k) {
    Drafted d;
    d.place = min(k, p.n_drafts - 1) * p.items_pixels + at;
    d.label = p.draft[d.place];
    d.u0 = p.uniforms[d.place];
    d.u1 = p.uniforms[drafts + d.place];
    return d;
  };
  const auto fetch_costs = [&](Drafted& d) {
    const int64_t from = pixel + min(d.label, n - 1) * step;
    d.cost = p.cost[from];
    d.draft_cost = COSTS ? p.draft_cost[from] : 0.f;
  };
  Drafted d = fetch_label(s);
  float a[NV], b[NV];
  {
    LaneLoads<NV, S, LAST, float> target, draft;
    const int mode = LAST ? run_mode_of(p.mode, first, (unsigned)(count * n)) : (int)kEach;
    target.load(p.cost + first, p.t, p0, count, mode, tid);
    if (COSTS) draft.load(p.draft_cost + first, p.t, p0, count, mode, tid);
    fetch_costs(d);
    target.to_tile(tile, p.t, count, mode, tid);
    __syncthreads();
    from_lane_tile<NV, S>(tile, px, s, a);
    if (COSTS) {
      __syncthreads();
      draft.to_tile(tile, p.t, count, mode, tid);
      __syncthreads();
      from_lane_tile<NV, S>(tile, px, s, b);
    }
  }
  const int image = (int)((unsigned)item / (unsigned)p.n_cv);
  const Scale scale = scale_of(p.temperature, p.temperature_all, image),
              draft_scale = COSTS ? scale_of(p.draft_temperature, p.draft_temperature_all, image) : scale;
  const Weights wa = weights32<NV, S>(a, scale, s), wb = COSTS ? weights32<NV, S>(b, draft_scale, s) : wa;
  const bool empty = wa.best == kInf;
  // (no draft of the pixel can be told)
  const bool blind = !(wa.best > -kInf) || scale.far || (COSTS && wb.best < kInf && (!(wb.best > -kInf) || draft_scale.far));
  const float to_target = COSTS && wb.total > 0 ? wa.total / wb.total : 0.f;
  if (COSTS) {
    // what the draft leaves
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float rest = a[j] - b[j] * to_target;
      b[j] = rest > 0 ? rest : 0.f;
    }
  }

  // Running sums to LDS, and the last of them: the lanes of a pixel are of one wavefront, and nobody else reads its place any
  // more.
  float* const sums = &tile[px * Tile::kStride];
  const auto sum_up = [&](const float (&x)[NV]) {
    float sum = lanes_before<S>(tree_sum(x), s);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NV; j += 4) {
      const float two = x[j] + x[j + 1], three = two + x[j + 2], four = two + (x[j + 2] + x[j + 3]);
      const float4 q = {sum + x[j], sum + two, sum + three, sum + four};
      *reinterpret_cast<float4*>(sums + s * NV + j) = q;
      sum = q.w;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return lanes_max<S>(sum);
  };
  // The first label whose sum is above the target, by halving; `taken` of the sums from label `from` on does not count.
  const int top = 1 << (31 - __builtin_clz(n));
  const float too_near = kNear * wa.total;
  const auto find = [&](float target, int from, float taken, bool& near) {
    int label = 0;
    float least = -kInf;  // the last sum that is not above the target
    for (int step = top; step > 0; step >>= 1) {
      const int to = label + step;
      const float sum = sums[min(to, n) - 1] - (to > from ? taken : 0.f);
      if (to <= n && sum <= target) {
        label = to;
        least = sum;
      }
    }
    const float most = sums[min(label, n - 1)] - (label >= from ? taken : 0.f);
    near = !(least <= target - too_near && most > target + too_near) || label >= n;
    return label;
  };
  bool unsure = false;
  bool ready = false;  // whether the sums in LDS are those that labels are drawn from
  float left = 0;
  for (int base = 0; base < p.n_drafts; base += S) {
    if (base > 0) {
      d = fetch_label(base + s);
      fetch_costs(d);
    }
    const bool mine = base + s < p.n_drafts && px < count;
    const bool exists = d.label < n;
    const float c = candidate(d.cost), dc = candidate(d.draft_cost);
    const bool has_p = exists && (scale.cold ? d.label == wa.first : c < kInf);
    const bool has_q = exists && (!COSTS || (draft_scale.cold ? d.label == wb.first : dc < kInf));
    const float far_a = scale.cold || scale.flat || !has_p ? 0.f : (wa.best - c) * scale.to_exponent;
    const float far_b = !COSTS || draft_scale.cold || draft_scale.flat || !has_q ? 0.f : (wb.best - dc) * draft_scale.to_exponent;
    const float p_d = has_p ? __builtin_amdgcn_exp2f(far_a) : 0.f;
    const float q_d = !has_q ? 0.f : COSTS ? __builtin_amdgcn_exp2f(far_b) * to_target : wa.total;
    const float u0 = positive(d.u0) ? (d.u0 < 1.f ? d.u0 : 1.f) : 0.f, u1 = positive(d.u1) ? (d.u1 < 2.f ? d.u1 : 2.f) : 0.f;
    const float least = u0 * q_d, off = (64 + 2 * kSteps - 3 * (far_a < far_b ? far_a : far_b)) * kU;
    const bool kept = has_q && least < p_d;
    bool near = has_q && (q_d < kLeast || fabsf(least - p_d) <= off * (least + p_d) + kLeast || (positive(d.u0) && d.u0 > 1.f));
    int label = d.label;
    // what the draft leaves, or all of p
    const bool draws = mine && !empty && !kept && !near && !blind;
    const bool draws_left = draws && (has_q || !COSTS), draws_all = draws && !has_q && COSTS;
    if (__builtin_amdgcn_ballot_w64(draws_left) != 0) {
      if (!ready) left = sum_up(COSTS ? b : a);
      ready = true;
      const float taken = !COSTS && exists ? p_d : 0.f;
      bool close;
      const int drawn = find(u1 * (left - taken), d.label, taken, close);
      label = draws_left ? drawn : label;
      near |= draws_left && close;
    }
    if (COSTS && __builtin_amdgcn_ballot_w64(draws_all) != 0) {
      const float all = sum_up(a);
      ready = false;
      bool close;
      const int drawn = find(u1 * all, 0, 0.f, close);
      label = draws_all ? drawn : label;
      near |= draws_all && close;
    }
    if (mine && !empty && (near || blind)) {
      atomicOr(&asked[px], 1u << ((base + s) % 32));
      unsure = true;
    } else if (mine) {
      p.labels[d.place] = (uint8_t)(empty ? 0 : label);
      p.kept[d.place] = kept && !empty ? 1 : 0;
    }
  }
  unsure = lanes_max<S>(unsure ? 1 : 0) != 0;
  const auto exactly = [&](int of) {
    const int64_t from = first + (LAST ? (p0 + of) * n : p0 + of);
    verify_exactly<COSTS>(
        p, image, item * p.t.pixels + p0 + of, (uint32_t)uniform_i((int)asked[of]), [&](int l) { return p.cost[from + l * step]; },
        [&](int l) { return p.draft_cost[from + l * step]; });
  };
  if (S == 1) {
    // (one wavefront)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (uint64_t rest = __builtin_amdgcn_ballot_w64(unsure); rest != 0; rest &= rest - 1) exactly(__builtin_ctzll(rest));
  } else {
    if (unsure && s == 0) atomicOr(&left_over[px >> 5], 1u << (px & 31));
    __syncthreads();
    int turn = 0;
    for (uint64_t rest = (uint64_t)left_over[1] << 32 | left_over[0]; rest != 0; rest &= rest - 1)
      if (turn++ % S == uniform_i(tid / 64)) exactly(__builtin_ctzll(rest));
  }
}

// Labels per lane and lanes per pixel.  us, one draft but where said, fewer lanes / this / more: 60 labels 375x450 26.2 / 23.1 /
// 29.5, 8 drafts 41.9 / 32.6 / 39.0, 60 labels 1000x2000 185 / 184 / 288; 96 labels 384x1248 101 / 79 / 90.  Where a quarter or a
// sixth of the lanes' labels would be none: 72 labels 500x1000 78 -> 72, 104 98 -> 91, 150 164 -> 151, 220 225 -> 200.
// Up to 48 labels a single draft has a lane or two to a pixel, and several have as many more as go over them at a time.  us, more /
// fewer lanes, 40 M costs, labels first and last: one draft, 10 labels 120 / 78 and 148 / 79, 14 labels 98 / 77 and 101 / 73, 18: 89 /
// 73 and 107 / 70, 21: 79 / 74 and 93 / 75, 26: 73 / 71 and 91 / 69, 38 (four lanes or two) 83 / 72 and 100 / 80, 46: 74 / 71 and 68 /
// 63; eight drafts, 14 labels 1000x2000 144 / 178, 21 labels 1000x1000 87 / 106, 46 labels 1000x800 110 / 121, two drafts 44 / 51 for
// 21 labels and 70 / 68 for 46.
template <bool COSTS, bool LAST>
void launch(const Verify& p, unsigned blocks, hipStream_t st) {
  const int n = p.t.n;
  const bool one = p.n_drafts == 1;
  if (n <= 4)
    verify_kernel<4, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 8)
    verify_kernel<8, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 12)
    verify_kernel<12, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 16 && one)
    verify_kernel<16, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 16)
    verify_kernel<8, 2, COSTS, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 20 && one)
    verify_kernel<20, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 24 && one)
    verify_kernel<24, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 24)
    verify_kernel<12, 2, COSTS, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 28 && one)
    verify_kernel<28, 1, COSTS, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 32)
    verify_kernel<16, 2, COSTS, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 40 && one)
    verify_kernel<20, 2, COSTS, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 48 && one)
    verify_kernel<24, 2, COSTS, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 48)
    verify_kernel<12, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 64)
    verify_kernel<16, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 80)
    verify_kernel<20, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 96)
    verify_kernel<24, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 112)
    verify_kernel<28, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 128)
    verify_kernel<32, 4, COSTS, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 160)
    verify_kernel<20, 8, COSTS, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else if (n <= 192)
    verify_kernel<24, 8, COSTS, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else if (n <= 224)
    verify_kernel<28, 8, COSTS, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else
    verify_kernel<32, 8, COSTS, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
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
  Verify p;
  if (!make_lane_tiles(p.t, (int64_t)batch * n_cv, n_disp, pixels, labels_first != 0, 4))
    return fail(MPL_EINVAL, "verify_labels: too many pixels");
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
  p.items_pixels = (int64_t)batch * n_cv * pixels;
  p.n_cv = n_cv;
  p.n_drafts = n_drafts;
  p.mode = run_mode(n_disp, (((uintptr_t)cost | (uintptr_t)draft_cost) & 15) == 0);
  const unsigned blocks = (unsigned)(p.t.tiles * batch * n_cv);
  const hipStream_t st = (hipStream_t)stream;
  if (draft_cost != nullptr)
    labels_first ? launch<true, false>(p, blocks, st) : launch<true, true>(p, blocks, st);
  else
    labels_first ? launch<false, false>(p, blocks, st) : launch<false, true>(p, blocks, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "verify_labels: %s", hipGetErrorString(e));
}
