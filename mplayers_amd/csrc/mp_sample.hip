// Labels drawn from the layers' costs, for gfx950.
//
// A pixel's costs c[l] are energies: label l has weight w[l] = exp((best - c[l]) / T).  Of the labels that top_k,
// top_p and min_p leave, in label order, the first one whose running sum exceeds u * (sum of all) is drawn, u given
// by the caller.  Costs of +inf and NaN are no candidates, T <= 0 is top_k = 1, equal costs order by label.
//
// All three filters keep the best labels down to a threshold (a cost, and how many of the labels that have exactly
// that cost): top_k the cost of the k-th best, top_p the least cost whose labels down to it weigh enough, min_p
// best + T * ln(1 / min_p).  So no sort: the threshold is found by halving the range of costs and then going from one
// cost that occurs to the next (find).
//
// The costs are read once: a tile of 64 pixels lies in registers, a pixel's labels over one to eight lanes beside each
// other.  (Tiles in the operators' layout, and of more than one lane to a pixel, get there through LDS, which turns rows of
// labels into labels of a pixel.)  Without filters that bounds the call: 192 labels 1500x2000 0.45 ms, 5.1 TB/s, where a
// large copy moves 4.7.  The filters are bound by the instructions they issue: 96 labels 384x1248 with all three and 4 draws
// 131 us, 2650 vector instructions to a wavefront of 16 pixels, which issue 97 % of the time.
//
// Which label is drawn must not depend on how the sums are formed, or two correct programs would disagree on the
// pixels whose target falls next to a border.  So the borders are those of sums in 64 bits, which are off by 2^-50 or
// so, and 32 bits, which take a third of the time, only where they tell (see sample_kernel): with 64 bits throughout 192
// labels 1500x2000 took 1.42 ms.

#include "mp_lanes.h"

using namespace mpl;

namespace {

constexpr int kPixels = 64;  // pixels of a workgroup
// Draws from which on each has a lane of its own that halves the running sums in LDS; below, all lanes of a pixel count the
// sums up to the target.  us, counting / halving: 1 draw: 60 labels 375x450 13.7 / 15.0, 192 labels 256x512 25.0 / 28.2; 2:
// 15.9 / 15.5, 29.1 / 30.1; 4: 19.7 / 16.5, 38.4 / 33.2; 16: 39.2 / 23.9, 77.3 / 42.0.
constexpr int kSearchFrom = 2;
constexpr unsigned kFewTiles = 4096;  // see mpl_sample_labels
constexpr int kFewDraws = 4;          // one after the other in draw_exactly, more a lane each

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
  double inv_t_all, reach_all;  // 1 / T; of min_p, where temperature and min_p are numbers
  int64_t pixels, tiles, items_pixels;
  int n, n_cv, n_draws;
  uint32_t reciprocal;  // 2^32 / n, rounded up
  int quads;            // labels last: whole and aligned quads
  int xcd_group;        // tiles beside each other that go to one die (xcd_block)
};

// Closes the range lo <= t <= hi of the least cost t with sum(of labels with cost <= t) >= target; hi where no sum
// reaches it.  sum_upto(mid, below, above) gives the sum, the greatest cost that is not above mid and the least that
// is; reached(sum) decides, or sets `unsure`, which ends the search where it is.  lo is a cost that occurs, or one
// that t is above.
template <int S, typename SumUpTo, typename Reached>
__device__ __forceinline__ void threshold(float& lo, float& hi, const bool& unsure, SumUpTo sum_upto, Reached reached) {
#pragma unroll 1
  for (int step = 0; __builtin_amdgcn_ballot_w64(lo < hi && !unsure) != 0; ++step) {
    // Halves the costs, and after a while what lies between their bit patterns: costs that grow from one to the next
    // by factors would lose one a step.
    float mid = 0.5f * lo + 0.5f * hi;
    if (step >= 10) {
      const int a = float_key(__builtin_bit_cast(int, lo)), b = float_key(__builtin_bit_cast(int, hi));
      mid = __builtin_bit_cast(float, float_key((int)(((int64_t)a + b) >> 1)));
    }
    if (!(mid >= lo && mid < hi)) mid = lo;
    float below = lo, above = hi;
    const auto sum = lanes_sum<S>(sum_upto(mid, below, above));
    below = lanes_max<S>(below);
    above = lanes_min<S>(above);
    if (lo < hi) {
      const bool down = reached(sum);
      if (!unsure) {
        if (down)
          hi = below;
        else
          lo = above;
      }
    }
  }
}

// The same for the costs v of a lane, in steps of a third and half the instructions: a few that only halve the range,
// then from its lower end up from one cost to the next.  What that leaves open, costs close together in a wide range,
// threshold() closes.  On return t is the cost, `at` the number of labels at it, `less` the sum of those below.
//   labels        how many there are about: a halving for each time they can be halved leaves one or two
//   value(a)      what a label of cost a adds
//   sum_upto(c)   this lane's sum of the labels with cost <= c
constexpr int kSteps = 6;
template <int NV, int S, typename V, typename Value, typename SumUpTo, typename Reached>
__device__ __forceinline__ void find(const float (&v)[NV], int labels, float best, float worst, bool& unsure, Value value,
                                     SumUpTo sum_upto, Reached reached, float& t, int& at, V& less) {
  const int halves = 32 - __builtin_clz(labels | 7);
  // t > lo, and less is the sum up to lo
  float lo = best < kInf ? best - (fabsf(best) * 0x1p-20f + 0x1p-100f) : best, hi = worst;
  less = V(0);
#pragma unroll 1
  for (int step = 0; step < halves; ++step) {
    const float mid = 0.5f * lo + 0.5f * hi;
    const V sum = lanes_sum<S>(sum_upto(mid));
    if (mid > lo && mid < hi) {
      const bool down = reached(sum);
      hi = down && !unsure ? mid : hi;
      lo = down || unsure ? lo : mid;
      less = down || unsure ? less : sum;
    }
  }
  bool open = true;
  t = hi;
  at = 0;
#pragma unroll 1
  for (int step = 0; step < kSteps && __builtin_amdgcn_ballot_w64(open && !unsure) != 0; ++step) {
    float next = kInf;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float above = v[j] > lo ? v[j] : kInf;
      next = above < next ? above : next;
    }
    next = lanes_min<S>(next);
    int ties = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) ties += v[j] == next ? 1 : 0;
    ties = lanes_sum<S>(ties);
    if (open) {
      const V sum = less + (V)ties * value(next);
      if (!(next < kInf) || reached(sum)) {
        open = false;
        t = next;
        at = ties;
      } else {
        lo = next;
        less = sum;
      }
    }
  }
  if (__builtin_amdgcn_ballot_w64(open && !unsure) != 0) {
    if (!open) lo = hi = t;
    threshold<S>(
        lo, hi, unsure,
        [&](float mid, float& below, float& above) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const bool in = v[j] <= mid;
            const float b = in ? v[j] : below, a = in ? above : v[j];
            below = b > below ? b : below;
            above = a < above ? a : above;
          }
          return sum_upto(mid);
        },
        reached);
    int ties = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) ties += v[j] == hi ? 1 : 0;
    ties = lanes_sum<S>(ties);
    const V sum = lanes_sum<S>(sum_upto(hi));
    if (open) {
      t = hi;
      at = ties;
      less = sum - (V)ties * value(hi);
    }
  }
}

// What the parameters of an image come to.
struct Parameters {
  float temperature, top_p;
  int top_k;
  bool warm, bounded;  // T > 0; min_p > 0
  double inv_t, reach;  // 1 / T; T * ln(1 / min_p)
};
__host__ __device__ __forceinline__ double reach_of(float temperature, float min_p) {
  return min_p >= 1.f ? 0.0 : -(double)temperature * log((double)min_p);
}
template <bool FILTER>
__device__ __forceinline__ Parameters parameters(const Sample& p, int image) {
  Parameters q;
  q.temperature = p.temperature != nullptr ? p.temperature[image] : p.temperature_all;
  q.warm = positive(q.temperature);
  q.inv_t = p.temperature == nullptr ? p.inv_t_all : q.warm ? 1.0 / (double)q.temperature : 0.0;
  q.top_k = p.n;
  q.top_p = 1.f;
  q.bounded = false;
  q.reach = 0;
  if (FILTER) {
    const int k = p.top_k != nullptr ? p.top_k[image] : p.top_k_all;
    if (k > 0 && k < p.n) q.top_k = k;
    if (!q.warm) q.top_k = 1;
    if (q.warm) {
      q.top_p = p.top_p != nullptr ? p.top_p[image] : p.top_p_all;
      const float min_p = p.min_p != nullptr ? p.min_p[image] : p.min_p_all;
      q.bounded = positive(min_p);
      if (q.bounded) q.reach = p.min_p != nullptr || p.temperature != nullptr ? reach_of(q.temperature, min_p) : p.reach_all;
    }
  }
  return q;
}

// The greatest cost that min_p leaves: the greatest float whose distance from the best is at most T * ln(1 / min_p).
__device__ __forceinline__ float farthest(const Parameters& q, float best) {
  if (best == -kInf) return best;
  const auto within = [&](float c) { return (double)c - (double)best <= q.reach; };
  const float far = (float)((double)best + q.reach);
  if (!(far < kInf)) return kInf;
  const int key = float_key(__builtin_bit_cast(int, far));
  const float next = __builtin_bit_cast(float, float_key(key + 1)), previous = __builtin_bit_cast(float, float_key(key - 1));
  const float c = within(next) ? next : within(far) ? far : previous;
  return c < best ? best : c;
}

// One pixel by a whole wavefront, four labels to a lane, in 64 bits: cost(l) gives its costs, at is its place in the
// uniform numbers and the labels.
template <bool FILTER, typename Cost>
__device__ void draw_exactly(const Sample& p, const Parameters& q, int64_t at, Cost cost) {
  const int lane = (int)(threadIdx.x & 63);
  const float mine = lane < p.n_draws ? p.uniforms[lane * p.items_pixels + at] : 0.f;  // of draw `lane`
  float v[4], best = kInf;
  double w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int l = 4 * lane + j;
    v[j] = l < p.n ? candidate(cost(l)) : kInf;
    best = v[j] < best ? v[j] : best;
  }
  best = lanes_min<64>(best);
  const auto weight = [&](float c) {
    const double e = exp2_64(((double)best - (double)c) * (q.inv_t * 1.4426950408889634));
    return !(c < kInf) ? 0.0 : c == best ? 1.0 : best == -kInf ? 0.0 : e;
  };
  if (FILTER) {
    const auto worst = [&]() {
      float m = best;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = v[j] < kInf && v[j] > m ? v[j] : m;
      return lanes_max<64>(m);
    };
    // takes out what is worse than t, and of the labels at t those that do not stay by their rank
    const auto cut = [&](float t, auto stays) {
      int rank = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t ties = __builtin_amdgcn_ballot_w64(v[j] == t);
        rank += __builtin_amdgcn_mbcnt_hi((uint32_t)(ties >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ties, 0));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool tie = v[j] == t;
        if (v[j] > t || (tie && !stays(rank))) v[j] = kInf;
        rank += tie ? 1 : 0;
      }
    };
    constexpr bool unsure = false;
    const auto search = [&](auto target, auto add) {
      float lo = best, hi = worst();
      threshold<64>(
          lo, hi, unsure,
          [&](float mid, float& below, float& above) {
            auto sum = target;
            sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              below = v[j] <= mid && v[j] > below ? v[j] : below;
              above = v[j] > mid && v[j] < above ? v[j] : above;
              if (v[j] <= mid) sum += add(j);
            }
            return sum;
          },
          [&](auto sum) { return sum >= target; });
      return hi;
    };
    if (q.top_k < p.n) {
      const float t = search(q.top_k, [](int) { return 1; });
      int less = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) less += v[j] < t ? 1 : 0;
      less = lanes_sum<64>(less);
      cut(t, [&](int rank) { return less + rank < q.top_k; });
    }
    if (q.top_p < 1.f) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = weight(v[j]);
      const double target = (double)q.top_p * lanes_sum<64>((w[0] + w[1]) + (w[2] + w[3]));
      const float t = search(target, [&](int j) { return w[j]; });
      double less = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) less += v[j] < t ? w[j] : 0.0;
      less = lanes_sum<64>(less);
      const double each = weight(t);
      cut(t, [&](int rank) { return less + rank * each < target || (t == best && rank == 0); });
    }
    if (q.bounded) {
      const float far = farthest(q, best);
      cut(far, [](int) { return true; });
    }
  }
  double sum = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = weight(v[j]);
    sum += w[j];
  }
  // Each lane adds up in an order of its own, so that a sum may fall by a rounding from one lane to the next, or rise over
  // a lane whose labels weigh nothing, where a target may come to lie.  So they are made to rise at lanes that weigh only.
  const double ragged = wave_upto(sum, [](double a, double b) { return a + b; });
  const double upto = wave_upto(sum > 0 ? ragged : 0.0, [](double a, double b) { return b > a ? b : a; });
  const double total = from_lane(upto, 63), before = move_or_0<0x138>(upto);
  int last = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (w[j] > 0) last = 4 * lane + j;
  last = lanes_max<64>(last);
  // (a label's sum may pass the total by a rounding)
  const auto target_of = [&](float u) {
    return positive(u) && u >= 1.f ? __builtin_huge_val() : (positive(u) ? (double)u : 0.0) * total;
  };
  // of lane `who`, `run` before it and e its weights: the first label whose sum passes the target, or the last that weighs
  const auto within = [&](int who, double run, const double (&e)[4], double target) {
    int label = last;
    bool found = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      run += e[j];
      if (!found && e[j] > 0) {
        label = 4 * who + j;
        found = run > target;
      }
    }
    return label;
  };
  // The label is of the first lane whose sum, which is `before` of the next, passes the target; with many draws one to a
  // lane, which finds it by halving.
  if (p.n_draws <= kFewDraws) {
    for (int d = 0; d < p.n_draws; ++d) {
      const double target = target_of(from_lane(mine, d));
      const int label = within(lane, before, w, target);
      const uint64_t past = __builtin_amdgcn_ballot_w64(before > target) >> 1 | (uint64_t)(total > target) << 63;
      const int drawn = past != 0 ? from_lane(label, __builtin_ctzll(past)) : last;
      if (lane == 0) p.labels[d * p.items_pixels + at] = (uint8_t)drawn;
    }
    return;
  }
  for (int first = 0; first < p.n_draws; first += 64) {
    const int d = first + lane;
    const double target = target_of(first == 0 ? mine : d < p.n_draws ? p.uniforms[d * p.items_pixels + at] : 0.f);
    int who = 0;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1)
      if (__shfl(before, who + step) <= target) who += step;
    const double e[4] = {__shfl(w[0], who), __shfl(w[1], who), __shfl(w[2], who), __shfl(w[3], who)};
    const int label = within(who, __shfl(before, who), e, target);
    if (d < p.n_draws) p.labels[d * p.items_pixels + at] = (uint8_t)label;
  }
}

// S lanes per pixel, NV labels per lane: lane s owns labels s * NV ... s * NV + NV - 1.
//
// Weights and sums are formed in 32 bits, with a bound on how far they may be off, relative to the sum of all:
//   a weight  3 roundings of its exponent a (2^-24 * 3 * a * w, and sum(a * w) <= ln(n) * sum(w): the entropy of n labels),
//             1 ulp of the exponential: (2 + 3 * ln 256) * 2^-24 < 19 * 2^-24
//   a sum     NV - 1 additions in a lane, S over the lanes: (NV + S) * 2^-24
// and as much for a target, which is a product with such a sum (and is rounded itself).  Where a sum is as close to a
// target as both (kNear), 32 bits do not tell, and draw_exactly() takes the pixel: with costs as a layer gives them one
// draw in 400 of 192 labels, one in 4000 of 21.  (One wavefront for all pixels it had in registers took longer: its 64-bit
// weights cost every call the registers of a third of its wavefronts, and each of its pixels waited for one.)
template <int NV, int S, bool FILTER, bool LAST, bool SEARCH>
__global__ void __launch_bounds__(kPixels* S) sample_kernel(Sample p) {
  constexpr int kQuads = S * NV / 4, kJ = NV / 4;  // of four labels: in all, per lane
  constexpr int kStride = 4 * (kQuads | 1);
  constexpr bool kTile = S > 1 || LAST;  // costs through LDS
  constexpr float kNear = 2 * (NV + S + 25) * 0x1p-24f;
  __shared__ __align__(16) float tile[kTile || SEARCH ? kPixels * kStride : 4];
  __shared__ uint32_t left_over[2];  // pixels for draw_exactly()
  const unsigned block = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.xcd_group), tiles = (unsigned)p.tiles;
  const int64_t item = block / tiles, p0 = (int64_t)(block - (unsigned)item * tiles) * kPixels;
  const int count = (int)min((int64_t)kPixels, p.pixels - p0);
  const int tid = (int)threadIdx.x;
  const float* cost = p.cost + item * p.n * p.pixels;
  float v[NV];
  const int px = tid / S, s = tid % S;
  if (tid < 2) left_over[tid] = 0;
  // The quads of a pixel lie in the order in which its lanes read them: quad q, of lane q / kJ, at place q % kJ * S + q / kJ.
  const auto place = [](int q) { return (q % kJ * S + q / kJ) * 4; };
  // Rows of labels: the labels behind the last and the pixels behind the last are read from the last's place, so that
  // no branch lies between the loads.
  const auto row = [&](int l) { return cost + (int64_t)min(l, p.n - 1) * p.pixels + p0; };
  if (!kTile) {
    const int of = min(px, count - 1);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = row(j)[of];
  } else {
    if (LAST) {
      const unsigned n = (unsigned)p.n, total = (unsigned)count * n;
      const float* from = cost + p0 * p.n;
      if (p.quads) {
        float4 c[kJ];
#pragma unroll
        for (int k = 0; k < kJ; ++k)
          c[k] = *reinterpret_cast<const float4*>(from + min((unsigned)(tid + k * kPixels * S) * 4, total - 4));
#pragma unroll
        for (int k = 0; k < kJ; ++k) {
          const unsigned i = min((unsigned)(tid + k * kPixels * S) * 4, total - 4);
          const unsigned of = __umulhi(i, p.reciprocal), l = i - of * n;
          *reinterpret_cast<float4*>(&tile[of * kStride + place((int)(l >> 2))]) = c[k];
        }
      } else {
        float c[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) c[k] = from[min((unsigned)(tid + k * kPixels * S), total - 1)];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const unsigned i = min((unsigned)(tid + k * kPixels * S), total - 1);
          const unsigned of = n == 1 ? i : __umulhi(i, p.reciprocal), l = i - of * n;
          tile[of * kStride + place((int)(l >> 2)) + (l & 3)] = c[k];
        }
      }
    } else {
      const int of = min(tid % kPixels, count - 1), wave = uniform_i(tid / kPixels);
      float4 c[kJ];
#pragma unroll
      for (int i = 0; i < kJ; ++i) {
        const int l = 4 * (wave + i * S);
        c[i] = float4{row(l)[of], row(l + 1)[of], row(l + 2)[of], row(l + 3)[of]};
      }
#pragma unroll
      for (int i = 0; i < kJ; ++i)
        *reinterpret_cast<float4*>(&tile[tid % kPixels * kStride + place(wave + i * S)]) = c[i];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = tile[px * kStride + ((j >> 2) * S + s) * 4 + (j & 3)];
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = s * NV + j < p.n && px < count ? candidate(v[j]) : kInf;
  float best = v[0];
#pragma unroll
  for (int j = 1; j < NV; ++j) best = v[j] < best ? v[j] : best;
  best = lanes_min<S>(best);

  const Parameters q = parameters<FILTER>(p, (int)((unsigned)item / (unsigned)p.n_cv));
  const bool empty = best == kInf;
  // what the bound above needs: no overflow in the exponents; and find() a cost below the best
  bool unsure = !empty && (!(best > -kInf) || (q.warm && !(q.temperature > 1e-30f && q.temperature < 1e30f)));
  const float to_exponent = (float)(q.inv_t * 1.4426950408889634);
  const auto weight = [&](float c) {
    const float e = __builtin_amdgcn_exp2f((best - c) * to_exponent);
    return !FILTER || q.warm ? e : c < kInf ? 1.f : 0.f;
  };
  float w[NV];
  if (FILTER) {
    // takes out what is worse than t, and of the `at` labels at t those behind the first `ties`
    const auto cut = [&](float t, int at, int ties) {
      if (__builtin_amdgcn_ballot_w64(at > ties) == 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = v[j] > t ? kInf : v[j];
        return;
      }
      int mine = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) mine += v[j] == t ? 1 : 0;
      int rank = lanes_before<S>(mine, s);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const bool tie = v[j] == t;
        if (v[j] > t || (tie && rank >= ties)) v[j] = kInf;
        rank += tie ? 1 : 0;
      }
    };
    float worst = best;
    if (q.top_k < p.n || q.top_p < 1.f) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const float c = v[j] < kInf ? v[j] : best;
        worst = c > worst ? c : worst;
      }
      worst = lanes_max<S>(worst);
    }
    if (q.top_k < p.n) {
      bool whole = false;  // (whole numbers are never unsure)
      int at, less;
      float t;
      find<NV, S>(
          v, p.n, best, q.top_k == 1 ? best : worst, whole, [](float) { return 1; },
          [&](float mid) {
            int labels = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) labels += v[j] <= mid ? 1 : 0;
            return labels;
          },
          [&](int labels) { return labels >= q.top_k; }, t, at, less);
      cut(t, at, q.top_k - less);
      worst = t < worst ? t : worst;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) w[j] = weight(v[j]);
    float t = kInf;
    int at = 0, ties = 0;
    if (q.top_p < 1.f) {
      float total = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) total += w[j];
      total = lanes_sum<S>(total);
      const float target = q.top_p * total, near = kNear * total;
      // Labels further than T * ln(2 n / (1 - top_p)) from the best weigh less than half of what may go.
      const float rest = 1.f - q.top_p;
      const float reach = rest > 1e-3f ? q.temperature * __logf(2.f * (float)p.n / rest) : kInf;
      float less;
      find<NV, S>(
          v, q.top_k, best, best + reach < worst ? best + reach : worst, unsure, weight,
          [&](float mid) {
            float sum = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) sum += v[j] <= mid ? w[j] : 0.f;
            return sum;
          },
          [&](float sum) {
            unsure |= fabsf(sum - target) <= near;
            return sum >= target;
          },
          t, at, less);
      ties = at;
      if (__builtin_amdgcn_ballot_w64(at > 1) != 0) {
        const float each = weight(t), left = target - less;
        const float stay = ceilf(left / each);
        if (at > 1) {
          // the nearest of the sums that the ties give
          unsure |= fabsf(left - rintf(left / each) * each) <= 2 * near || !(stay < 512.f);
          ties = min(at, max(1, (int)stay));
        }
      }
    }
    if (q.bounded) {
      const float far = farthest(q, best);
      if (far < t) {
        t = far;
        at = 0;
        ties = p.n;  // all stay, also where another pixel has the wavefront cut
      }
    }
    if (q.top_p < 1.f || q.bounded) {
      if (__builtin_amdgcn_ballot_w64(at > ties) != 0) cut(t, at, ties);
#pragma unroll
      for (int j = 0; j < NV; ++j) w[j] = v[j] > t ? 0.f : w[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) w[j] = weight(v[j]);
  }

  float sum = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    sum += w[j];
    w[j] = sum;
  }
  const float before = lanes_before<S>(sum, s);
  const float total = lanes_max<S>(before + sum);  // (lanes_sum would add in another order)
  const float near = kNear * total;
  const int64_t at = item * p.pixels + p0;
  const int of = min(px, count - 1);
  if (SEARCH) {
    // Running sums to LDS (the lanes of a pixel are of one wavefront, and nobody else reads its costs any more), a draw
    // to a lane, and the first sum above the target by halving.
    float* sums = &tile[px * kStride];
#pragma unroll
    for (int j = 0; j < NV; j += 4)
      *reinterpret_cast<float4*>(sums + s * NV + j) =
          float4{before + w[j], before + w[j + 1], before + w[j + 2], before + w[j + 3]};
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int top = 1 << (31 - __builtin_clz(p.n));
    for (int d = s; d < p.n_draws; d += S) {
      const float u = p.uniforms[d * p.items_pixels + at + of];
      const float target = (positive(u) ? u : 0.f) * total;
      int label = 0;
      float least = -kInf;  // the last sum that is not above the target
      for (int step = top; step > 0; step >>= 1) {
        const int to = label + step;
        const float sum = sums[min(to, p.n) - 1];
        if (to <= p.n && sum <= target) {
          label = to;
          least = sum;
        }
      }
      const float most = sums[min(label, p.n - 1)];
      const bool near_one = !(least <= target - near && most > target + near) || label >= p.n;
      unsure |= near_one;
      if (px < count && (empty || !unsure)) p.labels[d * p.items_pixels + at + of] = (uint8_t)(empty ? 0 : label);
    }
    unsure = lanes_max<S>(unsure ? 1 : 0) != 0;
  } else {
    for (int d = 0; d < p.n_draws; ++d) {
      const float u = p.uniforms[d * p.items_pixels + at + of];
      const float target = (positive(u) ? u : 0.f) * total - before;
      const float low = target - near, high = target + near;
      int label = 0, most = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        label += w[j] <= low ? 1 : 0;
        most += w[j] <= high ? 1 : 0;
      }
      label = lanes_sum<S>(label);
      unsure |= label != lanes_sum<S>(most) || label >= p.n;
      if (s == 0 && px < count && (empty || !unsure)) p.labels[d * p.items_pixels + at + of] = (uint8_t)(empty ? 0 : label);
    }
  }

  unsure = unsure && !empty && px < count;
  const auto exactly = [&](int of) {
    if (kTile && !SEARCH) {
      draw_exactly<FILTER>(p, q, at + of, [&](int l) { return tile[of * kStride + place(l >> 2) + (l & 3)]; });
    } else {  // (the tile has the running sums)
      const float* c = cost + (LAST ? (p0 + of) * p.n : p0 + of);
      const int64_t step = LAST ? 1 : p.pixels;
      draw_exactly<FILTER>(p, q, at + of, [&](int l) { return c[l * step]; });
    }
  };
  if (S == 1) {
    // (one wavefront)
    for (uint64_t rest = __builtin_amdgcn_ballot_w64(unsure); rest != 0; rest &= rest - 1) exactly(__builtin_ctzll(rest));
  } else {
    if (unsure && s == 0) atomicOr(&left_over[px >> 5], 1u << (px & 31));
    __syncthreads();
    int turn = 0;
    for (uint64_t rest = (uint64_t)left_over[1] << 32 | left_over[0]; rest != 0; rest &= rest - 1)
      if (turn++ % S == uniform_i(tid / 64)) exactly(__builtin_ctzll(rest));
  }
}

template <int NV, int S, bool FILTER, bool LAST>
void launch_draws(const Sample& p, unsigned blocks, hipStream_t st) {
  if (p.n_draws >= kSearchFrom)
    sample_kernel<NV, S, FILTER, LAST, true><<<blocks, kPixels * S, 0, st>>>(p);
  else
    sample_kernel<NV, S, FILTER, LAST, false><<<blocks, kPixels * S, 0, st>>>(p);
}
template <int NV, int S>
void launch(const Sample& p, bool filter, bool labels_first, unsigned blocks, hipStream_t st) {
  if (filter && labels_first)
    launch_draws<NV, S, true, false>(p, blocks, st);
  else if (filter)
    launch_draws<NV, S, true, true>(p, blocks, st);
  else if (labels_first)
    launch_draws<NV, S, false, false>(p, blocks, st);
  else
    launch_draws<NV, S, false, true>(p, blocks, st);
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
  // (a launch has less than 2^32 threads, at most eight per pixel)
  const int64_t threads = kPixels * (n_disp <= 32 ? 2 : 8);
  if (items > 0x7fffffff || pixels > ((int64_t)1 << 40) || tiles > 0xffffffff / threads / items)
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
  p.inv_t_all = temperature > 0 ? 1.0 / (double)temperature : 0.0;
  p.reach_all = temperature > 0 && min_p > 0 ? reach_of(temperature, min_p) : 0;
  p.pixels = pixels;
  p.tiles = tiles;
  p.items_pixels = items * pixels;
  p.n = n_disp;
  p.n_cv = n_cv;
  p.n_draws = n_draws;
  p.reciprocal = n_disp > 1 ? (uint32_t)((((uint64_t)1 << 32) + (uint64_t)n_disp - 1) / (uint64_t)n_disp) : 0u;
  p.quads = n_disp % 4 == 0 && ((uintptr_t)cost & 15) == 0;
  // Where rows are not whole cache lines the tiles beside each other share lines, which one die's L2 can join.  us, tiles dealt
  // out one by one -> groups of 16: 60 labels 375x451 14.0 -> 12.8, 16 labels 601x803 11.2 -> 10.1, 192 labels 1501x1999 479 ->
  // 465, 97 labels 301x803 28.5 -> 29.6.
  p.xcd_group = labels_first && pixels * 4 % kLineBytes != 0 ? 16 : 0;
  const bool filter = temperatures != nullptr || !(temperature > 0) || top_ks != nullptr || (top_k > 0 && top_k < n_disp) ||
                      top_ps != nullptr || top_p < 1.f || min_ps != nullptr || min_p > 0.f;
  const unsigned blocks = (unsigned)(tiles * items);
  const hipStream_t st = (hipStream_t)stream;
  const bool lf = labels_first != 0;
  // Labels per lane and lanes per pixel.  Many labels in a lane need fewer instructions, many lanes more wavefronts: up to
  // kFewTiles workgroups a launch is short of those.  us, few lanes / many: no filter, all filters: 30 labels
  // 129x129 (261 tiles) 5.3 / 4.5, 21.0 / 15.3; 60 labels 375x450, 16 draws, top-k (2637) 38.8 / 33.0; 45 labels 800x900
  // (11 250) 30.8 / 34.2, 88.6 / 99.6; 128 labels 375x1242 (7277) 60.6 / 63.2, 141 / 154; 96 labels 384x1248 (7488) 41 / 48,
  // 110 / 134.
  const bool few = blocks <= kFewTiles;
  if (n_disp <= 4)
    launch<4, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 8)
    launch<8, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 16)
    few ? launch<8, 2>(p, filter, lf, blocks, st) : launch<16, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 24)
    few ? launch<12, 2>(p, filter, lf, blocks, st) : launch<24, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 32)
    few ? launch<16, 2>(p, filter, lf, blocks, st) : launch<32, 1>(p, filter, lf, blocks, st);
  else if (n_disp <= 48)
    few ? launch<12, 4>(p, filter, lf, blocks, st) : launch<24, 2>(p, filter, lf, blocks, st);
  else if (n_disp <= 64)
    few ? launch<16, 4>(p, filter, lf, blocks, st) : launch<32, 2>(p, filter, lf, blocks, st);
  else if (n_disp <= 96)
    few ? launch<12, 8>(p, filter, lf, blocks, st) : launch<24, 4>(p, filter, lf, blocks, st);
  else if (n_disp <= 128)
    few ? launch<16, 8>(p, filter, lf, blocks, st) : launch<32, 4>(p, filter, lf, blocks, st);
  else if (n_disp <= 192)
    launch<24, 8>(p, filter, lf, blocks, st);
  else
    launch<32, 8>(p, filter, lf, blocks, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "sample_labels: %s", hipGetErrorString(e));
}

}  // extern "C"
