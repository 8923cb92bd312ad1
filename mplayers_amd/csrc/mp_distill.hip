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
// A tile of 64 pixels, a lane to each (mp_pixels.h).  The costs lie in LDS too, where the entries find the student's cost of
// their label; the wavefronts of a tile share the list, and each has weights of its own labels that serve the student's sum, the
// others' and the gradient, so there is one exponential to a label.  us, loss / gradient: 192 labels 1500x2000, lists of 8 in fp16
// and a rest, 596 / 945 (4.0 and 5.0 TB/s; with each wavefront going through the whole list 1190 / 2390); 21 labels
// 12x129x129, lists of 4, 9.2 / 12.5.  Bound by HBM, the loss by the instructions as well: 570 to a wavefront of 24 labels, 0.6 of
// the time.

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
  int mode;                  // of runs of both volumes
};

__device__ __forceinline__ float kept_cost(const Distill& p, int64_t base, unsigned of) {
  return p.kept == MPL_F32   ? load_at((const float*)p.costs + base, of)
         : p.kept == MPL_F16 ? (float)load_at((const _Float16*)p.costs + base, of)
                             : (float)load_at((const __bf16*)p.costs + base, of);
}

// A cost not above any of some costs, and the sum of their weights relative to it; (+inf, 0) of none.
struct Mass {
  float least, sum;
};
__device__ __forceinline__ float weight(float least, float c, float to_exponent) {
  return c == kInf ? 0.f : __builtin_amdgcn_exp2f((least - c) * to_exponent);
}
// The least of three numbers, of those that are numbers; one instruction (and comparisons that may meet NaN are two each).
__device__ __forceinline__ float least_of(float a, float b, float c) {
  float least;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(least) : "v"(a), "v"(b), "v"(c));
  return least;
}
// Those of the W wavefronts of a tile.
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

constexpr float kFaint = 0x1p-60f;  // others that weigh less than this beside the best label: see distill_kernel

// HELD: entries of the list that a wavefront keeps in registers, the rest is fetched twice or three times.
// (Up to 24 labels to a wavefront in 128 registers, so that two workgroups of eight share a compute unit.)
template <typename T, bool FIRST, bool GRAD, int W, int I, int G, int HELD>
__global__ void __launch_bounds__(64 * W * G, I <= 6 ? 4 : 1) distill_kernel(Distill p) {
  constexpr int kStride = tile_stride(W * I), kShift = W == 1 ? 0 : W == 2 ? 1 : W == 4 ? 2 : 3, kParts = W > 1 ? W : 1;
  __shared__ __align__(16) float tiles[G * kTilePixels * kStride];
  __shared__ float2 part[2][kParts][kTilePixels];
  __shared__ float part_far[kParts][kTilePixels];
  __shared__ uint32_t named_by[kParts][kTilePixels];  // of each wavefront's labels, those that the list names
  __shared__ uint32_t twice;                          // whether a list of the tile names one twice
  const int tid = (int)threadIdx.x % (64 * W), group = uniform_i((int)threadIdx.x / (64 * W));
  const int lane = tid % 64, w = uniform_i(tid / 64), n = p.t.labels;
  const unsigned at = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group) * G + group;
  if (at >= p.t.total) return;  // (W = 1: nobody waits for it)
  const unsigned item = at / p.t.per_item;
  const int64_t p0 = (int64_t)(at - item * p.t.per_item) * kTilePixels;
  const int count = (int)min((int64_t)kTilePixels, p.t.pixels - p0);
  const unsigned total = (unsigned)(count * n);
  const int of = min(lane, count - 1);
  const int64_t first = (int64_t)item * n * p.t.pixels, run = first + p0 * n, pixel = (int64_t)item * p.t.pixels + p0;
  const int mode = FIRST ? (int)kEach : run_mode_of(p.mode, first, total);
  float* const tile = tiles + group * kTilePixels * kStride;
  float* const mine = tile + lane * kStride;

  // Entry e of the lane's list.  This wavefront has the entries w, w + W, ..., of which the first ones stay in registers.
  struct Entry {
    int label;
    float cost;
  };
  const auto fetch = [&](int e) {
    const int64_t base = FIRST ? ((int64_t)item * p.k + e) * p.t.pixels + p0 : ((int64_t)item * p.t.pixels + p0) * p.k + e;
    const unsigned at = (unsigned)(FIRST ? of : of * p.k);
    return Entry{load_at(p.labels + base, at), kept_cost(p, base, at)};
  };
  Entry held[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = i == 0 || w + i * W < p.k ? fetch(min(w + i * W, p.k - 1)) : Entry{0, kInf};
  const auto entries = [&](auto f) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (w + i * W < p.k) f(held[i]);
    for (int e = w + HELD * W; e < p.k; e += W) f(fetch(e));
  };

  float c[I][4];
  if (FIRST) {
    load_rows<W, I>((const T*)p.cost + first + p0, p.t, w, of, c);
    to_tile<W, I>(mine, w, c);
  } else {
    Run<I, T> r;
    load_run<W, I>((const T*)p.cost + run, total, mode, tid, r);
    run_to_tile<W, I>(r, total, mode, tid, p.t, tile);
    tile_sync<W>();
    from_tile<W, I>(mine, w, c);
  }
  // weights of this wavefront's labels beside the least cost of them; labels behind the last are no candidates
  float a[I][4], least = kInf, sum = 0;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 4 * (w + i * W) + j < n ? c[i][j] : kInf;
#pragma unroll
  for (int i = 0; i < I; ++i) least = least_of(c[i][2], c[i][3], least_of(c[i][0], c[i][1], least));
  const float beside_least = least == kInf ? 0.f : least;  // (+inf weighs nothing beside any number)
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += a[i][j] = __builtin_amdgcn_exp2f((beside_least - c[i][j]) * p.to_exponent);
  if (W > 1) {
    named_by[w][lane] = 0;
    if (tid == 0) twice = 0;
  }
  const Mass student = join<W>(Mass{least, sum}, part[0], w, lane, p.to_exponent);

  // the list: what this wavefront's entries weigh, and that times log p - log q but for the logarithms of sums
  const auto cost_at = [&](int label) { return mine[min(label, n - 1)]; };
  const auto exists = [&](const Entry& e) { return e.cost != kInf && e.label < n; };
  const auto place = [&](int label) { return (label >> 2 >> kShift) * 4 + (label & 3); };
  Mass list = {kInf, 0.f};
  float far = 0;
  uint32_t named = 0;
  bool again = false;
  entries([&](const Entry& e) {
    if (!exists(e)) return;
    const uint32_t bit = 1u << place(e.label);
    if (W == 1) {
      again |= (named & bit) != 0;
      named |= bit;
    } else {
      again |= (atomicOr(&named_by[e.label >> 2 & (W - 1)][lane], bit) & bit) != 0;
    }
    list.least = cost_at(e.label) != kInf && e.cost < list.least ? e.cost : list.least;
  });
  entries([&](const Entry& e) {
    const float own = cost_at(e.label);
    const float x = exists(e) && own != kInf ? weight(list.least, e.cost, p.to_exponent) : 0.f;
    list.sum += x;
    if (!GRAD) far += x > 0 ? x * ((own - student.least) - (e.cost - list.least)) : 0.f;
  });
  if (W > 1) {
    if (GRAD && again) twice = 1;
    if (!GRAD) part_far[w][lane] = far;
    list = join<W>(list, part[1], w, lane, p.to_exponent);
    named = named_by[w][lane];
    if (!GRAD) {
      far = 0;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float2 of_wave = part[1][k][lane];
        const float x = weight(list.least, of_wave.x, p.to_exponent);
        far += x > 0 ? x * (part_far[k][lane] - of_wave.y * (of_wave.x - list.least)) : 0.f;
      }
    }
  }
  // the rest: the labels that the list does not name
  const auto is_named = [&](int i, int j) { return (named >> (4 * i + j) & 1) != 0; };
  Mass others = {kInf, 0.f};
  float rest = kInf;
  if (p.rest != nullptr) {
    rest = load_at(p.rest + pixel, of);
    Mass own = {least, 0.f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) own.sum += is_named(i, j) ? 0.f : a[i][j];
    others = join<W>(own, part[0], w, lane, p.to_exponent);  // (the list's join: the student's parts are read)
    // Beside the best label they may weigh next to nothing in fp32, where they are to be told from each other: then they
    // are weighed beside the least cost of theirs.  (Every wavefront of the tile finds the same.)
    const bool faint = !(others.sum >= kFaint);
    if (__builtin_amdgcn_ballot_w64(faint) != 0) {
      if (W > 1) tile_sync<W>();  // (the parts are read)
      float next = kInf, weigh = 0;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) next = !is_named(i, j) && c[i][j] < next ? c[i][j] : next;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) weigh += is_named(i, j) ? 0.f : weight(next, c[i][j], p.to_exponent);
      const Mass nearer = join<W>(Mass{next, weigh}, part[0], w, lane, p.to_exponent);
      others = faint ? nearer : others;
    }
    rest = others.sum == 0.f ? kInf : rest;
  }
  const float top = rest < list.least ? rest : list.least;  // the least cost of all classes
  const float list_scale = weight(top, list.least, p.to_exponent), rest_weight = weight(top, rest, p.to_exponent);
  const float mass = (list.least == kInf ? list.sum : list.sum * list_scale) + rest_weight;
  if (!GRAD) {
    far = list_scale > 0 ? list_scale * (far - list.sum * (list.least - top)) * p.inv_t : 0.f;
    if (rest_weight > 0) far += rest_weight * (((others.least - student.least) - (rest - top)) * p.inv_t - logf(others.sum));
    const float loss = far / mass + (logf(student.sum) - logf(mass));
    if (w == 0 && lane < count) store_at(p.loss + pixel, lane, mass == 0.f ? 0.f : loss);
  } else {
    // p of the list's labels, in LDS where the costs were
    const float per_mass = 1.f / mass;
    const float none[I][4] = {};
    to_tile<W, I>(mine, w, none);  // (the list's join: all entries have found their costs)
    tile_sync<W>();
    const bool in_turn = W > 1 && twice != 0;
    if (W == 1) {
      entries([&](const Entry& e) {
        if (exists(e)) mine[e.label] += weight(top, e.cost, p.to_exponent) * per_mass;
      });
    } else if (!in_turn) {
      entries([&](const Entry& e) {
        if (exists(e)) mine[e.label] = weight(top, e.cost, p.to_exponent) * per_mass;
      });
    } else {
      // a label's entries one after the other, in their order, by the wavefront whose label it is
      for (int e = 0; e < p.k; ++e) {
        const Entry x = fetch(e);
        if (exists(x) && (x.label >> 2 & (W - 1)) == w) mine[x.label] += weight(top, x.cost, p.to_exponent) * per_mass;
      }
    }
    tile_sync<W>();
    float d[I][4];
    from_tile<W, I>(mine, w, d);
    const float scale = load_at(p.dloss + pixel, of) * p.inv_t, of_student = 1.f / student.sum;
    const float share = rest_weight > 0 ? rest_weight * per_mass / others.sum : 0.f;
    const bool beside = others.least == student.least;  // (the others' weights are those of a)
    // (the difference first: where the rest is all there is, it is 0)
    const float own = weight(student.least, least, p.to_exponent);
    const float of_named = -own * of_student, of_others = own * ((beside ? share : 0.f) - of_student);
    const float nan = mass - mass;  // 0, or NaN where the teacher has one
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[i][j] += a[i][j] * (is_named(i, j) ? of_named : of_others) + nan;
      }
    if (__builtin_amdgcn_ballot_w64(!beside && share > 0) != 0) {
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d[i][j] += beside || !(share > 0) || is_named(i, j) ? 0.f : share * weight(others.least, c[i][j], p.to_exponent);
    }
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[i][j] = c[i][j] == kInf || mass == 0.f ? 0.f : d[i][j] * scale;
    if (FIRST) {
      if (lane < count) store_rows<W, I>((T*)p.dcost + first + p0, p.t, w, lane, d);
    } else {
      to_tile<W, I>(mine, w, d);
      tile_sync<W>();
      store_run<W, I>((T*)p.dcost + run, total, mode, tid, p.t, tile);
    }
  }
}

// Eight entries of a list are held by the wavefronts of a tile, and four where the list has no more and one wavefront has it.  us,
// loss and gradient, 40 M costs, one / four / eight held: 4 labels, lists of 4 142 / 114 / 119 and 201 / 155 / 182; 8 labels, 4 entries 67 /
// 56 / 58 and 133 / 98 / 111, 8 entries 125 / 116 / 99 and 206 / 179 / 150; 21 labels, 4 entries 45 / 38 / 40 and 103 / 82 / 85, 8
// entries 64 / 60 / 52 and 147 / 132 / 107; 40 labels on two wavefronts, 8 entries, two and four each 54 / 48 and 103 / 87; 60 labels on
// four, one and two each 44 / 40 and 92 / 83.
template <typename T, bool FIRST, bool GRAD>
void launch(const Distill& p, hipStream_t st) {
  with_shape(p.t.labels, [&](auto s) {
    constexpr int W = s.kW, I = s.kI, G = s.kG;
    const auto go = [&](auto held) {
      distill_kernel<T, FIRST, GRAD, W, I, G, held.value><<<(p.t.total + G - 1) / G, 64 * W * G, 0, st>>>(p);
    };
    if constexpr (W > 1)
      go(std::integral_constant<int, 8 / W>());
    else if constexpr (I == 1)
      go(std::integral_constant<int, 4>());
    else if (p.k <= 4)
      go(std::integral_constant<int, 4>());
    else
      go(std::integral_constant<int, 8>());
  });
}
template <bool GRAD>
int run(const char* what, int dtype, int labels_first, Distill& p, int kept_dtype, int k, float temperature, int items, int n_disp,
        int64_t pixels, hipStream_t st) {
  if (dtype < 0 || dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d", what, dtype);
  if (kept_dtype < 0 || kept_dtype > MPL_BF16) return fail(MPL_EINVAL, "%s: unknown data type %d of the list", what, kept_dtype);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "%s: n_disp must be in [1, %d], got %d", what, kMaxL, n_disp);
  if (k < 1 || k > kMaxL) return fail(MPL_EINVAL, "%s: the list must have 1 to %d entries, got %d", what, kMaxL, k);
  if (!(temperature > 0 && temperature < kInf && (float)(1.4426950408889634 / (double)temperature) < kInf))
    return fail(MPL_EINVAL, "%s: the temperature must be finite and above 0, and its inverse finite", what);
  if (items < 0 || pixels < 0) return fail(MPL_EINVAL, "%s: negative size", what);
  if (items == 0 || pixels == 0) return MPL_OK;
  if (p.cost == nullptr || p.labels == nullptr || p.costs == nullptr ||
      (GRAD ? p.dloss == nullptr || p.dcost == nullptr : p.loss == nullptr))
    return fail(MPL_EINVAL, "%s: null pointer", what);
  if (!make_tiles(p.t, items, n_disp, pixels, labels_first != 0, dtype == MPL_F32 ? 4 : 2))
    return fail(MPL_EINVAL, "%s: too many pixels", what);
  p.k = k;
  p.kept = kept_dtype;
  p.to_exponent = (float)(1.4426950408889634 / (double)temperature);
  p.inv_t = 1.f / temperature;
  const uintptr_t aligned = dtype == MPL_F32 ? 15 : 7;
  p.mode = run_mode(n_disp, (((uintptr_t)p.cost | (uintptr_t)p.dcost) & aligned) == 0);
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
