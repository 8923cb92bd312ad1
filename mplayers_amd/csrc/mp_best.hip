// The labels of least cost of every pixel, in order, their costs, and what the others weigh: what is kept of a teacher.
// For gfx950.
//
// cost -> k labels by cost, equal ones by label, with their costs relative to the best one (what a softmax of them needs, and what
// fits a narrow type), and rest = -T log(sum over the other candidates of exp(-(c - best) / T)).  +inf and NaN are no candidates.
// A difference that the list's type has no number for is not in the list, so its label is one of the others.
//
// The costs are read once, a pixel's labels over S lanes (mp_lanes.h), and stay in LDS; a lane has the least cost of each quad of
// its labels in registers.  A place of the list is the least of those over the lanes: the first lane that has it looks its
// quad up, takes the label out and finds the quad's next.  So a place costs the instructions of the quads and not of the
// labels, and no sort is needed.  us: 96 labels 384x1248, lists of 8, 53 (3.9 TB/s; label by label 83), 810 instructions to a
// wavefront of 16 pixels, 0.8 of the time; 21 labels 12x129x129, lists of 4, 8.5; 192 labels 377x501, lists of 32, 106, bound by
// the instructions.

#include "mp_lanes.h"

using namespace mpl;

namespace {

// Places of the list that wait in LDS for whole rows.  us for 48 M costs, lists of 8, with 16 / 8 / 4: 21 labels 86 / 68 / 73, 192
// labels 66 / 55 / 57; lists of 32, 192 labels 377x501 124 / 109 / 116.
constexpr int kChunk = 8;

struct Best {
  LaneTiles t;
  const void* cost;
  uint8_t* labels;
  void* costs;
  float* rest;  // or nullptr
  int k, kept;  // places of the list, type of their costs
  float limit;  // from here on a difference is +inf in that type
  float temperature, to_exponent;  // T, log2(e) / T
  int mode;  // of runs
};

template <typename T, int NV, int S, bool LAST>
__global__ void __launch_bounds__(kLanePixels* S) best_kernel(Best p) {
  __shared__ __align__(16) float tile[kLanePixels * LaneTile<NV, S>::kStride];
  __shared__ float found_cost[kChunk][kLanePixels];
  __shared__ uint8_t found_label[kChunk][kLanePixels];
  const unsigned block = (unsigned)xcd_block((int)blockIdx.x, (int)gridDim.x, p.t.xcd_group), tiles = (unsigned)p.t.tiles;
  const int64_t item = block / tiles, p0 = (int64_t)(block - (unsigned)item * tiles) * kLanePixels;
  const int count = (int)min((int64_t)kLanePixels, p.t.pixels - p0);
  const int tid = (int)threadIdx.x, px = tid / S, s = tid % S;
  using Tile = LaneTile<NV, S>;
  constexpr int kJ = Tile::kJ;
  {
    LaneLoads<NV, S, LAST, T> loads;
    const int64_t at = item * p.t.n * p.t.pixels;
    const int mode = LAST ? run_mode_of(p.mode, at, (unsigned)(count * p.t.n)) : (int)kEach;
    loads.load((const T*)p.cost + at, p.t, p0, count, mode, tid);
    loads.to_tile(tile, p.t, count, mode, tid);
  }
  __syncthreads();
  // quad g of this lane is at own[g * 4 * S]; nobody else reads or writes it from here on
  float* const own = &tile[px * Tile::kStride + s * 4];
  const auto quad = [&](int g) { return *reinterpret_cast<const float4*>(own + g * 4 * S); };
  const auto least_of = [](const float4& q) {
    const float a = q.x < q.y ? q.x : q.y, b = q.z < q.w ? q.z : q.w;
    return a < b ? a : b;
  };
  float least[kJ];
#pragma unroll
  for (int g = 0; g < kJ; ++g) least[g] = least_of(quad(g));
  const auto mine = [&]() {
    float m = least[0];
#pragma unroll
    for (int g = 1; g < kJ; ++g) m = least[g] < m ? least[g] : m;
    return m;
  };
  float best = lanes_min<S>(mine());
  if (__builtin_amdgcn_ballot_w64(best == -kInf) != 0) {
    // beside a cost of -inf only others of -inf are candidates
    if (best == -kInf) {
      for (int g = 0; g < kJ; ++g)
        for (int j = 0; j < 4; ++j) own[g * 4 * S + j] = own[g * 4 * S + j] == -kInf ? 0.f : kInf;
#pragma unroll
      for (int g = 0; g < kJ; ++g) least[g] = least[g] == -kInf ? 0.f : kInf;
      best = 0;
    }
  }
  for (int first = 0; first < p.k; first += kChunk) {
    const int here = min(kChunk, p.k - first);
    for (int k = 0; k < here; ++k) {
      const float m = mine(), all = lanes_min<S>(m);
      const int who = S == 1 ? 0 : lanes_min<S>(m == all ? s : S);
      int g = 0;
#pragma unroll
      for (int i = kJ - 1; i >= 0; --i) g = least[i] == all ? i : g;
      if (s == who) {
        float* const at = own + g * 4 * S;
        float4 q = *reinterpret_cast<const float4*>(at);
        const int j = q.x == all ? 0 : q.y == all ? 1 : q.z == all ? 2 : 3;
        const float c = all < kInf ? all - best : kInf;
        const bool fits = c < p.limit;
        if (fits) {  // (else it stays, for the rest)
          at[j] = kInf;
          q.x = j == 0 ? kInf : q.x;
          q.y = j == 1 ? kInf : q.y;
          q.z = j == 2 ? kInf : q.z;
          q.w = j == 3 ? kInf : q.w;
          const float next = least_of(q);
#pragma unroll
          for (int i = 0; i < kJ; ++i) least[i] = i == g ? next : least[i];
        }
        found_cost[k][px] = fits ? c : kInf;
        found_label[k][px] = (uint8_t)(fits ? s * NV + 4 * g + j : 0);
      }
    }
    __syncthreads();
    // whole rows of pixels, or of places
    for (int i = tid; i < here * kLanePixels; i += kLanePixels * S) {
      const int k = LAST ? i % here : i / kLanePixels, of = LAST ? i / here : i % kLanePixels;
      if (of < count) {
        const int64_t at = LAST ? (item * p.t.pixels + p0 + of) * p.k + first + k : (item * p.k + first + k) * p.t.pixels + p0 + of;
        const float c = found_cost[k][of];
        p.labels[at] = found_label[k][of];
        if (p.kept == MPL_F32)
          ((float*)p.costs)[at] = c;
        else if (p.kept == MPL_F16)
          ((_Float16*)p.costs)[at] = (_Float16)c;
        else
          ((__bf16*)p.costs)[at] = (__bf16)c;
      }
    }
    __syncthreads();
  }
  if (p.rest != nullptr) {
    const float m = lanes_min<S>(mine());
    float sum = 0;
#pragma unroll
    for (int g = 0; g < kJ; ++g) {
      const float4 q = quad(g);
      const float c[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += __builtin_amdgcn_exp2f((m - c[j]) * p.to_exponent);  // (0 of +inf beside a number)
    }
    sum = lanes_sum<S>(sum);
    if (s == 0 && px < count) p.rest[item * p.t.pixels + p0 + px] = m < kInf ? (m - best) - p.temperature * logf(sum) : kInf;
  }
}

// Labels per lane and lanes per pixel.  us for 48 M costs, lists of 8: 16 labels 74 (a lane) / 86 (two), 24: 82 / 87, 32: 70 / 73,
// 48: 69 / 63, 64: 61 (two) / 61 (four), 96: 64 / 55, 128: 67 / 54, 192: 72 (four) / 67 (eight), 256: 68 / 60.  Where a quarter or a
// sixth of the lanes' labels would be none: 40 M costs, lists of 4, 4 labels 106 -> 82, 10 56 -> 49, 18 45 -> 38, 26 44 -> 36; 72 labels 500x1000 52 -> 46, 150 93 -> 89, 220 134 -> 129 (104: 68 -> 69, not taken).
template <typename T, bool LAST>
void launch(const Best& p, unsigned blocks, hipStream_t st) {
  const int n = p.t.n;
  if (n <= 4)
    best_kernel<T, 4, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 8)
    best_kernel<T, 8, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 12)
    best_kernel<T, 12, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 16)
    best_kernel<T, 16, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 20)
    best_kernel<T, 20, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 24)
    best_kernel<T, 24, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 28)
    best_kernel<T, 28, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 32)
    best_kernel<T, 32, 1, LAST><<<blocks, kLanePixels, 0, st>>>(p);
  else if (n <= 48)
    best_kernel<T, 24, 2, LAST><<<blocks, kLanePixels * 2, 0, st>>>(p);
  else if (n <= 64)
    best_kernel<T, 16, 4, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 80)
    best_kernel<T, 20, 4, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 96)
    best_kernel<T, 24, 4, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 128)
    best_kernel<T, 32, 4, LAST><<<blocks, kLanePixels * 4, 0, st>>>(p);
  else if (n <= 160)
    best_kernel<T, 20, 8, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else if (n <= 192)
    best_kernel<T, 24, 8, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else if (n <= 224)
    best_kernel<T, 28, 8, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
  else
    best_kernel<T, 32, 8, LAST><<<blocks, kLanePixels * 8, 0, st>>>(p);
}

}  // namespace

extern "C" int mpl_best_labels(int dtype, int labels_first, const void* cost, int n_kept, float temperature, int kept_dtype,
                               uint8_t* kept_labels, void* kept_costs, float* rest, int items, int n_disp, int64_t pixels,
                               void* stream) {
  if (dtype < 0 || dtype > MPL_BF16) return fail(MPL_EINVAL, "best_labels: unknown data type %d", dtype);
  if (kept_dtype < 0 || kept_dtype > MPL_BF16) return fail(MPL_EINVAL, "best_labels: unknown data type %d of the list", kept_dtype);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "best_labels: n_disp must be in [1, %d], got %d", kMaxL, n_disp);
  if (n_kept < 1 || n_kept > n_disp)
    return fail(MPL_EINVAL, "best_labels: the list must have 1 to n_disp = %d places, got %d", n_disp, n_kept);
  if (!(temperature > 0 && temperature < kInf && (float)(1.4426950408889634 / (double)temperature) < kInf))
    return fail(MPL_EINVAL, "best_labels: the temperature must be finite and above 0, and its inverse finite");
  if (items < 0 || pixels < 0) return fail(MPL_EINVAL, "best_labels: negative size");
  if (items == 0 || pixels == 0) return MPL_OK;
  if (cost == nullptr || kept_labels == nullptr || kept_costs == nullptr) return fail(MPL_EINVAL, "best_labels: null pointer");
  Best p = {};
  if (!make_lane_tiles(p.t, items, n_disp, pixels, labels_first != 0, dtype == MPL_F32 ? 4 : 2))
    return fail(MPL_EINVAL, "best_labels: too many pixels");
  p.cost = cost;
  p.labels = kept_labels;
  p.costs = kept_costs;
  p.rest = rest;
  p.k = n_kept;
  p.kept = kept_dtype;
  // (half a step above the type's largest number)
  p.limit = kept_dtype == MPL_F16 ? 65520.f : kept_dtype == MPL_BF16 ? 0x1.ffp127f : kInf;
  p.temperature = temperature;
  p.to_exponent = (float)(1.4426950408889634 / (double)temperature);
  p.mode = run_mode(n_disp, ((uintptr_t)cost & (dtype == MPL_F32 ? 15 : 7)) == 0);
  const unsigned blocks = (unsigned)(p.t.tiles * items);
  const auto by_type = [&](auto type) {
    using T = decltype(type);
    labels_first != 0 ? launch<T, false>(p, blocks, (hipStream_t)stream) : launch<T, true>(p, blocks, (hipStream_t)stream);
  };
  if (dtype == MPL_F32)
    by_type(float());
  else if (dtype == MPL_F16)
    by_type((_Float16)0);
  else
    by_type((__bf16)0);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "best_labels: %s", hipGetErrorString(e));
}
