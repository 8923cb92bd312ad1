// What the operators that draw and rank labels share: candidates, a weight in 64 bits, and reductions over the lanes of a pixel.
#ifndef MPLAYERS_AMD_MP_LANES_H_
#define MPLAYERS_AMD_MP_LANES_H_

#include "mp_common.h"
#include "mp_offsets.h"

namespace mpl {

constexpr float kInf = __builtin_huge_valf();

// +inf for what is no candidate.  By bits: the library is compiled for code without NaNs.
__device__ __forceinline__ float candidate(float c) {
  return (__builtin_bit_cast(int, c) & 0x7fffffff) > 0x7f800000 ? kInf : c;
}
// The same in two instructions.  A minimum of two is the other one beside a NaN, or, beside a signalling one, that NaN made quiet,
// which the second is of.  (In asm: where there are no NaNs the compiler takes a minimum with +inf for the number itself.  And no
// comparison: a select may read a lane mask only two issue slots after it was written, which nothing in asm waits for.)
__device__ __forceinline__ float candidate_of(float c) {
  float out;
  asm("v_min_f32 %0, %2, %1\n\tv_min_f32 %0, %2, %0" : "=v"(out) : "v"(c), "s"(kInf));
  return out;
}

// 2^y, y <= 0, to about 2^-51: the exponential series of the fraction, whose 14th term is below 2^-52 of the first.
__device__ __forceinline__ double exp2_64(double y) {
  y = y > -2000.0 ? y : -2000.0;
  const double whole = rint(y), x = (y - whole) * 0.69314718055994530942;
  // (coefficients in scalar registers: the kernels have few others to spare)
  const auto scalar = [](double c) {
    asm("" : "+s"(c));
    return c;
  };
  double e = scalar(1.0 / 6227020800);
  e = fma(e, x, scalar(1.0 / 479001600));
  e = fma(e, x, scalar(1.0 / 39916800));
  e = fma(e, x, scalar(1.0 / 3628800));
  e = fma(e, x, scalar(1.0 / 362880));
  e = fma(e, x, scalar(1.0 / 40320));
  e = fma(e, x, scalar(1.0 / 5040));
  e = fma(e, x, scalar(1.0 / 720));
  e = fma(e, x, scalar(1.0 / 120));
  e = fma(e, x, scalar(1.0 / 24));
  e = fma(e, x, scalar(1.0 / 6));
  e = fma(e, x, 0.5);
  e = fma(e, x, 1.0);
  e = fma(e, x, 1.0);
  return ldexp(e, (int)whole);
}
// x > 0 and a number
__device__ __forceinline__ bool positive(float x) {
  const int bits = __builtin_bit_cast(int, x);
  return bits > 0 && bits <= 0x7f800000;
}

// Reductions over the S lanes of a pixel, neighbours: within a row of 16, or the whole wavefront (S = 64, all lanes at
// work; the four rows meet in scalar registers).
template <int CTRL>
__device__ __forceinline__ int move(int x) {
  return __builtin_amdgcn_mov_dpp(x, CTRL, 0xf, 0xf, true);  // (0 where there is no such lane: part of what uses it)
}
template <int CTRL>
__device__ __forceinline__ float move(float x) {
  return __builtin_bit_cast(float, move<CTRL>(__builtin_bit_cast(int, x)));
}
template <int CTRL>
__device__ __forceinline__ double move(double x) {
  const int64_t bits = __builtin_bit_cast(int64_t, x);
  const uint32_t lo = (uint32_t)move<CTRL>((int)(uint32_t)bits), hi = (uint32_t)move<CTRL>((int)(bits >> 32));
  return __builtin_bit_cast(double, (int64_t)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ int from_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ float from_lane(float x, int lane) { return readlane_f(x, lane); }
__device__ __forceinline__ double from_lane(double x, int lane) {
  const int64_t bits = __builtin_bit_cast(int64_t, x);
  const uint32_t lo = (uint32_t)from_lane((int)(uint32_t)bits, lane), hi = (uint32_t)from_lane((int)(bits >> 32), lane);
  return __builtin_bit_cast(double, (int64_t)(((uint64_t)hi << 32) | lo));
}
template <int S, typename V, typename F>
__device__ __forceinline__ V over_lanes(V x, F f) {
  if (S > 1) x = f(x, move<0xB1>(x));   // the other of a pair
  if (S > 2) x = f(x, move<0x4E>(x));   // the other pair of four
  if (S > 4) x = f(x, move<0x141>(x));  // the other four of eight
  if (S > 8) x = f(x, move<0x140>(x));  // the other eight
  if (S > 16) x = f(f(from_lane(x, 0), from_lane(x, 16)), f(from_lane(x, 32), from_lane(x, 48)));
  return x;
}
template <int S, typename V>
__device__ __forceinline__ V lanes_min(V x) {
  return over_lanes<S>(x, [](V a, V b) { return b < a ? b : a; });
}
template <int S, typename V>
__device__ __forceinline__ V lanes_max(V x) {
  return over_lanes<S>(x, [](V a, V b) { return b > a ? b : a; });
}
template <int S, typename V>
__device__ __forceinline__ V lanes_sum(V x) {
  return over_lanes<S>(x, [](V a, V b) { return a + b; });
}
// x of the lane that CTRL names, in the rows of MASK; 0 where there is none
template <int CTRL, int MASK = 0xf>
__device__ __forceinline__ double move_or_0(double x) {
  const int64_t bits = __builtin_bit_cast(int64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CTRL, MASK, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(bits >> 32), CTRL, MASK, 0xf, false);
  return __builtin_bit_cast(double, (int64_t)(((uint64_t)hi << 32) | lo));
}
// f over the wavefront's lanes up to this one, where f(x, 0) is x
template <typename F>
__device__ __forceinline__ double wave_upto(double x, F f) {
  x = f(x, move_or_0<0x111>(x));       // one lane up a row, two, four, eight
  x = f(x, move_or_0<0x112>(x));
  x = f(x, move_or_0<0x114>(x));
  x = f(x, move_or_0<0x118>(x));
  x = f(x, move_or_0<0x142, 0xa>(x));  // the last of a row to the next row: rows 1 and 3
  x = f(x, move_or_0<0x143, 0xc>(x));  // the last of row 1 to rows 2 and 3
  return x;
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


// ------------------------------------------------------------------------------------------------------------------
// Tiles of 64 pixels in registers, a pixel's NV * S labels over S lanes beside each other: lane s owns labels s * NV ...
// s * NV + NV - 1.  A workgroup of 64 * S threads.
constexpr int kLanePixels = 64;

struct LaneTiles {
  int64_t pixels, tiles;  // of an item
  int n;
  uint32_t reciprocal;    // 2^32 / n, rounded up
  int xcd_group;          // tiles beside each other that go to one die (xcd_block)
};
// False where a launch would have too many threads, eight to a pixel at most.  bytes: of a cost; rows: in the network's layout,
// where tiles share the cache lines of rows that are not whole ones.
inline bool make_lane_tiles(LaneTiles& t, int64_t items, int n_disp, int64_t pixels, bool rows, int bytes) {
  const int64_t threads = kLanePixels * (n_disp <= 32 ? 2 : 8);
  if (items > 0x7fffffff || pixels > ((int64_t)1 << 40)) return false;
  t.pixels = pixels;
  t.tiles = (pixels + kLanePixels - 1) / kLanePixels;
  if (t.tiles > 0xffffffff / threads / items) return false;
  t.n = n_disp;
  t.reciprocal = n_disp > 1 ? (uint32_t)((((uint64_t)1 << 32) + (uint64_t)n_disp - 1) / (uint64_t)n_disp) : 0u;
  t.xcd_group = rows && pixels * bytes % kLineBytes != 0 ? 16 : 0;
  return true;
}

// In LDS the quads of a pixel lie in the order in which its lanes read them: quad q, of lane q / (NV / 4), at place
// q % (NV / 4) * S + q / (NV / 4); pixels an odd number of quads apart.
template <int NV, int S>
struct LaneTile {
  static constexpr int kQuads = S * NV / 4, kJ = NV / 4, kStride = 4 * (kQuads | 1);
  // (q is below 64, where these multiplications of 24 bits divide by kJ)
  static __device__ __forceinline__ unsigned place(unsigned q) {
    if (S == 1) return q * 4;
    const unsigned lane = __umul24(q, (256 + kJ - 1) / kJ) >> 8;
    return (__umul24(q - __umul24(lane, kJ), S) + lane) * 4;
  }
};

// What a thread loads of a tile: the costs of the item begin at `cost`, the tile at pixel p0, `count` pixels of it are there.
// Labels behind the last and pixels behind the last are read from the last's place, so that no branch lies between the loads.
template <int NV, int S, bool LAST, typename T>
struct LaneLoads {
  T c[NV];

  __device__ __forceinline__ void load(const T* cost, const LaneTiles& t, int64_t p0, int count, int mode, int tid) {
    constexpr int kJ = NV / 4, kThreads = kLanePixels * S;
    const int n = t.n;
    if (LAST) {
      const unsigned total = (unsigned)(count * n);
      const T* from = cost + p0 * n;
      if (mode != kEach) {
#pragma unroll
        for (int k = 0; k < kJ; ++k) {
          T q[4];
          load_quad(from, min((unsigned)(tid + k * kThreads), total / 4 - 1), q);
#pragma unroll
          for (int j = 0; j < 4; ++j) c[4 * k + j] = q[j];
        }
      } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) c[k] = load_at(from, min((unsigned)(tid + k * kThreads), total - 1));
      }
    } else {
      const int of = min(tid % kLanePixels, count - 1), wave = uniform_i(tid / kLanePixels);
#pragma unroll
      for (int i = 0; i < kJ; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          c[4 * i + j] = cost[(int64_t)min(4 * (wave + i * S) + j, n - 1) * t.pixels + p0 + of];
    }
  }
  // What is no candidate goes there as +inf, and what lies behind the last label too.
  __device__ __forceinline__ void to_tile(float* tile, const LaneTiles& t, int count, int mode, int tid) const {
    using Tile = LaneTile<NV, S>;
    constexpr int kJ = NV / 4, kThreads = kLanePixels * S;
    const auto cost = [&](int k) { return candidate_of((float)c[k]); };
    if (LAST) {
      for (int l = t.n + tid % S; l < S * NV; l += S) tile[tid / S * Tile::kStride + Tile::place(l >> 2) + (l & 3)] = kInf;
    }
    if (LAST) {
      const unsigned n = (unsigned)t.n, total = (unsigned)count * n;
      if (mode == kQuads) {
#pragma unroll
        for (int k = 0; k < kJ; ++k) {
          const unsigned i = min((unsigned)(tid + k * kThreads) * 4, total - 4);
          const unsigned of = __umulhi(i, t.reciprocal), l = i - of * n;
          *reinterpret_cast<float4*>(&tile[of * Tile::kStride + Tile::place(l >> 2)]) =
              float4{cost(4 * k), cost(4 * k + 1), cost(4 * k + 2), cost(4 * k + 3)};
        }
      } else if (mode == kFours) {
        // (which need not be of one pixel)
#pragma unroll
        for (int k = 0; k < kJ; ++k) {
          const unsigned i = min((unsigned)(tid + k * kThreads) * 4, total - 4);
          const unsigned of = n == 1 ? i : __umulhi(i, t.reciprocal);
          unsigned l = i - of * n, row = of * Tile::kStride;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            tile[row + Tile::place(l >> 2) + (l & 3)] = cost(4 * k + j);
            const bool last = l + 1 == n;
            row += last ? Tile::kStride : 0;
            l = last ? 0 : l + 1;
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const unsigned i = min((unsigned)(tid + k * kThreads), total - 1);
          const unsigned of = n == 1 ? i : __umulhi(i, t.reciprocal), l = i - of * n;
          tile[of * Tile::kStride + Tile::place(l >> 2) + (l & 3)] = cost(k);
        }
      }
    } else {
      const int wave = uniform_i(tid / kLanePixels);
#pragma unroll
      for (int i = 0; i < kJ; ++i) {
        const int l = 4 * (wave + i * S);
        float4* const to = reinterpret_cast<float4*>(&tile[tid % kLanePixels * Tile::kStride + Tile::place(wave + i * S)]);
        if (l + 3 < t.n) {
          *to = float4{cost(4 * i), cost(4 * i + 1), cost(4 * i + 2), cost(4 * i + 3)};
        } else {
          const auto of = [&](int j) { return l + j < t.n ? cost(4 * i + j) : kInf; };
          *to = float4{of(0), of(1), of(2), of(3)};
        }
      }
    }
  }
};

// The lane's costs out of LDS.
template <int NV, int S>
__device__ __forceinline__ void from_lane_tile(const float* tile, int px, int s, float (&v)[NV]) {
#pragma unroll
  for (int g = 0; g < NV / 4; ++g) {
    const float4 q = *reinterpret_cast<const float4*>(&tile[px * LaneTile<NV, S>::kStride + (g * S + s) * 4]);
    v[4 * g] = q.x;
    v[4 * g + 1] = q.y;
    v[4 * g + 2] = q.z;
    v[4 * g + 3] = q.w;
  }
}

}  // namespace mpl

#endif  // MPLAYERS_AMD_MP_LANES_H_
