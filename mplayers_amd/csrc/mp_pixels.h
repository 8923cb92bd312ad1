// Tiles of 64 pixels with a lane to a pixel, for the operators that stand around the layers.
//
// W wavefronts share the labels of a tile: wavefront w owns the quads (four labels) w, w + W, ..., I of them at most, so
// that every one has as many labels as the others but for one quad.  With W = 1 the G wavefronts of a workgroup have a tile
// each and meet nobody.
//
// In the network's layout (labels in front of the pixels) a lane reads its pixel in the row of each of its labels: 256 bytes to
// an instruction in fp32.  In the operators' layout (labels innermost) a tile is one run of memory, which goes through LDS: the
// labels of a pixel side by side, an odd number of quads apart, which keeps the 16-byte accesses of either side off each
// other's banks.
#ifndef MPLAYERS_AMD_MP_PIXELS_H_
#define MPLAYERS_AMD_MP_PIXELS_H_

#include "mp_common.h"
#include "mp_offsets.h"

namespace mpl {

constexpr int kTilePixels = 64;

struct Tiles {
  int64_t pixels;       // of an item
  unsigned per_item;    // tiles
  unsigned total;
  int labels;
  uint32_t reciprocal;  // 2^32 / labels, rounded up
  int xcd_group;        // workgroups beside each other that go to one die (xcd_block)
};

// W wavefronts of I quads each to a tile, G tiles to a workgroup.
template <int W, int I, int G>
struct TileShape {
  static_assert(W == 1 || G == 1, "wavefronts that share a tile meet at the workgroup's barrier");
  static constexpr int kW = W, kI = I, kG = G;
};
// Shapes for every four labels up to 32, us for 40 M costs in place of those for the next eight: the divergence and its gradient
// together, lists of 4, 10 labels 147 -> 141, labels last 160 -> 133, 18 labels 133 -> 114 and 130 -> 112, 26 labels 133 -> 116 and 125 ->
// 109; layer norm's forward pass (its gradient has shapes of its own) 10 labels 65.5 -> 64.5, 18 labels 67.4 -> 64.3, bf16 47.4 ->
// 45.9, 26 labels 64.8 -> 64.2 and 45.7 -> 43.7.
template <typename F>
inline void with_shape(int n, F f) {
  if (n <= 4)
    f(TileShape<1, 1, 4>());
  else if (n <= 8)
    f(TileShape<1, 2, 4>());
  else if (n <= 12)
    f(TileShape<1, 3, 4>());
  else if (n <= 16)
    f(TileShape<1, 4, 4>());
  else if (n <= 20)
    f(TileShape<1, 5, 4>());
  else if (n <= 24)
    f(TileShape<1, 6, 4>());
  else if (n <= 28)
    f(TileShape<1, 7, 4>());
  else if (n <= 32)
    f(TileShape<1, 8, 4>());
  else if (n <= 48)
    f(TileShape<2, 6, 1>());
  else if (n <= 64)
    f(TileShape<4, 4, 1>());
  else if (n <= 96)
    f(TileShape<4, 6, 1>());
  else if (n <= 128)
    f(TileShape<8, 4, 1>());
  else if (n <= 192)
    f(TileShape<8, 6, 1>());
  else
    f(TileShape<8, 8, 1>());
}

// False where a launch would have too many threads.  bytes: of a cost; rows: in the network's layout.
// Where rows are not whole cache lines the tiles beside each other share lines, which one die's L2 can join.  us, tiles dealt
// out one by one -> groups of 8 -> 16: layer norm forward 192 labels 377x501 69 -> 63 -> 63, 60 labels 375x451 16.6 -> 15.8 ->
// 15.1, its gradient 126 -> 115 -> 116, 28.6 -> 26.8 -> 26.4, 97 labels 301x803 68 -> 62 -> 63, bf16 21 labels 12x129x129 12.3 ->
// 12.4 -> 12.9; distillation's gradient 192 labels 76 -> 68 -> 66, 97 labels 63 -> 58 -> 57.
inline bool make_tiles(Tiles& t, int items, int n_disp, int64_t pixels, bool rows, int bytes) {
  int threads = 0;
  with_shape(n_disp, [&](auto s) { threads = kTilePixels * s.kW; });
  if (pixels > ((int64_t)1 << 40)) return false;
  const int64_t per_item = (pixels + kTilePixels - 1) / kTilePixels;
  // (less than 2^31 threads, so that tiles and workgroups are ints as well)
  if (per_item > 0x7fffffff / threads / items) return false;
  t.pixels = pixels;
  t.per_item = (unsigned)per_item;
  t.total = (unsigned)per_item * (unsigned)items;
  t.labels = n_disp;
  t.reciprocal = n_disp > 1 ? (uint32_t)((((uint64_t)1 << 32) + (uint64_t)n_disp - 1) / (uint64_t)n_disp) : 0u;
  t.xcd_group = rows && pixels * bytes % kLineBytes != 0 ? 16 : 0;
  return true;
}

constexpr int tile_stride(int quads) { return 4 * (quads | 1); }  // floats from pixel to pixel in LDS

// What the wavefronts of a tile wait for each other with.
template <int W>
__device__ __forceinline__ void tile_sync() {
  if (W > 1) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Rows of the network's layout: from = the item's first label at the tile's first pixel.  Labels behind the last are read
// from the last's place, so that there is no branch between the loads.
template <int W, int I, typename T>
__device__ __forceinline__ void load_rows(const T* from, const Tiles& t, int w, int of, float (&x)[I][4]) {
  T raw[I][4];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[i][j] = from[(int64_t)min(4 * (w + i * W) + j, t.labels - 1) * t.pixels + of];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i][j] = (float)raw[i][j];
}

template <int W, int I, typename T>
__device__ __forceinline__ void store_rows(T* to, const Tiles& t, int w, int of, const float (&x)[I][4]) {
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int l = 4 * (w + i * W) + j;
      if (l < t.labels) to[(int64_t)l * t.pixels + of] = (T)x[i][j];
    }
}

// A run of the operators' layout, `total` labels of whole pixels, as the threads of a tile hold it on its way.
template <int I, typename T>
struct Run {
  T x[4 * I];
};

// Entry i of a run in the tile.
template <int STRIDE>
__device__ __forceinline__ unsigned tile_place(unsigned i, const Tiles& t) {
  const unsigned p = t.labels == 1 ? i : __umulhi(i, t.reciprocal);
  return p * STRIDE + (i - p * (unsigned)t.labels);
}

// Calls f with the place in the tile of each of the four entries from i on, which need not be of one pixel.
template <int STRIDE, typename F>
__device__ __forceinline__ void four_places(unsigned i, const Tiles& t, F f) {
  const unsigned n = (unsigned)t.labels, p = n == 1 ? i : __umulhi(i, t.reciprocal);
  unsigned l = i - p * n, place = p * STRIDE + l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f(j, place);
    const bool last = l + 1 == n;
    place += last ? STRIDE + 1 - n : 1;
    l = last ? 0 : l + 1;
  }
}

// mode: of the run (run_mode_of), with FOURS any, else not kFours.  tid: of the 64 * W threads of the tile.
template <int W, int I, bool FOURS = true, typename T>
__device__ __forceinline__ void load_run(const T* from, unsigned total, int mode, int tid, Run<I, T>& r) {
  constexpr int kThreads = 64 * W;
  if (mode != kEach) {
#pragma unroll
    for (int k = 0; k < I; ++k) {
      T q[4];
      load_quad(from, min((unsigned)(tid + k * kThreads), total / 4 - 1), q);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.x[4 * k + j] = q[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4 * I; ++k) r.x[k] = load_at(from, min((unsigned)(tid + k * kThreads), total - 1));
  }
}
template <int W, int I, bool FOURS = true, typename T>
__device__ __forceinline__ void run_to_tile(const Run<I, T>& r, unsigned total, int mode, int tid, const Tiles& t, float* tile) {
  constexpr int kThreads = 64 * W, kStride = tile_stride(W * I);
  if (FOURS ? mode == kQuads : mode != kEach) {
#pragma unroll
    for (int k = 0; k < I; ++k)
      *reinterpret_cast<float4*>(&tile[tile_place<kStride>(min((unsigned)(tid + k * kThreads) * 4, total - 4), t)]) =
          float4{(float)r.x[4 * k], (float)r.x[4 * k + 1], (float)r.x[4 * k + 2], (float)r.x[4 * k + 3]};
  } else if (FOURS && mode == kFours) {
#pragma unroll
    for (int k = 0; k < I; ++k)
      four_places<kStride>(min((unsigned)(tid + k * kThreads) * 4, total - 4), t,
                           [&](int j, unsigned place) { tile[place] = (float)r.x[4 * k + j]; });
  } else {
#pragma unroll
    for (int k = 0; k < 4 * I; ++k)
      tile[tile_place<kStride>(min((unsigned)(tid + k * kThreads), total - 1), t)] = (float)r.x[k];
  }
}
template <int W, int I, bool FOURS = true, typename T>
__device__ __forceinline__ void store_run(T* to, unsigned total, int mode, int tid, const Tiles& t, const float* tile) {
  constexpr int kThreads = 64 * W, kStride = tile_stride(W * I);
  if (FOURS ? mode == kQuads : mode != kEach) {
    for (unsigned i = (unsigned)tid * 4; i < total; i += kThreads * 4) {
      const float4 x = *reinterpret_cast<const float4*>(&tile[tile_place<kStride>(i, t)]);
      store_quad(to, i / 4, (T)x.x, (T)x.y, (T)x.z, (T)x.w);
    }
  } else if (FOURS && mode == kFours) {
    for (unsigned i = (unsigned)tid * 4; i < total; i += kThreads * 4) {
      float x[4];
      four_places<kStride>(i, t, [&](int j, unsigned place) { x[j] = tile[place]; });
      store_quad(to, i / 4, (T)x[0], (T)x[1], (T)x[2], (T)x[3]);
    }
  } else {
    for (unsigned i = (unsigned)tid; i < total; i += kThreads) store_at(to, i, (T)tile[tile_place<kStride>(i, t)]);
  }
}

// A lane's labels in the tile: tile = its pixel's.
template <int W, int I>
__device__ __forceinline__ void from_tile(const float* tile, int w, float (&x)[I][4]) {
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const float4 q = *reinterpret_cast<const float4*>(&tile[4 * (w + i * W)]);
    x[i][0] = q.x;
    x[i][1] = q.y;
    x[i][2] = q.z;
    x[i][3] = q.w;
  }
}
template <int W, int I>
__device__ __forceinline__ void to_tile(float* tile, int w, const float (&x)[I][4]) {
#pragma unroll
  for (int i = 0; i < I; ++i)
    *reinterpret_cast<float4*>(&tile[4 * (w + i * W)]) = float4{x[i][0], x[i][1], x[i][2], x[i][3]};
}

}  // namespace mpl

#endif  // MPLAYERS_AMD_MP_PIXELS_H_
