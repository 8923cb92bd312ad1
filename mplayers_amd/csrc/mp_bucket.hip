// Pairwise tables whose entries go by buckets of the label distance, and their gradient, for gfx950.
//
// A layer of n labels with a learned 1-D table has n - 1 entries to learn, of which the far ones see few pairs.
// With buckets it learns n_buckets: context[k] = table[bucket(k)], k = |a - b|, as a vector or as the (n, n) table
// of all pairs of labels.  Bucket b is the distances starts[b] <= k < starts[b + 1], so its gradient is the sum of the
// context's over these distances.
//
// At most 256 labels: a vector is 1 KiB, a square table 256 KiB, so the launches are what these calls cost.  Hence
// one launch each, and the borders travel as kernel arguments (no copy to the device, nothing a capture could not
// hold).  us, table / gradient: 256 labels, 32 buckets 2.0 / 2.3; 21x21, 8 buckets 2.4 / 2.8; 16 tables of 256x256, 64 buckets
// 3.6 / 6.6.

#include "mp_common.h"

using namespace mpl;

namespace {

struct BucketOf {
  uint8_t of[kMaxL];
};
struct BucketStarts {
  int16_t at[kMaxL + 1];
};
struct BucketGroups {
  int16_t at[kMaxL + 1];  // first bucket of each group
};

// One thread per entry of a row; a workgroup of 64 x 4 threads takes kRows rows of a square table, or one vector.
constexpr int kRows = 16;
template <bool SQUARE>
__global__ void __launch_bounds__(256) bucket_context_kernel(BucketOf map, const float* __restrict__ table,
                                                             float* __restrict__ context, int n_buckets, int n,
                                                             int lower) {
  const int tid = (int)(threadIdx.y * 64 + threadIdx.x);
  const float* t = table + (int64_t)blockIdx.y * n_buckets;
  if (!SQUARE) {
    if (tid < n) context[(int64_t)blockIdx.y * n + tid] = t[map.of[tid]];
    return;
  }
  __shared__ float value[kMaxL];
  if (tid < n) value[tid] = t[map.of[tid]];
  __syncthreads();
  float* c = context + (int64_t)blockIdx.y * n * n;
  const int end = min(n, ((int)blockIdx.x + 1) * kRows);
  for (int a = (int)blockIdx.x * kRows + (int)threadIdx.y; a < end; a += 4)
    for (int b = (int)threadIdx.x; b < n; b += 64) c[a * n + b] = b >= a || lower ? value[abs(a - b)] : 0.f;
}

// A vector's gradient: one wavefront per bucket and table.
__global__ void __launch_bounds__(64) bucket_sums_kernel(BucketStarts starts, const float* __restrict__ dcontext,
                                                         float* __restrict__ dtable, int n_buckets, int n) {
  const int b = (int)blockIdx.x, t = (int)threadIdx.x;
  const float* d = dcontext + (int64_t)blockIdx.y * n;
  double sum = 0;
  for (int k = starts.at[b] + t; k < starts.at[b + 1]; k += 64) sum += (double)d[k];
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if (t == 0) dtable[(int64_t)blockIdx.y * n_buckets + b] = (float)sum;
}

// A square table's gradient: one workgroup per table and group of whole buckets that hold kRun distances or more.  kRun
// threads beside each other take a distance each, so that narrow buckets read runs of a row too; the others take other
// rows.  (With a workgroup per bucket, a bucket of one distance reads a cache line for each entry: 16 tables of 256
// labels, 64 buckets 7.8 us.)  Sums in 64 bits and in a fixed order: a bucket adds up to 65 536 entries.
constexpr int kRun = 32, kThreads = 1024;
__global__ void __launch_bounds__(kThreads) bucket_square_sums_kernel(BucketStarts starts, BucketGroups groups,
                                                                      const float* __restrict__ dcontext,
                                                                      float* __restrict__ dtable, int n_buckets, int n,
                                                                      int lower) {
  __shared__ double part[kThreads / 64][kRun];
  __shared__ double sums[kMaxL];  // of the group's distances
  const int t = (int)threadIdx.x, lane = t & 63, wave = t >> 6;
  const int first = groups.at[blockIdx.x], last = groups.at[blockIdx.x + 1];  // buckets
  const int from = starts.at[first], to = starts.at[last];
  const float* d = dcontext + (int64_t)blockIdx.y * n * n;
  for (int k0 = from; k0 < to; k0 += kRun) {
    const int k = k0 + t % kRun;
    double sum = 0;
    // (no branch between the loads: what is not there is read from the diagonal and left out)
#pragma unroll 8
    for (int a = t / kRun; a < n; a += kThreads / kRun) {
      const bool right = k < to && a + k < n, left = k < to && lower && k > 0 && a >= k;
      const float x = d[a * (n + 1) + (right ? k : 0)], y = d[a * (n + 1) - (left ? k : 0)];
      sum += (double)(right ? x : 0.f) + (double)(left ? y : 0.f);
    }
    sum += __shfl_xor(sum, kRun);
    if (lane < kRun) part[wave][lane] = sum;
    __syncthreads();
    if (t < kRun && k < to) {
      double all = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i) all += part[i][t];
      sums[k - from] = all;
    }
    __syncthreads();
  }
  for (int b = first + wave; b < last; b += kThreads / 64) {
    double sum = 0;
    for (int k = starts.at[b] + lane; k < starts.at[b + 1]; k += 64) sum += sums[k - from];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
    if (lane == 0) dtable[(int64_t)blockIdx.y * n_buckets + b] = (float)sum;
  }
}

int check_buckets(const char* what, const void* a, const void* b, const int32_t* starts, int n_tables, int n_buckets,
                  int n_disp) {
  if (a == nullptr || b == nullptr || starts == nullptr) return fail(MPL_EINVAL, "%s: null pointer", what);
  if (n_disp < 1 || n_disp > kMaxL) return fail(MPL_EINVAL, "%s: n_disp must be in [1, %d], got %d", what, kMaxL, n_disp);
  if (n_buckets < 1 || n_buckets > kMaxL)
    return fail(MPL_EINVAL, "%s: n_buckets must be in [1, %d], got %d", what, kMaxL, n_buckets);
  if (n_tables < 0 || n_tables > 65535) return fail(MPL_EINVAL, "%s: n_tables must be in [0, 65535]", what);
  if (starts[0] != 0 || starts[n_buckets] != n_disp)
    return fail(MPL_EINVAL, "%s: the buckets must run from distance 0 to n_disp", what);
  for (int i = 0; i < n_buckets; ++i)
    if (starts[i] > starts[i + 1]) return fail(MPL_EINVAL, "%s: the buckets must be in order", what);
  return MPL_OK;
}

}  // namespace

extern "C" {

int mpl_bucket_context(const float* table, const int32_t* starts, int n_tables, int n_buckets, int n_disp, int square,
                       float* context, void* stream) {
  if (int rc = check_buckets("bucket_context", table, context, starts, n_tables, n_buckets, n_disp)) return rc;
  if (square < 0 || square > 2) return fail(MPL_EINVAL, "bucket_context: square must be 0, 1 or 2, got %d", square);
  if (n_tables == 0) return MPL_OK;
  BucketOf map = {};
  for (int b = 0; b < n_buckets; ++b)
    for (int k = starts[b]; k < starts[b + 1]; ++k) map.of[k] = (uint8_t)b;
  const hipStream_t st = (hipStream_t)stream;
  if (square)
    bucket_context_kernel<true><<<dim3((unsigned)((n_disp + kRows - 1) / kRows), (unsigned)n_tables), dim3(64, 4), 0, st>>>(
        map, table, context, n_buckets, n_disp, square == 2);
  else
    bucket_context_kernel<false><<<dim3(1, (unsigned)n_tables), dim3(64, 4), 0, st>>>(map, table, context, n_buckets,
                                                                                     n_disp, 0);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "bucket_context: %s", hipGetErrorString(e));
}

int mpl_bucket_sums(const float* dcontext, const int32_t* starts, int n_tables, int n_buckets, int n_disp, int square,
                    float* dtable, void* stream) {
  if (int rc = check_buckets("bucket_sums", dcontext, dtable, starts, n_tables, n_buckets, n_disp)) return rc;
  if (square < 0 || square > 2) return fail(MPL_EINVAL, "bucket_sums: square must be 0, 1 or 2, got %d", square);
  if (n_tables == 0) return MPL_OK;
  BucketStarts at = {};
  for (int b = 0; b <= n_buckets; ++b) at.at[b] = (int16_t)starts[b];
  const hipStream_t st = (hipStream_t)stream;
  if (square) {
    BucketGroups groups = {};
    int n_groups = 0;
    for (int b = 1; b < n_buckets; ++b)
      if (starts[b] - starts[groups.at[n_groups]] >= kRun) groups.at[++n_groups] = (int16_t)b;
    groups.at[++n_groups] = (int16_t)n_buckets;
    bucket_square_sums_kernel<<<dim3((unsigned)n_groups, (unsigned)n_tables), kThreads, 0, st>>>(
        at, groups, dcontext, dtable, n_buckets, n_disp, square == 2);
  } else {
    bucket_sums_kernel<<<dim3((unsigned)n_buckets, (unsigned)n_tables), 64, 0, st>>>(at, dcontext, dtable, n_buckets, n_disp);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MPL_OK : fail(MPL_ELAUNCH, "bucket_sums: %s", hipGetErrorString(e));
}

}  // extern "C"
