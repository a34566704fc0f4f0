// Eviction by demand (include/dilution_hip.h: dil_evict): of a slice's `length`
// cached keys the first `first`, the last `recent` and the most demanded of those
// between move to a new cache, in their order.
//
//   evict_select  (slices)              the positions kept
//   evict_move    (row blocks x slices) K, V and demand rows to their places, zero
//                                       past the last
#include "dil_common.hpp"
#include "dil_internal.hpp"

namespace dil {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A demand as an integer of the same order: -0 as +0, NaN above everything.
__device__ __forceinline__ uint32_t demand_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The w-th largest key of [j0, j1) is found a byte at a time (the counts of the
// keys that share the bytes found so far), then the kept positions are written in
// order: all above it, and as many of its equals, lowest first, as are wanted.
__global__ __launch_bounds__(kSelThreads) void evict_select(const float* __restrict__ committed, int64_t cap, int64_t length,
                                                            int64_t keep, int64_t first, int64_t recent,
                                                            int32_t* __restrict__ index) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const float* row = committed + static_cast<int64_t>(blockIdx.x) * cap;
  int32_t* dst = index + static_cast<int64_t>(blockIdx.x) * keep;
  const int64_t j1 = length - recent;
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_want;
  __shared__ int cnt[2][kSelThreads / 64];
  uint32_t prefix = 0, mask = 0;
  int want = static_cast<int>(keep - first - recent);
  for (int64_t j = t; j < first; j += kSelThreads) dst[j] = static_cast<int32_t>(j);
  for (int64_t j = t; j < recent; j += kSelThreads) dst[keep - recent + j] = static_cast<int32_t>(j1 + j);
  if (want == 0) return;                        // the same in every thread
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    for (int64_t j = first + t; j < j1; j += kSelThreads) {
      const uint32_t k = demand_key(row[j]);
      if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1);
    }
    __syncthreads();
    if (t == 0) {
      int left = want, b = 255;
      while (b > 0 && hist[b] < left) left -= hist[b--];
      s_prefix = prefix | static_cast<uint32_t>(b) << shift;
      s_want = left;
    }
    __syncthreads();
    prefix = s_prefix;
    want = s_want;
    mask |= 0xffu << shift;
  }
  // want: how many keys equal to the threshold `prefix` stay
  int ties = 0;
  int64_t at = first;
  for (int64_t b = first; b < j1; b += kSelThreads) {
    const int64_t j = b + t;
    const uint32_t k = j < j1 ? demand_key(row[j]) : 0;
    const bool above = j < j1 && k > prefix, equal = j < j1 && k == prefix;
    const uint64_t ma = __ballot(above), me = __ballot(equal);
    const uint64_t below = (uint64_t{1} << lane) - 1;
    __syncthreads();                            // the counts of the round before are read
    if (lane == 0) {
      cnt[0][wave] = __popcll(ma);
      cnt[1][wave] = __popcll(me);
    }
    __syncthreads();
    int a0 = 0, e0 = 0, at_all = 0, e_all = 0;
    for (int w = 0; w < kSelThreads / 64; ++w) {
      if (w < wave) {
        a0 += cnt[0][w];
        e0 += cnt[1][w];
      }
      at_all += cnt[0][w];
      e_all += cnt[1][w];
    }
    const int eq_before = ties + e0 + __popcll(me & below);   // equals at lower positions
    const int64_t place = at + a0 + __popcll(ma & below) + (min(eq_before, want) - min(ties, want));
    if (above || (equal && eq_before < want)) dst[place] = static_cast<int32_t>(j);
    at += at_all + min(ties + e_all, want) - min(ties, want);
    ties += e_all;
  }
}

__global__ __launch_bounds__(kMoveThreads) void evict_move(const u32x4* __restrict__ k, const u32x4* __restrict__ v,
                                                           const float* __restrict__ committed, int64_t cap,
                                                           const int32_t* __restrict__ index, int64_t keep, int64_t out_cap,
                                                           int units, u32x4* __restrict__ ko, u32x4* __restrict__ vo,
                                                           float* __restrict__ co, int64_t slice0) {
  const int64_t slice = slice0 + blockIdx.y;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x;   // 16-byte unit of the output slice
  const int64_t r = u / units;
  if (r >= out_cap) return;
  const int64_t c = u - r * units;
  const int64_t to = (slice * out_cap + r) * units + c;
  if (r < keep) {
    const int64_t src = slice * cap + index[slice * keep + r];
    ko[to] = k[src * units + c];
    vo[to] = v[src * units + c];
    if (c == 0) co[slice * out_cap + r] = committed[src];
  } else {
    ko[to] = vo[to] = u32x4{0, 0, 0, 0};
    if (c == 0) co[slice * out_cap + r] = 0.f;
  }
}

}  // namespace

int64_t evict_workspace_bytes(int64_t n, int64_t length, int64_t keep) {
  (void)n;
  (void)length;
  (void)keep;
  return 256;
}

int evict(const EvictArgs& a) {
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  DIL_TIMED("evict_select", st,
            (evict_select<<<dim3(static_cast<unsigned>(a.n)), kSelThreads, 0, st>>>(a.committed, a.cap, a.length, a.keep, a.first,
                                                                           a.recent, a.index)));
  const int units = a.head_dim * (a.dtype == DT_F32 ? 4 : 2) / 16;
  const int64_t blocks = (a.out_cap * units + kMoveThreads - 1) / kMoveThreads;
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    DIL_TIMED("evict_move", st,
              (evict_move<<<dim3(static_cast<unsigned>(blocks), ns), kMoveThreads, 0, st>>>(
                  static_cast<const u32x4*>(a.k_cache), static_cast<const u32x4*>(a.v_cache), a.committed, a.cap, a.index, a.keep,
                  a.out_cap, units, static_cast<u32x4*>(a.k_out), static_cast<u32x4*>(a.v_out), a.committed_out, s0)));
  });
  return static_cast<int>(hipGetLastError());
}

}  // namespace dil
