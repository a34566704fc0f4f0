// Eviction by demand (include/dilution_hip.h: dil_evict): of a slice's `length`
// cached keys the first `first`, the last `recent` and the most demanded of those
// between move to a new cache, in their order.
//
// The want-th largest demand of a slice is found digit by digit (11, 11 and 10 bits
// of an integer that orders as the demand does): the counts of the keys that share
// the digits found so far, summed from the top digit down.  Above it every key stays,
// and of its equals the first that are wanted.
//
//   evict_select  (slices)              up to 32768 keys between: the slice in one
//                                       workgroup, its keys in registers (and its rows
//                                       moved there, where they are few)
//   evict_digit   (chunks x slices)     longer: four launches, each of them reads the
//                                       demand once; a chunk's counts go through memory
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

constexpr int kWaves = kSelThreads / 64;
constexpr int kBins = 2048;
// digit `level` of a key: bits [shift, shift + width)
__host__ __device__ constexpr int digit_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__host__ __device__ constexpr uint32_t digit_mask(int level) { return level == 2 ? 1023u : 2047u; }

// One bin's place: the counts of thread t's two bins (2 t and 2 t + 1), with the
// counts of the higher bins before them.
struct Found {
  int bin, left, count;           // the bin that holds the want-th largest, how many of it are wanted, and how many it has
};
// Every thread of the workgroup calls.
__device__ __forceinline__ Found find_bin(int h0, int h1, int want, int* scratch) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int suffix = h0 + h1;           // over the lanes from this one on
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_down(suffix, o, 64);
    if (lane + o < 64) suffix += x;
  }
  __syncthreads();
  if (lane == 0) scratch[wave] = suffix;
  __syncthreads();
  int above = suffix - h0 - h1;
  for (int w = wave + 1; w < kWaves; ++w) above += scratch[w];
  if (above < want && want <= above + h1) {
    scratch[kWaves] = 2 * t + 1;
    scratch[kWaves + 1] = want - above;
    scratch[kWaves + 2] = h1;
  } else if (above + h1 < want && want <= above + h1 + h0) {
    scratch[kWaves] = 2 * t;
    scratch[kWaves + 1] = want - above - h1;
    scratch[kWaves + 2] = h0;
  }
  __syncthreads();
  return {scratch[kWaves], scratch[kWaves + 1], scratch[kWaves + 2]};
}

// Counts a key's digit.  The lanes that have the first counting lane's digit count
// as one: demands crowd into few digits (all of them where many keys hold none), and
// equal addresses of a wave's atomics take turns.
__device__ __forceinline__ void count_digit(int* hist, uint32_t digit, bool on) {
  const uint64_t active = __ballot(on);
  if (active == 0) return;
  const int lead = __ffsll(static_cast<unsigned long long>(active)) - 1;
  const bool same = on && digit == static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(digit), lead));
  const uint64_t with = __ballot(same);
  if (same) {
    if ((threadIdx.x & 63) == lead) atomicAdd(&hist[digit], __popcll(with));
  } else if (on) {
    atomicAdd(&hist[digit], 1);
  }
}

// The kept positions of one block of keys, in order.  Key e of thread t is position
// j0 + e * 1024 + t; `ties` equals came before the block, and its first kept
// position is number `at`.  Both move past the block.
template <int E>
__device__ __forceinline__ void emit_kept(const uint32_t (&key)[E], int64_t j0, int64_t j1, uint32_t least, int want,
                                          int& ties, int64_t& at, int32_t* dst, int2 (*cnt)[kWaves], int2* total) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint64_t below = (uint64_t{1} << lane) - 1;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = j0 + e * kSelThreads + t < j1;
    const uint64_t ma = __ballot(in && key[e] > least), me = __ballot(in && key[e] == least);
    if (lane == 0) cnt[e][wave] = make_int2(__popcll(ma), __popcll(me));
  }
  __syncthreads();
  if (wave == 0) {                 // exclusive sums over the (e, wave) runs, in order
    int2 run = make_int2(0, 0);
    for (int b = 0; b < E * kWaves; b += 64) {
      int2* c = &cnt[0][0] + b + lane;
      const bool in = b + lane < E * kWaves;
      const int2 mine = in ? *c : make_int2(0, 0);
      int2 x = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int xa = __shfl_up(x.x, o, 64), xe = __shfl_up(x.y, o, 64);
        if (lane >= o) {
          x.x += xa;
          x.y += xe;
        }
      }
      if (in) *c = make_int2(run.x + x.x - mine.x, run.y + x.y - mine.y);
      run.x += __shfl(x.x, 63, 64);
      run.y += __shfl(x.y, 63, 64);
    }
    if (lane == 0) *total = run;
  }
  __syncthreads();
  const int taken = min(ties, want);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t j = j0 + e * kSelThreads + t;
    const bool in = j < j1, above = in && key[e] > least, equal = in && key[e] == least;
    const uint64_t ma = __ballot(above), me = __ballot(equal);
    const int2 c = cnt[e][wave];
    const int rank = ties + c.y + __popcll(me & below);          // equals at lower positions
    if (above || (equal && rank < want)) dst[at + c.x + __popcll(ma & below) + min(rank, want) - taken] = static_cast<int32_t>(j);
  }
  at += total->x + min(ties + total->y, want) - taken;
  ties += total->y;
}

// The positions that stay whatever they carry.
__device__ __forceinline__ void emit_ends(int32_t* dst, int64_t length, int64_t keep, int64_t first, int64_t recent) {
  for (int64_t j = threadIdx.x; j < first; j += kSelThreads) dst[j] = static_cast<int32_t>(j);
  for (int64_t j = threadIdx.x; j < recent; j += kSelThreads) dst[keep - recent + j] = static_cast<int32_t>(length - recent + j);
}

// Where the rows go; a row is 2^shift units of 16 bytes.
struct Move {
  const u32x4* k;
  const u32x4* v;
  u32x4* ko;
  u32x4* vo;
  float* co;
  int64_t out_cap;
  int shift;
  bool here;                       // evict_select moves the rows itself
};

struct Select {
  const float* committed;
  int64_t cap, length, keep, first, recent;
  int32_t* index;
  int64_t slice0;
  // the chunked form
  int64_t chunk;
  int chunks;
  int* hist;                       // (3 levels, n, chunks, kBins)
  int64_t level_stride;
  int4* state;                     // (n): after level k the digits found so far, and how many equals are wanted
  int* before;                     // (n, chunks): keys above the digits found so far in the chunks before
  Move m;
};

// Units u0, u0 + stride, ... (kMoveUnits of them, K and V of all in flight) of an
// output slice.
constexpr int kMoveUnits = 4;

__device__ __forceinline__ void move_units(const Move& m, const float* committed, int64_t cap, const int32_t* index, int64_t keep,
                                           int64_t slice, int64_t u0, int64_t stride) {
  const int64_t units = m.out_cap << m.shift;
  const int part = (1 << m.shift) - 1;
  u32x4 x[kMoveUnits], y[kMoveUnits];
  float c[kMoveUnits];
#pragma unroll
  for (int i = 0; i < kMoveUnits; ++i) {
    const int64_t u = u0 + i * stride, r = u >> m.shift;
    x[i] = y[i] = u32x4{0, 0, 0, 0};
    c[i] = 0.f;
    if (r < keep) {
      const int64_t row = slice * cap + index[slice * keep + r], src = (row << m.shift) + (u & part);
      x[i] = m.k[src];
      y[i] = m.v[src];
      if ((u & part) == 0) c[i] = committed[row];
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveUnits; ++i) {
    const int64_t u = u0 + i * stride;
    if (u >= units) return;
    const int64_t to = slice * units + u;
    m.ko[to] = x[i];
    m.vo[to] = y[i];
    if ((u & part) == 0) m.co[slice * m.out_cap + (u >> m.shift)] = c[i];
  }
}

template <int E>
__device__ __forceinline__ void load_keys(uint32_t (&key)[E], const float* row, int64_t j0, int64_t j1) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t j = j0 + e * kSelThreads + threadIdx.x;
    key[e] = demand_key(row[j < j1 ? j : j1 - 1]);
  }
}

// The slice in one workgroup: 1024 E keys at most.
template <int E>
__global__ __launch_bounds__(kSelThreads) void evict_select(Select A) {
  __shared__ int hist[kBins];
  __shared__ int scratch[kWaves + 3];
  __shared__ int2 cnt[E][kWaves], total;
  const int t = threadIdx.x;
  const int64_t slice = A.slice0 + blockIdx.x;
  int32_t* dst = A.index + slice * A.keep;
  const int64_t j0 = A.first, j1 = A.length - A.recent;
  int want = static_cast<int>(A.keep - A.first - A.recent);
  emit_ends(dst, A.length, A.keep, A.first, A.recent);
  auto move = [&] {
    if (!A.m.here) return;
    __syncthreads();                            // the positions are written
    const int64_t units = A.m.out_cap << A.m.shift;
    for (int64_t u = t; u < units; u += kSelThreads * kMoveUnits)
      move_units(A.m, A.committed, A.cap, A.index, A.keep, slice, u, kSelThreads);
  };
  if (want == 0) {                              // the same in every thread
    move();
    return;
  }
  uint32_t key[E];
  load_keys(key, A.committed + slice * A.cap, j0, j1);
  uint32_t digits = 0, mask = 0;
#pragma unroll
  for (int level = 0; level < 3; ++level) {
    hist[t] = hist[t + kSelThreads] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      count_digit(hist, key[e] >> digit_shift(level) & digit_mask(level),
                  j0 + e * kSelThreads + t < j1 && (key[e] & mask) == digits);
    __syncthreads();
    const Found f = find_bin(hist[2 * t], hist[2 * t + 1], want, scratch);
    digits |= static_cast<uint32_t>(f.bin) << digit_shift(level);
    mask |= digit_mask(level) << digit_shift(level);
    want = f.left;
    if (f.left == f.count) break;               // all that share these digits stay: the others need not be known
  }
#pragma unroll
  for (int e = 0; e < E; ++e) key[e] &= mask;
  int ties = 0;
  int64_t at = A.first;
  emit_kept<E>(key, j0, j1, digits, want, ties, at, dst, cnt, &total);
  move();
}

constexpr int kChunkKeys = 16;     // per thread and block

// Level LEVEL of the chunked form: the digit of level LEVEL - 1 from its counts, then
// the counts of the next digit; the last writes the positions.
template <int LEVEL>
__global__ __launch_bounds__(kSelThreads) void evict_digit(Select A) {
  __shared__ int hist[kBins];
  __shared__ int scratch[kWaves + 3];
  __shared__ int2 cnt[kChunkKeys][kWaves], total;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int c = blockIdx.x;
  const int64_t slice = A.slice0 + blockIdx.y;
  const int64_t end = A.length - A.recent;
  const int64_t j0 = A.first + c * A.chunk, j1 = min(j0 + A.chunk, end);
  uint32_t digits = 0;
  int want = static_cast<int>(A.keep - A.first - A.recent);
  int before = 0, ties = 0;                     // keys above the threshold, and equal to it, in the chunks before
  if constexpr (LEVEL > 0) {
    if constexpr (LEVEL > 1) {
      const int4 s = A.state[slice * 2 + (LEVEL - 2)];
      digits = static_cast<uint32_t>(s.x);
      want = s.y;
      before = A.before[(slice * 2 + LEVEL - 2) * A.chunks + c];
    }
    const int* h = A.hist + (LEVEL - 1) * A.level_stride + slice * A.chunks * kBins + 2 * t;
    int all0 = 0, all1 = 0, pre0 = 0, pre1 = 0;
#pragma unroll 4
    for (int i = 0; i < A.chunks; ++i) {
      const int2 x = *reinterpret_cast<const int2*>(h + static_cast<int64_t>(i) * kBins);
      all0 += x.x;
      all1 += x.y;
      pre0 += i < c ? x.x : 0;
      pre1 += i < c ? x.y : 0;
    }
    const Found f = find_bin(all0, all1, want, scratch);
    digits |= static_cast<uint32_t>(f.bin) << digit_shift(LEVEL - 1);
    want = f.left;
    int up = (2 * t > f.bin ? pre0 : 0) + (2 * t + 1 > f.bin ? pre1 : 0);
    int eq = (2 * t == f.bin ? pre0 : 0) + (2 * t + 1 == f.bin ? pre1 : 0);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      up += __shfl_xor(up, o, 64);
      eq += __shfl_xor(eq, o, 64);
    }
    if (lane == 0) cnt[0][wave] = make_int2(up, eq);
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
      before += cnt[0][w].x;
      ties += cnt[0][w].y;
    }
    if (LEVEL < 3 && t == 0) {
      A.before[(slice * 2 + LEVEL - 1) * A.chunks + c] = before;
      if (c == 0) A.state[slice * 2 + LEVEL - 1] = make_int4(static_cast<int>(digits), want, 0, 0);
    }
  }
  const float* row = A.committed + slice * A.cap;
  if constexpr (LEVEL < 3) {
    constexpr uint32_t kFoundMask = LEVEL == 0 ? 0u : LEVEL == 1 ? ~0u << 21 : ~0u << 10;
    hist[t] = hist[t + kSelThreads] = 0;
    __syncthreads();
    for (int64_t b = j0; b < j1; b += kChunkKeys * kSelThreads) {
      uint32_t key[kChunkKeys];
      load_keys(key, row, b, j1);
#pragma unroll
      for (int e = 0; e < kChunkKeys; ++e)
        count_digit(hist, key[e] >> digit_shift(LEVEL) & digit_mask(LEVEL),
                    b + e * kSelThreads + t < j1 && (key[e] & kFoundMask) == digits);
    }
    __syncthreads();
    int* h = A.hist + LEVEL * A.level_stride + (slice * A.chunks + c) * kBins;
    h[t] = hist[t];
    h[t + kSelThreads] = hist[t + kSelThreads];
  } else {
    int32_t* dst = A.index + slice * A.keep;
    if (c == 0) emit_ends(dst, A.length, A.keep, A.first, A.recent);
    int64_t at = A.first + before + min(ties, want);
    for (int64_t b = j0; b < j1; b += kChunkKeys * kSelThreads) {
      uint32_t key[kChunkKeys];
      load_keys(key, row, b, j1);
      emit_kept<kChunkKeys>(key, b, j1, digits, want, ties, at, dst, cnt, &total);
    }
  }
}

__global__ __launch_bounds__(kMoveThreads) void evict_move(Move m, const float* committed, int64_t cap, const int32_t* index,
                                                           int64_t keep, int64_t slice0) {
  move_units(m, committed, cap, index, keep, slice0 + blockIdx.y,
             static_cast<int64_t>(blockIdx.x) * (kMoveThreads * kMoveUnits) + threadIdx.x, kMoveThreads);
}

}  // namespace

namespace {

// The most keys that one workgroup selects from, as many as its registers hold.  us a call
// (head_dim 64, half of the keys stay), one workgroup a slice -> chunks:
//   8192 keys: 1, 16, 64, 256 slices 16 -> 31, 19 -> 36, 34 -> 51, 120 -> 139
//   16384 21 -> 36, 31 -> 45, 66 -> 81, 237 -> 253;  24576 35 -> 37, 47 -> 51, 113 -> 118, 352 -> 379
//   32768 36.2 -> 37.5, 56.2 -> 55.7, 142 -> 143, 462 -> 488
constexpr int64_t kOneMax = 32 * kSelThreads;
constexpr int64_t kMaxChunks = 64;

// The chunked form's chunks: of 16384 keys, longer ones where that makes more than 64.
int64_t chunk_of(int64_t keys) {
  const int64_t block = kChunkKeys * kSelThreads, per = (keys + kMaxChunks - 1) / kMaxChunks;
  return (per + block - 1) / block * block;
}
// Places for the most chunks that any first and recent leave of `length` keys: by the
// length alone, as the workspace's size.
struct EvictScratch {
  size_t hist, state, before, total;
  EvictScratch(int64_t n, int64_t length) {
    const int64_t blocks = (length + kChunkKeys * kSelThreads - 1) / (kChunkKeys * kSelThreads);
    const int64_t chunks = length <= kOneMax ? 0 : blocks < kMaxChunks ? blocks : kMaxChunks;
    hist = 0;
    state = hist + align_up(sizeof(int) * 3 * n * chunks * kBins);
    before = state + align_up(sizeof(int4) * 2 * n * (chunks != 0));
    total = before + align_up(sizeof(int) * 2 * n * chunks);
  }
};

}  // namespace

int64_t evict_workspace_bytes(int64_t n, int64_t length, int64_t keep) {
  (void)keep;
  return n < 1 || length < 1 ? 0 : static_cast<int64_t>(EvictScratch(n, length).total) + 256;
}

int evict(const EvictArgs& a) {
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int64_t keys = a.length - a.first - a.recent;
  int shift = 0;                                           // head_dim is a power of two
  while (16 << shift < a.head_dim * (a.dtype == DT_F32 ? 4 : 2)) ++shift;
  const bool one = keys <= kOneMax || a.keep == a.first + a.recent;
  // Up to 64 KB of K rows a slice the selecting workgroup moves them itself and saves
  // the launch; above, a launch of its own has more workgroups for them.  us a call, own
  // launch -> here: 16 slices of 16, 32, 64, 128 KB 10.7 -> 8.4, 10.6 -> 8.5, 10.6 -> 9.5, 12.1
  // -> 13.2; 64 slices 10.6 -> 8.6, 10.7 -> 9.2, 11.7 -> 11.3, 15.4 -> 15.7; 256 slices 11.9 -> 9.3,
  // 14.4 -> 11.5, 19.3 -> 16.8, 34.7 -> 33.1.
  constexpr int64_t kHereUnits = 4096;
  const bool here = one && (a.out_cap << shift) <= kHereUnits;
  Select S{a.committed, a.cap, a.length, a.keep, a.first, a.recent, a.index, 0, 0, 0, nullptr, 0, nullptr, nullptr,
           Move{static_cast<const u32x4*>(a.k_cache), static_cast<const u32x4*>(a.v_cache), static_cast<u32x4*>(a.k_out),
                static_cast<u32x4*>(a.v_out), a.committed_out, a.out_cap, shift, here}};
  if (one) {
    // batches of slices: one grid holds fewer than 2^32 threads, those of 4194304 slices
    auto select = [&](auto e) {
      slice_batches(a.n, [&](int64_t s0, unsigned ns) {
        S.slice0 = s0;
        DIL_TIMED("evict_select", st, (evict_select<e()><<<dim3(ns), kSelThreads, 0, st>>>(S)));
      });
    };
    if (keys <= 4 * kSelThreads || a.keep == a.first + a.recent) select(std::integral_constant<int, 4>{});
    else if (keys <= 8 * kSelThreads) select(std::integral_constant<int, 8>{});
    else if (keys <= 16 * kSelThreads) select(std::integral_constant<int, 16>{});
    else select(std::integral_constant<int, 32>{});
  } else {
    const EvictScratch w(a.n, a.length);
    char* ws = static_cast<char*>(a.workspace);
    S.chunk = chunk_of(keys);
    S.chunks = static_cast<int>((keys + S.chunk - 1) / S.chunk);
    S.hist = reinterpret_cast<int*>(ws + w.hist);
    S.level_stride = a.n * S.chunks * kBins;
    S.state = reinterpret_cast<int4*>(ws + w.state);
    S.before = reinterpret_cast<int*>(ws + w.before);
    slice_batches(a.n, [&](int64_t s0, unsigned ns) {
      S.slice0 = s0;
      const dim3 grid(static_cast<unsigned>(S.chunks), ns);
      DIL_TIMED("evict_digit0", st, (evict_digit<0><<<grid, kSelThreads, 0, st>>>(S)));
      DIL_TIMED("evict_digit1", st, (evict_digit<1><<<grid, kSelThreads, 0, st>>>(S)));
      DIL_TIMED("evict_digit2", st, (evict_digit<2><<<grid, kSelThreads, 0, st>>>(S)));
      DIL_TIMED("evict_digit3", st, (evict_digit<3><<<grid, kSelThreads, 0, st>>>(S)));
    });
  }
  if (!here) {
    const int64_t blocks = ((a.out_cap << shift) + kMoveThreads * kMoveUnits - 1) / (kMoveThreads * kMoveUnits);
    slice_batches(a.n, [&](int64_t s0, unsigned ns) {
      DIL_TIMED("evict_move", st,
                (evict_move<<<dim3(static_cast<unsigned>(blocks), ns), kMoveThreads, 0, st>>>(S.m, a.committed, a.cap, a.index,
                                                                                    a.keep, s0)));
    });
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace dil
