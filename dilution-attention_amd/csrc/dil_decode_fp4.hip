// The decode step over caches in 4 bits (dil_decode_step_fp4; the format is in dil_fp4.hpp):
// dil_decode_step's mathematics on the values that codes and scales stand for,
//
//   a_j = log2(e) q.k_j / sqrt(D),  p_j = 2^(a_j - lse),  share_j = p_j / (committed_j + p_j + eps)
//   committed_j += p_j,  out = sum share_j v_j / (sum share_j + eps)
//
// in the same launches: fp4_one where one workgroup does a slice's whole step, else fp4_stats
// (affinities to scratch, chunk max and sum), fp4_apply (shares, demand, chunk sums of share v)
// and fp4_finish.
//
// A key costs D + 2 D / 32 bytes of codes and scales, 8 of demand and 8 of affinities (84 at
// D = 64, where 16-bit caches take 272).  A lane reads 16 bytes of codes, one block of 32
// elements, so the scales stay out of the walks: a K walk leaves each block's sum of q times
// codes in LDS, where one thread a key applies the scales and adds the blocks; the shares go
// into LDS once for each block, times the V scale.  bf16 queries multiply on v_dot2_f32_bf16
// (codes are exact in bf16), others in fp32.
#include <hip/hip_runtime.h>

#include "dil_decode_impl.hpp"
#include "dil_fp4.hpp"

namespace dil {
namespace {

constexpr int kQThreads = 1024;
constexpr int kQWaves = kQThreads / 64;

// E elements a lane, so that D / E neighbouring lanes hold a row
template <int D, int E> struct QLayout {
  static constexpr int kLanesPerRow = D / E;
  static constexpr int kRowsPerWave = 64 / kLanesPerRow;
  static constexpr int kRowsPerBlock = kRowsPerWave * kQWaves;
  static constexpr int kWords = E / 8;
};
template <int D> constexpr int kQElems = D < 32 ? D : 32;

template <int W> struct CodeWords {
  uint32_t w[W];
};
template <int W>
__device__ __forceinline__ CodeWords<W> load_codes(const uint8_t* p) {
  CodeWords<W> r;
  if constexpr (W == 4) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = x[2]; r.w[3] = x[3];
  } else if constexpr (W == 2) {
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = x[0]; r.w[1] = x[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

// The workgroup's walk over `count` rows of codes from `base` on (this lane's part of row 0),
// U rows a lane in flight; rows past the end are read as the last one.
template <int D, int E>
struct CodeStream {
  using L = QLayout<D, E>;
  static constexpr int U = 4, kRows = L::kRowsPerBlock;
  const uint8_t* src;
  int first, count;
  CodeWords<L::kWords> r[U];
  __device__ __forceinline__ CodeStream(const uint8_t* base, int wave, int lane, int n)
      : src(base), first(wave * L::kRowsPerWave + lane / L::kLanesPerRow), count(n) {}
  __device__ __forceinline__ void at(int jb) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load_codes<L::kWords>(src + static_cast<int64_t>(min(jb + u * kRows, count - 1)) * (D / 2));
  }
  __device__ __forceinline__ void load() {
    if (count > 0) at(first);
  }
  template <typename F>
  __device__ __forceinline__ void walk(F&& f) {
    for (int jb = first; jb < count; jb += U * kRows) {
      if (jb != first) at(jb);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * kRows;
        if (j < count) f(j, r[u]);
      }
    }
  }
};

// A lane's part of the query, and its products with codes
template <int E, int QT> struct QueryPart {
  float q[E];
  __device__ __forceinline__ QueryPart(const void* q1, int64_t idx, int qdt) {
#pragma unroll
    for (int e = 0; e < E; e += 8) {
      float x[8];
      load8_f32(q1, idx + e, qdt, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[e + i] = x[i];
    }
  }
  __device__ __forceinline__ float dot(const CodeWords<E / 8>& c) const {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < E / 8; ++w) {
      float v[8];
      fp4_values8(c.w[w], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(q[8 * w + i], v[i], s);
    }
    return s;
  }
};
template <int E> struct QueryPart<E, DT_BF16> {
  bf16x2 q[E / 2];
  __device__ __forceinline__ QueryPart(const void* q1, int64_t idx, int) {
#pragma unroll
    for (int e = 0; e < E / 8; ++e) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(q1) + idx + 8 * e);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[4 * e + i] = bf16x2{x[2 * i], x[2 * i + 1]};
    }
  }
  __device__ __forceinline__ float dot(const CodeWords<E / 8>& c) const {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < E / 8; ++w) {
      s = __builtin_amdgcn_fdot2_f32_bf16(q[4 * w], __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.w[w], 1.f, 0), s, false);
      s = __builtin_amdgcn_fdot2_f32_bf16(q[4 * w + 1], __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.w[w], 1.f, 1), s, false);
      s = __builtin_amdgcn_fdot2_f32_bf16(q[4 * w + 2], __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.w[w], 1.f, 2), s, false);
      s = __builtin_amdgcn_fdot2_f32_bf16(q[4 * w + 3], __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.w[w], 1.f, 3), s, false);
    }
    return s;
  }
};

// A key's block sums under its scales, in block order
template <int N>
__device__ __forceinline__ float scaled_sum(const float* part, typename ScaleWord<N>::type s) {
  float a = 0.f;
#pragma unroll
  for (int b = 0; b < N; ++b) a = fmaf(part[b], fp4_factor(static_cast<uint32_t>(s >> (8 * b)) & 255u), a);
  return a;
}
// A key's share for each block of its V row
template <int N>
__device__ __forceinline__ void scaled_shares(float* dst, float share, typename ScaleWord<N>::type s) {
#pragma unroll
  for (int b = 0; b < N; ++b) dst[b] = share * fp4_factor(static_cast<uint32_t>(s >> (8 * b)) & 255u);
}

// acc += w times a lane's codes
template <int E>
__device__ __forceinline__ void add_codes(float (&acc)[E], float w, const CodeWords<E / 8>& c) {
#pragma unroll
  for (int i = 0; i < E / 8; ++i) {
    float v[8];
    fp4_values8(c.w[i], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[8 * i + e] = fmaf(w, v[e], acc[8 * i + e]);
  }
}

// The sums of v over the lanes that differ in the bits O and above: each step halves what a
// lane holds, so that lane l ends with the sums of its element `at` alone (N - 1 moves and the
// rest of the 6 - log2 O steps one each, where a sum element by element takes N moves a step).
template <int N, int O>
__device__ __forceinline__ void scatter_sums(float (&v)[N], int lane, int& at) {
  if constexpr (O < 64) {
    if constexpr (N > 1) {
      constexpr int H = N / 2;
      const bool up = lane & O;
      float h[H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float keep = up ? v[i + H] : v[i], send = up ? v[i] : v[i + H];
        h[i] = keep + __shfl_xor(send, O, 64);
      }
      at += up ? H : 0;
      scatter_sums<H, 2 * O>(h, lane, at);
#pragma unroll
      for (int i = 0; i < H; ++i) v[i] = h[i];
    } else {
      v[0] += __shfl_xor(v[0], O, 64);
      scatter_sums<1, 2 * O>(v, lane, at);
    }
  }
}
// How many elements a lane ends with
constexpr int scattered(int n, int o) {
  while (o < 64 && n > 1) {
    n /= 2;
    o *= 2;
  }
  return n;
}
// The workgroup's sums of share v, one row of D for each wave
template <int D, int E>
__device__ __forceinline__ void wave_sums(float (&acc)[E], int lane, float* row) {
  using L = QLayout<D, E>;
  int at = (lane % L::kLanesPerRow) * E;
  scatter_sums<E, L::kLanesPerRow>(acc, lane, at);
#pragma unroll
  for (int i = 0; i < scattered(E, L::kLanesPerRow); ++i) row[at + i] = acc[i];   // lanes with the same `at` hold the same sums
}

// The new token's rows into position `pos`: 32 lanes of the first wave each for K and V
template <int D>
__device__ __forceinline__ void append_rows(const Fp4DecodeArgs& A, int64_t slice, int64_t pos) {
  using F = Fp4Row<D>;
  const int t = threadIdx.x, c = t & 31;
  if (t >= 64 || c >= D / 8) return;
  const void* src = t < 32 ? A.k1 : A.v1;
  const Fp4Cache cache = t < 32 ? A.k_cache : A.v_cache;
  float x[8];
  load8_f32(src, slice * D + 8 * c, A.q_dtype, x);
  floatx8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
  const uint32_t s = fp4_scale(block_top<D>(top_bits<DT_F32>(r)));
  static_cast<uint32_t*>(cache.codes)[(slice * A.capacity + pos) * (D / 8) + c] = fp4_codes8<DT_F32>(r, s);
  if (c * 8 % F::kBlock == 0)
    static_cast<uint8_t*>(cache.scales)[(slice * A.capacity + pos) * F::kBlocks + c * 8 / F::kBlock] = static_cast<uint8_t>(s);
}

template <int D>
__device__ __forceinline__ const uint8_t* code_rows(const Fp4Cache& c, int64_t row) {
  return static_cast<const uint8_t*>(c.codes) + row * (D / 2);
}
template <int D>
__device__ __forceinline__ const typename ScaleWord<Fp4Row<D>::kBlocks>::type* scale_rows(const Fp4Cache& c, int64_t row) {
  return static_cast<const typename ScaleWord<Fp4Row<D>::kBlocks>::type*>(c.scales) + row;
}

// A slice's whole step in one workgroup; s: floats of LDS, one for each key and block.
template <int D, int QT>
__device__ __forceinline__ void fp4_one_slice(const Fp4DecodeArgs& A, int64_t slice, int live, float qscale, float* s) {
  constexpr int E = kQElems<D>, N = Fp4Row<D>::kBlocks;
  using L = QLayout<D, E>;
  __shared__ float sm[kQWaves], ss[kQWaves];
  __shared__ float red[kQWaves][D + 1];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, sub = lane % L::kLanesPerRow;
  const int64_t row0 = slice * A.capacity;
  float* crow = A.committed + row0;
  if (A.k1 != nullptr && live > 0) {
    append_rows<D>(A, slice, live - 1);
    __syncthreads();
  }
  const QueryPart<E, QT> q(A.q1, slice * D + sub * E, A.q_dtype);
  {
    CodeStream<D, E> k(code_rows<D>(A.k_cache, row0) + sub * (E / 2), wave, lane, live);
    k.load();
    k.walk([&](int j, const CodeWords<E / 8>& c) { s[j * N + sub] = q.dot(c); });
  }
  CodeStream<D, E> v(code_rows<D>(A.v_cache, row0) + sub * (E / 2), wave, lane, live);
  v.load();                                             // in flight over the reductions
  const auto* ks = scale_rows<D>(A.k_cache, row0);
  const auto* vs = scale_rows<D>(A.v_cache, row0);
  __syncthreads();
  float m = -INFINITY;
  for (int j = t; j < live; j += kQThreads) {
    const float a = qscale * scaled_sum<N>(s + j * N, ks[j]);
    s[j * N] = a;
    m = fmaxf(m, a);
  }
  const float wm = wave_max(m);
  if (lane == 0) sm[wave] = wm;
  __syncthreads();
  float M = sm[0];
#pragma unroll
  for (int w = 1; w < kQWaves; ++w) M = fmaxf(M, sm[w]);
  float l = 0.f;
  for (int j = t; j < live; j += kQThreads) l += fast_exp2(s[j * N] - M);
  l = wave_sum(l);
  if (lane == 0) ss[wave] = l;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int w = 0; w < kQWaves; ++w) tot += ss[w];
  const float lse = M + __log2f(tot);
  float ssum = 0.f;
  for (int j = t; j < live; j += kQThreads) {
    const float p = fast_exp2(s[j * N] - lse);
    const float cm = crow[j];
    const float sh = p * fast_rcp(cm + p + kEps);
    crow[j] = cm + p;
    scaled_shares<N>(s + j * N, sh, vs[j]);
    ssum += sh;
  }
  ssum = wave_sum(ssum);
  if (lane == 0) red[wave][D] = ssum;
  __syncthreads();
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  v.walk([&](int j, const CodeWords<E / 8>& c) { add_codes<E>(acc, s[j * N + sub], c); });
  wave_sums<D, E>(acc, lane, red[wave]);
  __syncthreads();
  if (t < D) {
    float x = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kQWaves; ++w) {
      x += red[w][t];
      sum += red[w][D];
    }
    store_as(A.out, slice * D + t, A.q_dtype, x / (sum + kEps));
  }
}

template <int D, int QT>
__global__ __launch_bounds__(kQThreads) void fp4_one(Fp4DecodeArgs A, float qscale, int64_t slice0) {
  extern __shared__ float one_s[];
  fp4_one_slice<D, QT>(A, slice0 + blockIdx.x, static_cast<int>(live_length(A.dlen, A.length)), qscale, one_s);
}

// ONE: a device-resident length that may be short: one workgroup a slice then does the whole
// step, as in dec_stats.
template <int D, int QT, bool ONE>
__global__ __launch_bounds__(kQThreads) void fp4_stats(Fp4DecodeArgs A, float* __restrict__ aff, float2* __restrict__ part,
                                                       int64_t chunk, int nchunk, float qscale, int64_t slice0,
                                                       int64_t one_max) {
  constexpr int E = kQElems<D>, N = Fp4Row<D>::kBlocks;
  using L = QLayout<D, E>;
  const int64_t live = live_length(A.dlen, A.length);
  if constexpr (ONE) {
    extern __shared__ float one_s[];
    if (live <= one_max) {
      const unsigned block = blockIdx.y * gridDim.x + blockIdx.x;
      if (block < gridDim.y) fp4_one_slice<D, QT>(A, slice0 + block, static_cast<int>(live), qscale, one_s);
      return;
    }
  }
  const int64_t slice = slice0 + blockIdx.y;
  const int c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % L::kLanesPerRow;
  if (A.dlen != nullptr) chunk = decode_chunk(A.n, live);
  const int nlive = live_chunks(live, chunk);
  if (c >= nlive) return;
  const int64_t j0 = c * chunk, row0 = slice * A.capacity + j0;
  const int count = static_cast<int>(min(j0 + chunk, live) - j0);
  if (A.k1 != nullptr && c == nlive - 1) {
    append_rows<D>(A, slice, live - 1);
    __syncthreads();
  }
  CodeStream<D, E> k(code_rows<D>(A.k_cache, row0) + sub * (E / 2), wave, lane, count);
  k.load();
  const QueryPart<E, QT> q(A.q1, slice * D + sub * E, A.q_dtype);
  __shared__ float s[kDecMaxChunk * N];
  k.walk([&](int j, const CodeWords<E / 8>& w) { s[j * N + sub] = q.dot(w); });
  const auto* ks = scale_rows<D>(A.k_cache, row0);
  __syncthreads();
  float* arow = aff + slice * A.length + j0;
  float m = -INFINITY, l = 0.f;
  bool bad = false;
  for (int j = threadIdx.x; j < count; j += kQThreads) {
    const float a = qscale * scaled_sum<N>(s + j * N, ks[j]);
    arow[j] = a;
    bad |= a != a;
    const float mn = fmaxf(m, a);
    if (mn > -INFINITY) {
      l = l * fast_exp2(m - mn) + fast_exp2(a - mn);
      m = mn;
    }
  }
  const float wm = wave_max(m);
  float ws = wave_sum(bad ? NAN : m == -INFINITY ? 0.f : l * fast_exp2(m - wm));
  __shared__ float sm[kQWaves], ss[kQWaves];
  if (lane == 0) { sm[wave] = wm; ss[wave] = ws; }
  __syncthreads();
  if (threadIdx.x == 0) {
    float bm = -INFINITY, bs = 0.f;
    for (int w = 0; w < kQWaves; ++w) bm = fmaxf(bm, sm[w]);
    // a wave of NaN alone has no maximum, and its sum makes the slice's NaN
    for (int w = 0; w < kQWaves; ++w) bs += sm[w] > -INFINITY ? ss[w] * fast_exp2(sm[w] - bm) : ss[w];
    part[slice * nchunk + c] = make_float2(bm, bs);
  }
}

template <int D>
__global__ __launch_bounds__(kQThreads) void fp4_apply(Fp4DecodeArgs A, const float* __restrict__ aff,
                                                       const float2* __restrict__ part, float* __restrict__ part_out,
                                                       int64_t chunk, int nchunk, int64_t slice0, int64_t one_max) {
  constexpr int E = kQElems<D>, N = Fp4Row<D>::kBlocks;
  using L = QLayout<D, E>;
  const int64_t live = live_length(A.dlen, A.length);
  if (live <= one_max) return;                            // fp4_stats did the whole step
  const int64_t slice = slice0 + blockIdx.y;
  const int c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % L::kLanesPerRow;
  if (A.dlen != nullptr) chunk = decode_chunk(A.n, live);
  const int nlive = live_chunks(live, chunk);
  if (c >= nlive) return;
  const int64_t j0 = c * chunk, row0 = slice * A.capacity + j0;
  const int count = static_cast<int>(min(j0 + chunk, live) - j0);
  const float* arow = aff + slice * A.length + j0;
  float* crow = A.committed + row0;
  const auto* vs = scale_rows<D>(A.v_cache, row0);
  CodeStream<D, E> v(code_rows<D>(A.v_cache, row0) + sub * (E / 2), wave, lane, count);
  v.load();
  // this thread's keys, which do not wait for the statistics
  constexpr int kOwn = static_cast<int>(kDecMaxChunk / kQThreads);
  float av[kOwn], cv[kOwn];
  typename ScaleWord<N>::type sv[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int j = min(static_cast<int>(threadIdx.x) + u * kQThreads, count - 1);
    av[u] = arow[j];
    cv[u] = crow[j];
    sv[u] = vs[j];
  }
  // the slice's statistics from its chunks' (every wave by itself)
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < nlive; i += 64) {
    const float2 ps = part[slice * nchunk + i];
    const float mn = fmaxf(m, ps.x);
    l = (m > -INFINITY ? l * fast_exp2(m - mn) : l) + (ps.x > -INFINITY ? ps.y * fast_exp2(ps.x - mn) : ps.y);
    m = mn;
  }
  const float gm = wave_max(m);
  const float gs = wave_sum(m > -INFINITY ? l * fast_exp2(m - gm) : l);
  const float lse = gm + __log2f(gs);

  __shared__ float s[kDecMaxChunk * N];
  __shared__ float red[kQWaves][D + 1];
  float ssum = 0.f;
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int j = threadIdx.x + u * kQThreads;
    if (j >= count) break;
    const float p = fast_exp2(av[u] - lse);
    const float sh = p * fast_rcp(cv[u] + p + kEps);
    crow[j] = cv[u] + p;
    scaled_shares<N>(s + j * N, sh, sv[u]);
    ssum += sh;
  }
  ssum = wave_sum(ssum);
  if (lane == 0) red[wave][D] = ssum;
  __syncthreads();
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  v.walk([&](int j, const CodeWords<E / 8>& w) { add_codes<E>(acc, s[j * N + sub], w); });
  wave_sums<D, E>(acc, lane, red[wave]);
  __syncthreads();
  for (int i = threadIdx.x; i <= D; i += kQThreads) {
    float x = 0.f;
    for (int w = 0; w < kQWaves; ++w) x += red[w][i];
    part_out[(slice * nchunk + c) * (D + 1) + i] = x;
  }
}

// The most keys of a slice that one workgroup takes whole: an LDS float for each key and block.
template <int D>
int64_t fp4_one_max(int64_t n) {
  constexpr int64_t kKeyBytes = D + 2 * Fp4Row<D>::kBlocks + 8, kMost = 16384 / Fp4Row<D>::kBlocks;
  if (n >= 160) return kMost;
  const int64_t keys = ((272 + 3 * n) << 10) / kKeyBytes;
  return keys < 4096 ? (keys < kMost ? keys : kMost) : (4096 < kMost ? 4096 : kMost);
}

struct Fp4Scratch {
  size_t part, part_out, total;
  Fp4Scratch(int64_t n, int64_t length, int head_dim, int64_t nchunk) {
    part = align_up(sizeof(float) * n * length);
    part_out = part + align_up(sizeof(float2) * n * nchunk);
    total = part_out + align_up(sizeof(float) * n * nchunk * (head_dim + 1));
  }
};

template <int D, int QT>
int launch_fp4(const Fp4DecodeArgs& a) {
  const int64_t chunk = decode_chunk(a.n, a.length);
  const int nchunk = static_cast<int>(decode_chunks(a.n, a.length, a.dlen != nullptr));
  const float qscale = kLog2e / sqrtf(static_cast<float>(D));
  constexpr int N = Fp4Row<D>::kBlocks;
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int64_t keys = fp4_one_max<D>(a.n);
  const auto lds_of = [](int64_t k) { return sizeof(float) * static_cast<size_t>((k + 63) / 64 * 64 * N); };
  if (a.length <= keys) {
    slice_batches(a.n, [&](int64_t s0, unsigned ns) {
      DIL_TIMED("fp4_one", st, (fp4_one<D, QT><<<dim3(ns), kQThreads, lds_of(a.length), st>>>(a, qscale, s0)));
    });
    return static_cast<int>(hipGetLastError());
  }
  const int64_t one_max = a.dlen != nullptr ? keys : -1;
  const Fp4Scratch w(a.n, a.length, D, nchunk);
  char* ws = static_cast<char*>(a.workspace);
  float* aff = reinterpret_cast<float*>(ws);
  float2* part = reinterpret_cast<float2*>(ws + w.part);
  float* part_out = reinterpret_cast<float*>(ws + w.part_out);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    const dim3 grid(nchunk, ns);
    if (one_max >= 0)
      DIL_TIMED("fp4_stats", st,
                (fp4_stats<D, QT, true><<<grid, kQThreads, lds_of(one_max), st>>>(a, aff, part, chunk, nchunk, qscale, s0, one_max)));
    else
      DIL_TIMED("fp4_stats", st,
                (fp4_stats<D, QT, false><<<grid, kQThreads, 0, st>>>(a, aff, part, chunk, nchunk, qscale, s0, one_max)));
  });
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    DIL_TIMED("fp4_apply", st,
              (fp4_apply<D><<<dim3(nchunk, ns), kQThreads, 0, st>>>(a, aff, part, part_out, chunk, nchunk, s0, one_max)));
  });
  DIL_TIMED("fp4_finish", st,
            (dec_finish<D><<<dim3(static_cast<unsigned>(a.n)), kFinishThreads, 0, st>>>(part_out, nchunk, a.out, D, a.q_dtype,
                                                                                      a.length, chunk, a.dlen, one_max)));
  return static_cast<int>(hipGetLastError());
}

template <int D>
int decode_fp4_type(const Fp4DecodeArgs& a) {
  return a.q_dtype == DT_BF16 ? launch_fp4<D, DT_BF16>(a) : launch_fp4<D, DT_F32>(a);
}

}  // namespace

// Sized for a device-resident length up to `length`, as the decode step's.
int64_t decode_fp4_workspace_bytes(int64_t n, int64_t length, int head_dim) {
  if (n < 1 || length < 1) return 0;
  return static_cast<int64_t>(Fp4Scratch(n, length, head_dim, decode_chunks(n, length, true)).total);
}

int decode_fp4(const Fp4DecodeArgs& a) {
  switch (a.head_dim) {
    case 16: return decode_fp4_type<16>(a);
    case 32: return decode_fp4_type<32>(a);
    case 64: return decode_fp4_type<64>(a);
    case 128: return decode_fp4_type<128>(a);
    case 256: return decode_fp4_type<256>(a);
    default: return kErrHeadDim;
  }
}

}  // namespace dil
