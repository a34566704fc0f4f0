// Attention for a tree of drafted tokens over a decode cache, and the acceptance
// of one of its paths (include/dilution_hip.h: dil_tree_step, dil_tree_accept).
//
// A node's share of a key is p / (committed + the ancestors' p + p + eps): not
// linear in p, so the row statistics have to be known before any share.  Launches:
//
//   tree_stats  (chunks x slices)  per chunk and node: max and sum 2^(a - max)
//   tree_lse    (slices)           the chunks' statistics joined: lse
//   tree_apply  (chunks x slices)  one key per thread, the nodes in order: the
//                                  demand goes down the tree through LDS; partial
//                                  sums of the shares and of share V
//   tree_finish (nodes x slices)   the chunks' partials added
//
// and for the acceptance
//
//   tree_accept (chunks + 1 x slices)  the demand of the cached keys; the last
//                                      workgroup moves the drafted rows
#include "dil_common.hpp"
#include "dil_internal.hpp"

namespace dil {
namespace {

constexpr int kTreeThreads = 256;
constexpr int kTreeKeys = 256;                 // keys per workgroup, one a thread

template <int DT>
__device__ __forceinline__ float elem(const void* p, int64_t i) {
  if constexpr (DT == DT_F32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == DT_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(x), lane, 64), hi = __shfl(static_cast<uint32_t>(x >> 32), lane, 64);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// One lane per node (a whole wave calls): the nodes that node `lane` sees among
// the drafted (its ancestors and itself, as bits), 0 for an absent one.  The
// chains of parents are followed in 6 doubling steps (64 nodes).
__device__ __forceinline__ uint64_t nodes_seen(const int32_t* parents, int nodes, int lane) {
  const int par = lane < nodes ? parents[lane] : -2;
  int absent = par < -1 || par >= lane;
  int jump = absent || par < 0 ? lane : par;
  uint64_t seen = uint64_t{1} << lane;
#pragma unroll
  for (int step = 0; step < 6; ++step) {
    seen |= shfl64(seen, jump);
    absent |= __shfl(absent, jump, 64);
    jump = __shfl(jump, jump, 64);
  }
  return absent ? 0 : seen;
}

struct Tree {
  const void* q;
  RowsView qv;
  const void* k;
  const void* v;
  int64_t cap;
  const float* committed;
  int64_t length;
  int nodes;
  const int32_t* parents;
  int64_t parents_sb;
  int64_t heads;
  void* out;
  RowsView ov;
  float* lse;
  float2* part;
  float* part_out;
  int nchunk;
  float scale;
  int64_t slice0;
};

// a_ij of the drafted node in q_s against key row j (from memory)
template <int D, int DT>
__device__ __forceinline__ float score(const float* q_s, const void* k, int64_t row) {
  float s = 0.f;
  for (int d = 0; d < D; ++d) s = fmaf(q_s[d], elem<DT>(k, row + d), s);
  return s;
}

template <int D, int DT>
__global__ __launch_bounds__(kTreeThreads) void tree_stats(Tree A) {
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  __shared__ float q_s[D];
  __shared__ uint64_t seen_s[kTreeMaxNodes];
  __shared__ float sm[4], sl[4];
  if (wave == 0) seen_s[lane] = nodes_seen(A.parents + slice / A.heads * A.parents_sb, A.nodes, lane);
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kTreeKeys + t, end = A.length + A.nodes;
  const int64_t row = (slice * A.cap + (j < end ? j : end - 1)) * D;
  const int64_t qbase = A.qv.slice(slice);
  for (int i = 0; i < A.nodes; ++i) {
    __syncthreads();
    for (int d = t; d < D; d += kTreeThreads) q_s[d] = elem<DT>(A.q, qbase + i * A.qv.sr + d) * A.scale;
    __syncthreads();
    const uint64_t seen = seen_s[i];
    const bool on = seen != 0 && j < end && (j < A.length || (seen >> (j - A.length) & 1));
    const float a = on ? score<D, DT>(q_s, A.k, row) : -INFINITY;
    const float m = wave_max(a);
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float l = wave_sum(on ? exp2f(a - mm) : 0.f);
    if (lane == 0) sl[wave] = l;
    __syncthreads();
    if (t == 0)
      A.part[(slice * A.nchunk + blockIdx.x) * A.nodes + i] = make_float2(mm, sl[0] + sl[1] + sl[2] + sl[3]);
  }
}

__global__ void tree_lse(Tree A) {
  const int64_t slice = A.slice0 + blockIdx.x;
  const int i = threadIdx.x;
  const uint64_t seen = nodes_seen(A.parents + slice / A.heads * A.parents_sb, A.nodes, i);
  if (i >= A.nodes) return;
  float m = -INFINITY, l = 0.f;
  for (int c = 0; c < A.nchunk; ++c) {
    const float2 p = A.part[(slice * A.nchunk + c) * A.nodes + i];
    const float mn = fmaxf(m, p.x);
    if (p.y != 0.f || p.y != p.y) {
      l = l * exp2f(m - mn) + p.y * exp2f(p.x - mn);
      m = mn;
    }
  }
  A.lse[slice * A.nodes + i] = seen != 0 ? m + log2f(l) : INFINITY;
}

template <int D, int DT>
__global__ __launch_bounds__(kTreeThreads) void tree_apply(Tree A) {
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  __shared__ float q_s[D], sh_s[kTreeKeys], ss[4];
  __shared__ uint64_t seen_s[kTreeMaxNodes];
  __shared__ float t_s[kTreeMaxNodes][kTreeKeys];
  const int32_t* parents = A.parents + slice / A.heads * A.parents_sb;
  if (wave == 0) seen_s[lane] = nodes_seen(parents, A.nodes, lane);
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * kTreeKeys, j = j0 + t, end = A.length + A.nodes;
  const int64_t row = (slice * A.cap + (j < end ? j : end - 1)) * D;
  const float com = j < A.length ? A.committed[slice * A.cap + j] : 0.f;
  const int64_t qbase = A.qv.slice(slice);
  const int count = static_cast<int>(end - j0 < kTreeKeys ? end - j0 : kTreeKeys);
  for (int i = 0; i < A.nodes; ++i) {
    __syncthreads();
    for (int d = t; d < D; d += kTreeThreads) q_s[d] = elem<DT>(A.q, qbase + i * A.qv.sr + d) * A.scale;
    __syncthreads();
    const uint64_t seen = seen_s[i];
    float* po = A.part_out + ((slice * A.nchunk + blockIdx.x) * A.nodes + i) * (D + 1);
    if (seen == 0) continue;                       // the whole workgroup: an absent node
    const bool on = j < end && (j < A.length || (seen >> (j - A.length) & 1));
    const float p = on ? exp2f(score<D, DT>(q_s, A.k, row) - A.lse[slice * A.nodes + i]) : 0.f;
    const int par = parents[i];
    const float tot = (par < 0 ? com : t_s[par][t]) + p;
    t_s[i][t] = tot;
    const float sh = on ? p / (tot + kEps) : 0.f;
    sh_s[t] = on ? sh : -1.f;                      // -1: a key that the node does not see
    const float s = wave_sum(sh);
    if (lane == 0) ss[wave] = s;
    __syncthreads();
    for (int d = t; d < D; d += kTreeThreads) {
      float x = 0.f;
      for (int c = 0; c < count; ++c)
        if (!(sh_s[c] < 0.f)) x = fmaf(sh_s[c], elem<DT>(A.v, (slice * A.cap + j0 + c) * D + d), x);
      po[d] = x;
    }
    if (t == 0) po[D] = ss[0] + ss[1] + ss[2] + ss[3];
  }
}

template <int D, int DT>
__global__ void tree_finish(Tree A) {
  const int64_t slice = A.slice0 + blockIdx.y;
  const int i = blockIdx.x, d = threadIdx.x;
  const uint64_t seen = nodes_seen(A.parents + slice / A.heads * A.parents_sb, A.nodes, d & 63);
  const int here = __shfl(seen != 0, i, 64);
  if (d >= D) return;
  float x = 0.f, s = 0.f;
  if (here) {
    for (int c = 0; c < A.nchunk; ++c) {
      const float* po = A.part_out + ((slice * A.nchunk + c) * A.nodes + i) * (D + 1);
      x += po[d];
      s += po[D];
    }
    x /= s + kEps;
  }
  store_as(A.out, A.ov.slice(slice) + i * A.ov.sr + d, DT, x);
}

template <int D, int DT>
__global__ __launch_bounds__(kTreeThreads) void tree_accept_kernel(Tree A, float* committed, void* kc, void* vc,
                                                                   const int32_t* path, int64_t path_sb, int count) {
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x;
  __shared__ float q_s[D];
  const int32_t* pr = path + slice / A.heads * path_sb;
  const int64_t qbase = A.qv.slice(slice);
  float* crow = committed + slice * A.cap;
  auto stage = [&](int a) {
    __syncthreads();
    for (int d = t; d < D; d += kTreeThreads) q_s[d] = elem<DT>(A.q, qbase + a * A.qv.sr + d) * A.scale;
    __syncthreads();
  };
  const bool tail = blockIdx.x == static_cast<unsigned>(A.nchunk);
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kTreeKeys + t;
  const int mine = tail && t < count ? pr[t] : -1;
  const bool drafted = mine >= 0 && mine < A.nodes, cached = !tail && j < A.length;
  const int64_t row = (slice * A.cap + (tail ? A.length + (drafted ? mine : 0) : (cached ? j : A.length))) * D;
  float sum = cached ? crow[j] : 0.f;
  for (int r = 0; r < count; ++r) {
    const int a = pr[r];
    if (a < 0 || a >= A.nodes) continue;
    stage(a);
    if (cached || (drafted && r >= t)) sum += exp2f(score<D, DT>(q_s, A.k, row) - A.lse[slice * A.nodes + a]);
  }
  if (cached) crow[j] = sum;
  if (!tail) return;
  if (t < count) crow[A.length + t] = sum;
  // the rows: all into LDS, then to their places
  __shared__ uint32_t rows_s[kTreeMaxNodes * 32];
  constexpr int kWords = D * (DT == DT_F32 ? 4 : 2) / 4, kStep = kWords < 32 ? kWords : 32;
  for (int w0 = 0; w0 < kWords; w0 += kStep) {
    for (void* cache : {kc, vc}) {
      uint32_t* base = static_cast<uint32_t*>(cache) + (slice * A.cap + A.length) * kWords + w0;
      __syncthreads();
      for (int u = t; u < count * kStep; u += kTreeThreads) {
        const int a = pr[u / kStep];
        if (a >= 0 && a < A.nodes) rows_s[u] = base[static_cast<int64_t>(a) * kWords + u % kStep];
      }
      __syncthreads();
      for (int u = t; u < count * kStep; u += kTreeThreads) {
        const int a = pr[u / kStep];
        if (a >= 0 && a < A.nodes) base[static_cast<int64_t>(u / kStep) * kWords + u % kStep] = rows_s[u];
      }
    }
  }
}

int64_t tree_chunks(int64_t length, int64_t nodes) { return (length + nodes + kTreeKeys - 1) / kTreeKeys; }

Tree tree_of(const TreeArgs& a) {
  Tree A{};
  A.q = a.q;
  A.qv = a.qv;
  A.k = a.k_cache;
  A.v = a.v_cache;
  A.cap = a.cap;
  A.committed = a.committed;
  A.length = a.length;
  A.nodes = a.nodes;
  A.parents = a.parents;
  A.parents_sb = a.parents_sb;
  A.heads = a.heads;
  A.out = a.out;
  A.ov = a.ov;
  A.lse = a.lse;
  A.scale = kLog2e / sqrtf(static_cast<float>(a.head_dim));
  return A;
}

template <int D, int DT>
int launch_step(const TreeArgs& a) {
  Tree A = tree_of(a);
  A.nchunk = static_cast<int>(tree_chunks(a.length, a.nodes));
  A.part = static_cast<float2*>(a.workspace);
  A.part_out = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + align_up(sizeof(float2) * a.n * A.nchunk * a.nodes));
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    A.slice0 = s0;
    DIL_TIMED("tree_stats", st, (tree_stats<D, DT><<<dim3(A.nchunk, ns), kTreeThreads, 0, st>>>(A)));
    DIL_TIMED("tree_lse", st, (tree_lse<<<dim3(ns), 64, 0, st>>>(A)));
    DIL_TIMED("tree_apply", st, (tree_apply<D, DT><<<dim3(A.nchunk, ns), kTreeThreads, 0, st>>>(A)));
    DIL_TIMED("tree_finish", st, (tree_finish<D, DT><<<dim3(A.nodes, ns), D < 64 ? 64 : D, 0, st>>>(A)));
  });
  return static_cast<int>(hipGetLastError());
}

template <int D, int DT>
int launch_accept(const TreeArgs& a) {
  Tree A = tree_of(a);
  A.nchunk = static_cast<int>((a.length + kTreeKeys - 1) / kTreeKeys);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    A.slice0 = s0;
    DIL_TIMED("tree_accept", st,
              (tree_accept_kernel<D, DT><<<dim3(A.nchunk + 1, ns), kTreeThreads, 0, st>>>(A, a.committed, a.k_cache, a.v_cache,
                                                                                a.path, a.path_sb, a.count)));
  });
  return static_cast<int>(hipGetLastError());
}

// f(head dim, dtype) as integral constants
template <typename F>
int with_shape(int head_dim, int dtype, F&& f) {
  auto by_dtype = [&](auto d) {
    switch (dtype) {
      case DT_F32: return f(d, std::integral_constant<int, DT_F32>{});
      case DT_BF16: return f(d, std::integral_constant<int, DT_BF16>{});
      case DT_F16: return f(d, std::integral_constant<int, DT_F16>{});
      default: return kErrDtype;
    }
  };
  switch (head_dim) {
    case 16: return by_dtype(std::integral_constant<int, 16>{});
    case 32: return by_dtype(std::integral_constant<int, 32>{});
    case 64: return by_dtype(std::integral_constant<int, 64>{});
    case 128: return by_dtype(std::integral_constant<int, 128>{});
    case 256: return by_dtype(std::integral_constant<int, 256>{});
    default: return kErrHeadDim;
  }
}

}  // namespace

int64_t tree_workspace_bytes(int64_t n, int64_t length, int64_t nodes, int head_dim, int dtype) {
  const int64_t nchunk = tree_chunks(length, nodes);
  return static_cast<int64_t>(align_up(sizeof(float2) * n * nchunk * nodes) +
                              align_up(sizeof(float) * n * nchunk * nodes * (head_dim + 1)));
}

int tree_step(const TreeArgs& a) {
  return with_shape(a.head_dim, a.dtype, [&](auto d, auto t) { return launch_step<d(), t()>(a); });
}

int tree_accept(const TreeArgs& a) {
  return with_shape(a.head_dim, a.dtype, [&](auto d, auto t) { return launch_accept<d(), t()>(a); });
}

}  // namespace dil
