// Attention for a tree of drafted tokens over a decode cache, and the acceptance
// of one of its paths (include/dilution_hip.h: dil_tree_step, dil_tree_accept).
//
// For node i and key j, with anc(i) the ancestors of i among the drafted nodes:
//   a_ij = log2(e) / sqrt(D) q_i.k_j      lse_i = log2 sum_j 2^a_ij
//   p_ij = 2^(a_ij - lse_i)               t_ij  = committed_j + sum_{a in anc(i)} p_aj
//   share = p / (t + p + eps)             out_i = sum_j share v_j / (sum_j share + eps)
// A share is not linear in p, so lse has to be known first and K is read twice:
//
//   tree_stats   per chunk of keys and node: max and sum 2^(a - max)
//   tree_apply   joins the chunks' statistics; per chunk and node: the sums of
//                share and of share v
//   tree_finish  joins the chunks' sums
//                (short or many slices: tree_apply alone, a workgroup per slice)
//   tree_demand  the acceptance: committed_j += sum of the accepted nodes' p_ij
//
// The cached keys go through matrix instructions in tiles of 32 keys x 32 nodes
// (one or two node tiles), a wave per tile with no barrier and no LDS traffic but
// the queries.  tree_apply's chain keeps every intermediate in the accumulators:
//   1  S = Q K^T with the nodes as rows, permuted so that a lane (one key) holds
//      runs of 8 consecutive nodes: p = 2^(S - lse) is then the A operand of
//   2  t^T = P^T seen^T and p^T = P^T 1 (seen: the 0/1 matrix of a node's ancestors
//      and itself), which sum the demand down the tree for all nodes at once and
//      leave a lane one node and 16 keys.  committed + eps is the accumulator's
//      start value.
//   3  the shares, in place, are the B operand of out^T += V^T share^T (of a 16-bit
//      type in two parts), whose A operand takes V rows as loaded, two head dims a
//      register, regrouped by byte permutes.
// The drafted keys (at most 64) are a workgroup of their own: there the masks are, and
// what a node does not see it must not touch (NaN included), so their shares are
// summed in plain fp32.
// A node whose own row statistics are NaN would spoil the others in step 2: its
// bids are taken as 0 there, and tree_finish makes it and the nodes below it NaN.
#include "dil_tiles.hpp"

namespace dil {
namespace {

constexpr int kTreeThreads = 256;
constexpr int kTreeWaves = kTreeThreads / 64;
constexpr int kTileNodes = 32;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// fp16 shares are scaled by 2^14: shares lie in [0, 1], those of a long context
// near 1e-5 and below, under fp16's smallest normal number.
template <int DT> constexpr float kShareScale = DT == DT_F16 ? 16384.f : 1.f;

// One 16-byte piece of a row per lane (lane half h holds the h-th 16 bytes of each
// 32): 8 elements of a 16-bit type, one instruction; 4 fp32, four instructions.
template <int DT>
__device__ __forceinline__ floatx16 mma_piece(u32x4 a, u32x4 b, floatx16 c) {
  if constexpr (DT == DT_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == DT_F16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, hi}, bf16x2));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, hi}, f16x2));
}

// Two shares as the operands of step 3, each in two parts of the 16-bit type: with one
// alone they would be rounded to 8 (bf16) or 11 bits before V, an error of the size of
// the outputs' own rounding; with two it is 2^-17 or less.  A call of 128 slices of
// 65536 keys and 64 nodes takes 688 us with two parts and 635 with one; with one node
// tile the times are within 1%.
template <int DT>
__device__ __forceinline__ u32x2 split_shares(float x, float y) {
  if constexpr (DT == DT_BF16) {
    const uint32_t hi = pack_bf16(x, y);
    return {hi, pack_bf16(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u))};
  } else {
    const uint32_t hi = pack_f16(x, y);
    const f16x2 h = __builtin_bit_cast(f16x2, hi);
    return {hi, pack_f16(x - static_cast<float>(h[0]), y - static_cast<float>(h[1]))};
  }
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
  float2* part;              // (n, nstat + 1, nodes): entry 0 of a slice is the drafted keys'
  float* part_out;           // (n, nchunk + 1, nodes, D)
  float* part_sum;           // (n, nchunk + 1, nodes)
  float* aff;                // (n, nodes, nodes): the drafted keys' affinities
  uint64_t* seen;            // (n, 64): nodes_seen, for the launches after the first
  int nstat, nchunk;         // workgroups of a slice over its cached keys: the statistics, and the shares (or the acceptance)
  float scale;
  int64_t slice0;
  // the acceptance
  float* demand;
  void* k_move;
  void* v_move;
  const int32_t* path;
  int64_t path_sb;
  int count;
};

template <int D, int DT>
struct Shape {
  static constexpr int kElt = DT == DT_F32 ? 4 : 2;
  static constexpr int kRow = D * kElt;            // bytes
  static constexpr int kPieces = kRow / 32;        // per lane half
};

// The queries of up to NT * 32 rows in LDS, as pieces: [tile][piece][half][row].
// row_of(r): the node of row r, or -1 for a row of zeros.
template <int D, int DT, int NT, typename F>
__device__ __forceinline__ void stage_queries(u32x4* q_s, const Tree& A, int64_t slice, F&& row_of) {
  using S = Shape<D, DT>;
  constexpr int kUnits = S::kRow / 16;
  const char* base = static_cast<const char*>(A.q) + A.qv.slice(slice) * S::kElt;
  for (int u = threadIdx.x; u < NT * kTileNodes * kUnits; u += kTreeThreads) {
    const int r = u / kUnits, c = u % kUnits, node = row_of(r);
    u32x4 x = {0, 0, 0, 0};
    if (node >= 0) x = *reinterpret_cast<const u32x4*>(base + node * A.qv.sr * S::kElt + c * 16);
    q_s[(((r >> 5) * S::kPieces + (c >> 1)) * 2 + (c & 1)) * kTileNodes + (r & 31)] = x;
  }
}

// Workgroup c of a slice's `chunks` takes the blocks of 128 rows c, c + chunks, ...,
// its waves 32 rows each, all uniform in a wave: the workgroups' shares differ by one
// block at most, and no resource spans more than 32 rows, whatever the length.  (A
// stretch of its own for every workgroup takes the same time.)
constexpr int kBlockRows = kTreeWaves * 32;

// An address that is the same in every lane, in scalar registers.
__device__ __forceinline__ void* uniform(const void* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return reinterpret_cast<void*>((static_cast<uint64_t>(hi) << 32) | lo);
}

// The resource over the 32 rows from `row` on, as far as they exist: rows past the end
// read 0.  Offsets within it are per lane alone, which the range check covers.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const char* base, int64_t row, int64_t length, int rowbytes) {
  const int64_t left = length - row;
  const int n = left < 0 ? 0 : left < 32 ? static_cast<int>(left) : 32;
  return __builtin_amdgcn_make_buffer_rsrc(uniform(base + row * rowbytes), 0,
                                           __builtin_amdgcn_readfirstlane(n * rowbytes), 0x00020000);
}

// The constants that a load adds to `off` stay with the load, as its immediate offset:
// hoisted out of the loop over `row` each of them is a register.
__device__ __forceinline__ void keep_in_loop(uint32_t& off, int64_t row) { asm("" : "+v"(off) : "s"(row)); }

// Loads issued before this stay before it (everything but vector memory may cross):
// the next tile's go out here, not where they are used.
__device__ __forceinline__ void loads_go_out() { __builtin_amdgcn_sched_barrier(0x78F); }

// 32 rows, one per lane (l & 31).
template <int D, int DT>
struct KeyRows {
  u32x4 p[Shape<D, DT>::kPieces];
  __device__ __forceinline__ void load(const char* base, int64_t row, int64_t length, int lane) {
    load(rows_at(base, row, length, Shape<D, DT>::kRow), row, lane, lane & 31);
  }
  // the rows `mine` of the lanes among `rows` (at most 64) at base; none where negative
  __device__ __forceinline__ void gather(const char* base, int rows, int lane, int mine) {
    load(__builtin_amdgcn_make_buffer_rsrc(uniform(base), 0, rows * Shape<D, DT>::kRow, 0x00020000), 0, lane, mine);
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int64_t row, int lane, int mine) {
    uint32_t off = mine < 0 ? 0xf0000000u : static_cast<uint32_t>(mine) * Shape<D, DT>::kRow + (lane >> 5) * 16u;
    keep_in_loop(off, row);
#pragma unroll
    for (int g = 0; g < Shape<D, DT>::kPieces; ++g)
      p[g] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 32u * g, 0, 0));
  }
};

// 32 V rows as A operands of V^T: lane (d, h) of instruction step s, slot t holds key
// 16 s + 8 (t >> 2) + 4 h + (t & 3) (fp32: register i, key acc_row(i, h)).  A lane
// loads E = DV / 32 consecutive head dims of a row: row u of operand tile e is head
// dim E * u + e.  Read once, past the caches (the K rows of the pass before stay there:
// 8% of tree_apply at 128 slices of 16384 keys).
constexpr int kOnce = 2;                               // the non-temporal hint of a buffer load
template <int DV, int DT>
struct ValueRows {
  static constexpr int E = DV < 32 ? 1 : DV / 32;
  static constexpr int kBytes = E * (DT == DT_F32 ? 4 : 2);   // per lane and row: 2 to 32
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[16][kWords];
  __device__ __forceinline__ void load(const char* base, int64_t row, int64_t length, int lane, int rowbytes, int d0bytes) {
    const __amdgpu_buffer_rsrc_t r = rows_at(base, row, length, rowbytes);
    const int l32 = lane & 31, h = lane >> 5;
    uint32_t off = static_cast<uint32_t>(4 * h) * rowbytes + d0bytes + l32 * kBytes;
    if constexpr (DV < 32) {
      if (l32 >= DV) off = 0xf0000000u;              // past the end: zeros
    }
    keep_in_loop(off, row);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t o = off + static_cast<uint32_t>(8 * (i >> 2) + (i & 3)) * rowbytes;
      if constexpr (kBytes == 2) {
        w[i][0] = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, kOnce);
      } else if constexpr (kBytes == 4) {
        w[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, kOnce);
      } else if constexpr (kBytes == 8) {
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, kOnce));
        w[i][0] = x[0];
        w[i][1] = x[1];
      } else {
#pragma unroll
        for (int c = 0; c < kBytes / 16; ++c) {
          const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, o + 16u * c, 0, kOnce));
#pragma unroll
          for (int e = 0; e < 4; ++e) w[i][4 * c + e] = x[e];
        }
      }
    }
  }
  // 16-bit types: operand tile e, step s
  __device__ __forceinline__ u32x4 frag(int e, int s) const {
    u32x4 f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t lo = w[8 * s + 2 * t][e / 2], hi = w[8 * s + 2 * t + 1][e / 2];
      f[t] = __builtin_amdgcn_perm(hi, lo, e & 1 ? 0x07060302u : 0x05040100u);
    }
    return f;
  }
};

// ---------------------------------------------------------------------------
// the drafted keys

constexpr int kShareStride = kTreeMaxNodes + 4;         // floats: 16-byte rows, a column on 16 banks

// Sum over the wave in every lane, by lane moves of the vector unit (a shuffle through
// LDS takes about ten times as long).
__device__ __forceinline__ float wave_sum_dpp(float x) {
  auto moved = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  x += moved(x, std::integral_constant<int, 0xB1>{});    // quad_perm [1, 0, 3, 2]
  x += moved(x, std::integral_constant<int, 0x4E>{});    // quad_perm [2, 3, 0, 1]
  x += moved(x, std::integral_constant<int, 0x141>{});   // row_half_mirror
  x += moved(x, std::integral_constant<int, 0x140>{});   // row_mirror
  const int b = __float_as_int(x);
  return (__int_as_float(__builtin_amdgcn_readlane(b, 0)) + __int_as_float(__builtin_amdgcn_readlane(b, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(b, 32)) + __int_as_float(__builtin_amdgcn_readlane(b, 48)));
}

// Shares of the drafted keys and their part of the outputs, from the affinities that
// tree_stats left.  Wave w holds the nodes i = w + 4 u in registers, a lane one key;
// the demand goes down the chains by doubling (after k rounds a pair holds the bids
// of 2^k nodes of the chain).  What a node does not see enters as 0, and where a V row
// is not finite not at all.
template <int D, int DT>
__device__ void draft_apply(const Tree& A, int64_t slice, float (*t_s)[kTreeMaxNodes], float (*sh_s)[kShareStride],
                            const uint64_t* seen_s, const float* lse_s) {
  constexpr int kRows = kTreeMaxNodes / kTreeWaves;
  const int t = threadIdx.x, n = A.nodes, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t p0 = slice * (A.nchunk + 1) * n;
  const uint64_t above = seen_s[lane] & ~(uint64_t{1} << lane);
  int jump = above ? 63 - __clzll(static_cast<long long>(above)) : -1;    // node `lane`'s parent
  float p[kRows], tot[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int i = wave + kTreeWaves * u;
    p[u] = 0.f;
    if (i < n && (seen_s[i] >> lane & 1)) p[u] = fast_exp2(A.aff[(slice * n + i) * n + lane] - lse_s[i]);
    tot[u] = p[u];
  }
  for (int span = 1; span < n; span *= 2) {
#pragma unroll
    for (int u = 0; u < kRows; ++u)
      if (wave + kTreeWaves * u < n) t_s[wave + kTreeWaves * u][lane] = tot[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (wave + kTreeWaves * u >= n) break;
      const int j = __builtin_amdgcn_readlane(jump, wave + kTreeWaves * u);
      if (j >= 0) tot[u] += t_s[j][lane];
    }
    const int next = __shfl(jump, max(jump, 0), 64);
    jump = jump < 0 ? -1 : next;
    __syncthreads();
  }
  const int n4 = n <= 16 ? (n + 3) & ~3 : kTreeMaxNodes;    // the products below take at least 4 nodes at a time, or a block's
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int i = wave + kTreeWaves * u;
    if (i >= n4) break;
    const float sh = seen_s[i] >> lane & 1 ? p[u] * fast_rcp(tot[u] + kEps) : 0.f;
    sh_s[lane][i] = sh;
    const float sum = wave_sum_dpp(sh);
    if (lane == 0 && i < n) A.part_sum[p0 + i] = sum;
  }
  __syncthreads();
  constexpr int kPer = D < 64 ? D / 4 : 16;             // nodes of a thread at a time
  constexpr int kAhead = 16;                            // V rows in flight
  const int d = t % D;
  const int64_t vbase = (slice * A.cap + A.length) * D + d;
  auto value = [&](int a) {
    const int64_t at = vbase + static_cast<int64_t>(a) * D;
    if constexpr (DT == DT_F32) return static_cast<const float*>(A.v)[at];
    else if constexpr (DT == DT_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(A.v)[at]);
    else return f16_bits_to_f32(static_cast<const uint16_t*>(A.v)[at]);
  };
  for (int i0 = t / D * kPer; i0 < n; i0 += kTreeThreads / D * kPer) {
    float x[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) x[u] = 0.f;
    // `keys` V rows from a0 on: a whole block in straight code, or the fewer of the last
    auto block = [&](auto whole, int a0, int keys) {
      constexpr bool kWhole = decltype(whole)::value;
      float v[kAhead], odd = 0.f;
#pragma unroll
      for (int b = 0; b < kAhead; ++b) v[b] = kWhole || b < keys ? value(a0 + b) : 0.f;
#pragma unroll
      for (int b = 0; b < kAhead; ++b) odd += v[b] - v[b];        // 0, or NaN where a value is not finite
      if (__ballot(odd != 0.f) == 0) {
#pragma unroll
        for (int b = 0; b < kAhead; ++b) {
          if (!kWhole && b >= keys) break;
#pragma unroll
          for (int u = 0; u < kPer; u += 4) {
            if (!kWhole && i0 + u >= n) break;
            const floatx4 sh = *reinterpret_cast<const floatx4*>(&sh_s[a0 + b][i0 + u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u + e] = fmaf(sh[e], v[b], x[u + e]);
          }
        }
      } else {
        for (int b = 0; b < keys; ++b) {
          float vb = v[0];
#pragma unroll
          for (int c = 1; c < kAhead; ++c) vb = c == b ? v[c] : vb;
#pragma unroll
          for (int u = 0; u < kPer; ++u)
            if (seen_s[i0 + u] >> (a0 + b) & 1) x[u] = fmaf(sh_s[a0 + b][i0 + u], vb, x[u]);
        }
      }
    };
    int a0 = 0;
    for (; a0 + kAhead <= n; a0 += kAhead) block(std::true_type{}, a0, kAhead);
    if (a0 < n) block(std::false_type{}, a0, n - a0);
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (i0 + u < n) A.part_out[(p0 + i0 + u) * D + d] = x[u];
  }
}

// ---------------------------------------------------------------------------
// statistics

// One tile of 32 keys (the rows k) against every node: the lane's running maximum and
// sum, node u * 32 + (l & 31).  kind 0: 32 cached keys; 1: the last `left` ones of a
// slice; 2: the drafted keys from key0 on, masked, their affinities kept.
template <int D, int DT, int NT, int KIND>
__device__ __forceinline__ void stat_tile(const KeyRows<D, DT>& k, const u32x4* q_s, const Tree& A, int64_t slice,
                                          const uint64_t* seen_s, int key0, int left, int lane, float (&m)[NT], float (&l)[NT]) {
  using S = Shape<D, DT>;
  const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    floatx16 x = {};
#pragma unroll
    for (int g = 0; g < S::kPieces; ++g) x = mma_piece<DT>(k.p[g], q_s[(u * S::kPieces + g) * 64 + lane], x);
    if constexpr (KIND == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (acc_row(i, h) >= left) x[i] = -INFINITY;
    }
    if constexpr (KIND == 2) {
      const int node = u * kTileNodes + l32;
      const uint64_t seen = seen_s[node];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + acc_row(i, h);
        if (seen >> key & 1) A.aff[(slice * A.nodes + node) * A.nodes + key] = x[i] * A.scale;
        else x[i] = -INFINITY;
      }
    }
    float big = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) big = fmaxf(big, x[i]);
    const float mn = fmaxf(m[u], big * A.scale);
    const float mr = mn == -INFINITY ? 0.f : mn;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += fast_exp2(fmaf(x[i], A.scale, -mr));
    l[u] = fmaf(l[u], fast_exp2(m[u] - mr), sum);
    m[u] = mn;
  }
}

// A wave's statistics, its lane halves (different keys of the same nodes) joined.
template <int NT>
__device__ __forceinline__ void stat_halves(const float (&m)[NT], const float (&l)[NT], int lane, float2* dst) {
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const float mo = __shfl_xor(m[u], 32, 64), lo = __shfl_xor(l[u], 32, 64);
    const float mn = fmaxf(m[u], mo), mr = mn == -INFINITY ? 0.f : mn;
    if (lane < 32)
      dst[u * kTileNodes + lane] = make_float2(mn, l[u] * fast_exp2(m[u] - mr) + lo * fast_exp2(mo - mr));
  }
}

// Waves per SIMD that the registers are held to, by the bytes of a row.
template <int D, int DT, int NT>
constexpr int kStatWaves = Shape<D, DT>::kRow <= 128 ? 5 - NT : Shape<D, DT>::kRow <= 256 ? 4 - NT : 1;

template <int D, int DT, int NT>
__global__ __launch_bounds__(kTreeThreads, (kStatWaves<D, DT, NT>)) void tree_stats(Tree A) {
  using S = Shape<D, DT>;
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  __shared__ u32x4 q_s[NT * S::kPieces * 64];
  __shared__ uint64_t seen_s[kTreeMaxNodes];
  __shared__ float2 red[kTreeWaves][NT * kTileNodes];
  // the first workgroup of a slice takes the drafted keys, wave w the 32 from 32 w on
  const bool drafted = blockIdx.x == 0;
  if (drafted && wave == 0) {
    const uint64_t seen = nodes_seen(A.parents + slice / A.heads * A.parents_sb, A.nodes, lane);
    seen_s[lane] = seen;
    A.seen[slice * kTreeMaxNodes + lane] = seen;
  }
  stage_queries<D, DT, NT>(q_s, A, slice, [&](int r) { return r < A.nodes ? r : -1; });
  const char* keys = static_cast<const char*>(A.k) + slice * A.cap * S::kRow;
  const int64_t end = drafted ? A.length + A.nodes : A.length;
  int64_t row = (drafted ? A.length : static_cast<int64_t>(blockIdx.x - 1) * kBlockRows) + wave * 32;
  const int64_t step = static_cast<int64_t>(A.nstat) * kBlockRows;
  KeyRows<D, DT> cur, nxt;
  cur.load(keys, row, end, lane);
  __syncthreads();
  float m[NT], l[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
  }
  auto tile = [&](auto kind) {
    constexpr int kKind = decltype(kind)::value;
    asm volatile("" ::: "memory");                     // the queries stay in LDS (tree_apply)
    nxt.load(keys, row + step, end, lane);
    loads_go_out();
    stat_tile<D, DT, NT, kKind>(cur, q_s, A, slice, seen_s, static_cast<int>(row - A.length), static_cast<int>(end - row), lane,
                                m, l);
    cur = nxt;
  };
  if (drafted) {
    if (row < end) tile(std::integral_constant<int, 2>{});
  } else {
    for (; row + 32 <= end; row += step) tile(std::integral_constant<int, 0>{});
    if (row < end) tile(std::integral_constant<int, 1>{});
  }
  stat_halves<NT>(m, l, lane, red[wave]);
  __syncthreads();
  if (t < A.nodes) {
    float mn = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) mn = fmaxf(mn, red[w][t].x);
    const float mr = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) sum += red[w][t].y * fast_exp2(red[w][t].x - mr);
    A.part[(slice * (A.nstat + 1) + blockIdx.x) * A.nodes + t] = make_float2(mn, sum);
  }
}

// ---------------------------------------------------------------------------
// shares

// How step 2 takes the bids: 16-bit caches two bf16 parts, 16 bits (2^-17, as the shares'
// two parts in step 3, where the outputs' own rounding makes 2^-9 or 2^-12 at the end),
// fp32 caches three, all 24.  bf16 for its range: where no demand has gone yet a share is
// p / (p + 1e-9), so bids of 1e-9 count, which one fp16 part loses at any scale that holds 1.
template <int DT> constexpr int kBidParts = DT == DT_F32 ? 3 : 2;

// B operands of step 2 for the node of this lane's column: 0/1 by the bits
// 16 s + 8 h + [0, 8) of `mask`
__device__ __forceinline__ u32x4 bits_frag(uint32_t mask, int s, int h) {
  const uint32_t b = mask >> (16 * s + 8 * h);
  u32x4 f;
#pragma unroll
  for (int t = 0; t < 4; ++t) f[t] = (b >> (2 * t) & 1 ? 0x3f80u : 0u) | (b >> (2 * t + 1) & 1 ? 0x3f800000u : 0u);
  return f;
}

template <int D, int DT, int NT> constexpr int kApplyDV = D == 256 && NT == 2 ? 128 : D;

// Waves per SIMD that the registers are held to.  One node tile at head_dim up to 64
// takes V a tile ahead as K, at three waves: 128 slices of 16384 keys 97 -> 91 us, 16 of
// 131072 91 -> 84 against four waves without; elsewhere the registers for it are a wave
// (head_dim 128: 15 -> 18 us at 15 slices of 5003 keys).
template <int D, int DT, int NT>
constexpr int kApplyWaves = NT == 2 ? (DT != DT_F32 && D <= 64 ? 2 : 1) : D <= 64 ? 3 : D == 256 ? 1 : DT == DT_F32 ? 2 : 3;

// ONE: a short slice in one workgroup and one launch, its statistics first and its outputs
// last (one node tile; with two the drafted keys' sums spill beside the walk's).
template <int D, int DT, int NT, bool ONE>
__global__ __launch_bounds__(kTreeThreads, (kApplyWaves<D, DT, NT>)) void tree_apply(Tree A) {
  using S = Shape<D, DT>;
  constexpr int DV = kApplyDV<D, DT, NT>;
  using V = ValueRows<DV, DT>;
  constexpr int kParts = kBidParts<DT>;
  constexpr bool kValuesAhead = D <= 64 && NT == 1;
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), l32 = lane & 31, h = lane >> 5;
  constexpr int kRedStride = DV + 1;
  // a region of LDS for every wave's sums where that takes no workgroup off the CU
  constexpr int kRegionBytes = NT * kTileNodes * kRedStride * 4;
  constexpr int kRegions = kTreeWaves * kRegionBytes * kApplyWaves<D, DT, NT> <= 144 * 1024 ? kTreeWaves : 2;
  __shared__ union {
    u32x4 q[NT * S::kPieces * 64];
    struct {
      float p[kTreeMaxNodes][kTreeMaxNodes];
      float sh[kTreeMaxNodes][kShareStride];
    } draft;
    float red[kRegions][NT * kTileNodes][kRedStride];
    float2 st[kTreeWaves][kTreeMaxNodes];
  } s;
  __shared__ uint64_t seen_s[kTreeMaxNodes];
  __shared__ __attribute__((aligned(16))) float lse_s[kTreeMaxNodes];
  __shared__ float sum_s[kTreeWaves][NT * kTileNodes];
  __shared__ float2 one_st[ONE ? kTreeWaves : 1][NT * kTileNodes];
  const char* keys = static_cast<const char*>(A.k) + slice * A.cap * S::kRow;
  KeyRows<D, DT> cur;
  if constexpr (ONE) {
    if (wave == 0) seen_s[lane] = nodes_seen(A.parents + slice / A.heads * A.parents_sb, A.nodes, lane);
    stage_queries<D, DT, NT>(s.q, A, slice, [&](int r) { return r < A.nodes ? r : -1; });
    __syncthreads();
    float m[NT], l[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      m[u] = -INFINITY;
      l[u] = 0.f;
    }
    int64_t row = wave * 32;
    for (; row + 32 <= A.length; row += kBlockRows) {
      cur.load(keys, row, A.length, lane);
      stat_tile<D, DT, NT, 0>(cur, s.q, A, slice, seen_s, 0, 32, lane, m, l);
    }
    if (row < A.length) {
      cur.load(keys, row, A.length, lane);
      stat_tile<D, DT, NT, 1>(cur, s.q, A, slice, seen_s, 0, static_cast<int>(A.length - row), lane, m, l);
    }
    if (wave * 32 < A.nodes) {
      cur.load(keys, A.length + wave * 32, A.length + A.nodes, lane);
      stat_tile<D, DT, NT, 2>(cur, s.q, A, slice, seen_s, wave * 32, 0, lane, m, l);
    }
    stat_halves<NT>(m, l, lane, one_st[wave]);
  } else {
    if (wave == 0) seen_s[lane] = A.seen[slice * kTreeMaxNodes + lane];
    // the chunks' statistics joined: 64 nodes x 4 groups of entries
    float m = -INFINITY, l = 0.f;
    if (lane < A.nodes) {
      const float2* part = A.part + slice * (A.nstat + 1) * A.nodes + lane;
#pragma unroll 4
      for (int c = wave; c <= A.nstat; c += kTreeWaves) {
        const float2 e = part[static_cast<int64_t>(c) * A.nodes];
        const float mn = fmaxf(m, e.x), mr = mn == -INFINITY ? 0.f : mn;
        l = l * fast_exp2(m - mr) + e.y * fast_exp2(e.x - mr);
        m = mn;
      }
    }
    s.st[wave][lane] = make_float2(m, l);
  }
  __syncthreads();
  if (wave == 0) {
    auto st = [&](int w) {
      if constexpr (ONE) return lane < NT * kTileNodes ? one_st[w][lane] : make_float2(-INFINITY, 0.f);
      else return s.st[w][lane];
    };
    float mn = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) mn = fmaxf(mn, st(w).x);
    const float mr = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) l += st(w).y * fast_exp2(st(w).x - mr);
    // a row of -inf alone has no bids: NaN, as its softmax
    const float lse = seen_s[lane] == 0 ? INFINITY : mn == -INFINITY ? NAN : mn + fast_log2(l);
    lse_s[lane] = lse;
    if (blockIdx.x == 0 && blockIdx.z == 0 && lane < A.nodes) A.lse[slice * A.nodes + lane] = lse;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (blockIdx.z == 0) draft_apply<D, DT>(A, slice, s.draft.p, s.draft.sh, seen_s, lse_s);
    if constexpr (!ONE) return;
    __syncthreads();
  }
  stage_queries<D, DT, NT>(s.q, A, slice, [&](int r) { return r < A.nodes ? r : -1; });
  const char* values = static_cast<const char*>(A.v) + slice * A.cap * S::kRow;
  int64_t row = (ONE ? 0 : static_cast<int64_t>(blockIdx.x - 1) * kBlockRows) + wave * 32;
  const int64_t step = ONE ? kBlockRows : static_cast<int64_t>(A.nchunk) * kBlockRows;
  const float* com0 = A.committed + slice * A.cap;
  cur.load(keys, row, A.length, lane);

  // step 2's operands (a node sees itself: the sums include its own bid)
  u32x4 anc[NT][NT][2], one[2];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint64_t seen = seen_s[u * kTileNodes + l32];
#pragma unroll
    for (int w = 0; w <= u; ++w)
#pragma unroll
      for (int st = 0; st < 2; ++st) anc[u][w][st] = bits_frag(static_cast<uint32_t>(seen >> (w * kTileNodes)), st, h);
  }
#pragma unroll
  for (int st = 0; st < 2; ++st) one[st] = bits_frag(uint32_t{1} << l32, st, h);
  __syncthreads();

  floatx16 acc[NT][V::E];
  float ssum[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    ssum[u] = 0.f;
#pragma unroll
    for (int e = 0; e < V::E; ++e) acc[u][e] = floatx16{};
  }
  const int d0 = static_cast<int>(blockIdx.z) * DV * S::kElt;
  V val;
  if constexpr (kValuesAhead) val.load(values, row, A.length, lane, S::kRow, d0);
  // One tile.  The last one of a slice may be partly past the end: a form of its own,
  // so that the others are straight code.
  auto tile = [&](auto last) {
    constexpr bool kLast = decltype(last)::value;
    // the queries and row statistics stay in LDS: hoisted out of the loop they cost
    // a wave per SIMD
    asm volatile("" ::: "memory");
    const int left = kLast ? static_cast<int>(A.length - row) : 32;
    const float* com = com0 + row + 4 * h;
    if constexpr (!kValuesAhead) val.load(values, row, A.length, lane, S::kRow, d0);
    const V now = val;
    // committed + eps of this lane's keys in step 2's layout
    floatx16 c0;
    if constexpr (!kLast) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c0[4 * g + e] = com[8 * g + e];
      }
    } else {                                            // keys past the end have no demand and (below) no bids
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = com0[row + min(acc_row(i, h), left - 1)];
        c0[i] = acc_row(i, h) < left ? x : 0.f;
      }
    }
    // step 1
    u32x4 p[NT][kParts][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      floatx16 x = {};
#pragma unroll
      for (int g = 0; g < S::kPieces; ++g)
        x = mma_piece<DT>(s.q[(u * S::kPieces + g) * 64 + h * 32 + rho(l32)], cur.p[g], x);
      if constexpr (kLast) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = l32 < left ? x[i] : -INFINITY;
      }
      float v[16];
      // register i of half h: node perm_row(i, h), two runs of 8
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const floatx4 lse = *reinterpret_cast<const floatx4*>(&lse_s[u * kTileNodes + 16 * (g >> 1) + 8 * h + 4 * (g & 1)]);
#pragma unroll
        for (int e = 0; e < 4; ++e)          // NaN (a node without statistics) becomes 0
          v[4 * g + e] = __builtin_amdgcn_fmed3f(fast_exp2(fmaf(x[4 * g + e], A.scale, -lse[e])), 0.f, 1.f);
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 8 * st + 2 * e;
            const uint32_t b = pack_bf16(v[i], v[i + 1]);
            p[u][part][st][e] = b;
            if (part + 1 < kParts) {
              v[i] -= __uint_as_float(b << 16);
              v[i + 1] -= __uint_as_float(b & 0xffff0000u);
            }
          }
      }
    }
    cur.load(keys, row + step, A.length, lane);
    if constexpr (kValuesAhead) val.load(values, row + step, A.length, lane, S::kRow, d0);
#pragma unroll
    for (int i = 0; i < 16; ++i) c0[i] += kEps;
    // steps 2 and 3
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      floatx16 tot = c0, bid = {};
#pragma unroll
      for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          bid = mma_piece<DT_BF16>(p[u][part][st], one[st], bid);
#pragma unroll
          for (int w = 0; w <= u; ++w) tot = mma_piece<DT_BF16>(p[w][part][st], anc[u][w][st], tot);
        }
      float sh[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sh[i] = bid[i] * fast_rcp(tot[i]);
        ssum[u] += sh[i];
      }
      if constexpr (DT == DT_F32) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int e = 0; e < V::E; ++e)
            acc[u][e] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(now.w[i][e]), sh[i], acc[u][e], 0, 0, 0);
      } else {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          u32x4 hi, lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u32x2 b = split_shares<DT>(sh[8 * st + 2 * e] * kShareScale<DT>, sh[8 * st + 2 * e + 1] * kShareScale<DT>);
            hi[e] = b[0];
            lo[e] = b[1];
          }
#pragma unroll
          for (int e = 0; e < V::E; ++e) {
            const u32x4 f = now.frag(e, st);
            acc[u][e] = mma_piece<DT>(f, hi, mma_piece<DT>(f, lo, acc[u][e]));
          }
        }
      }
    }
  };
  for (; row + 32 <= A.length; row += step) tile(std::false_type{});
  if (row < A.length) tile(std::true_type{});
  // the waves' sums, in order
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const float o = ssum[u] + __shfl_xor(ssum[u], 32, 64);
    if (h == 0) sum_s[wave][u * kTileNodes + l32] = o;
  }
#pragma unroll
  for (int w = 0; w < kTreeWaves; w += kRegions) {
    __syncthreads();
    if (wave < w || wave >= w + kRegions) continue;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < V::E; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = V::E * acc_row(i, h) + e;
          if (DV >= 32 || d < DV) {
            float* dst = &s.red[wave - w][u * kTileNodes + l32][d];
            *dst = w == 0 ? acc[u][e][i] : *dst + acc[u][e][i];
          }
        }
  }
  __syncthreads();
  constexpr float kUnscale = 1.f / kShareScale<DT>;
  auto sum_of = [&](int o) {
    float x = s.red[0][o / DV][o % DV];
#pragma unroll
    for (int w = 1; w < kRegions; ++w) x += s.red[w][o / DV][o % DV];
    return x * kUnscale;
  };
  auto shares_of = [&](int i) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) x += sum_s[w][i];
    return x;
  };
  const int64_t p0 = (slice * (A.nchunk + 1) + blockIdx.x) * A.nodes;    // ONE: the drafted keys' entry
  if constexpr (ONE) {
    const uint64_t bad = __ballot(lse_s[lane] != lse_s[lane]);
    for (int o = t; o < A.nodes * DV; o += kTreeThreads) {
      const int i = o / DV, d = o % DV;
      const uint64_t seen = seen_s[i];
      float x = 0.f;
      if (seen != 0) x = (sum_of(o) + A.part_out[(p0 + i) * D + d]) / (shares_of(i) + A.part_sum[p0 + i] + kEps);
      store_as(A.out, A.ov.slice(slice) + i * A.ov.sr + d, DT, (bad & seen) != 0 ? NAN : x);
    }
  } else {
    for (int o = t; o < A.nodes * DV; o += kTreeThreads)
      A.part_out[(p0 + o / DV) * D + blockIdx.z * DV + o % DV] = sum_of(o);
    if (blockIdx.z == 0 && t < A.nodes) A.part_sum[p0 + t] = shares_of(t);
  }
}

// ---------------------------------------------------------------------------
// the chunks' sums joined: one workgroup per node and slice

template <int D, int DT>
__global__ __launch_bounds__(kTreeThreads) void tree_finish(Tree A) {
  constexpr int kGroups = kTreeThreads / D;
  const int64_t slice = A.slice0 + blockIdx.y;
  const int i = blockIdx.x, t = threadIdx.x, lane = t & 63, d = t % D, g = t / D;
  __shared__ float red[kGroups][D + 1];
  const uint64_t seen = A.seen[slice * kTreeMaxNodes + i];
  const float own = lane < A.nodes ? A.lse[slice * A.nodes + lane] : 0.f;
  const bool spoilt = (__ballot(own != own) & seen) != 0;
  const int64_t p0 = slice * (A.nchunk + 1) * A.nodes + i;
  float x = 0.f, sum = 0.f;
  if (seen != 0) {
#pragma unroll 4
    for (int c = g; c <= A.nchunk; c += kGroups) {
      const int64_t at = p0 + static_cast<int64_t>(c) * A.nodes;
      x += A.part_out[at * D + d];
      sum += A.part_sum[at];
    }
  }
  red[g][d] = x;
  if (d == 0) red[g][D] = sum;
  __syncthreads();
  if (t >= D) return;
  x = sum = 0.f;
#pragma unroll
  for (int w = 0; w < kGroups; ++w) {
    x += red[w][d];
    sum += red[w][D];
  }
  store_as(A.out, A.ov.slice(slice) + i * A.ov.sr + d, DT, seen == 0 ? 0.f : spoilt ? NAN : x / (sum + kEps));
}

// ---------------------------------------------------------------------------
// acceptance: one pass over K with step 1's product alone (a lane holds a key); the
// first workgroup of a slice sets the accepted positions' demand and moves their
// rows, all of them into LDS before the first is written.

template <int D, int DT, int NT>
__global__ __launch_bounds__(kTreeThreads) void tree_demand(Tree A) {
  using S = Shape<D, DT>;
  constexpr int kUnits = S::kRow / 16;
  const int64_t slice = A.slice0 + blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), l32 = lane & 31, h = lane >> 5;
  __shared__ union {
    u32x4 q[NT * S::kPieces * 64];
    u32x4 rows[NT * kTileNodes * kUnits];
  } s;
  __shared__ float lse_s[kTreeMaxNodes];
  __shared__ int node_s[kTreeMaxNodes];
  if (t < kTreeMaxNodes) {
    const int a = t < A.count ? A.path[slice / A.heads * A.path_sb + t] : -1;
    const bool ok = a >= 0 && a < A.nodes;
    node_s[t] = ok ? a : -1;
    lse_s[t] = ok ? A.lse[slice * A.nodes + a] : INFINITY;
  }
  __syncthreads();
  float* crow = A.demand + slice * A.cap;
  stage_queries<D, DT, NT>(s.q, A, slice, [&](int r) { return node_s[r]; });
  const char* keys = static_cast<const char*>(A.k) + slice * A.cap * S::kRow;
  if (blockIdx.x == 0) {
    bool moved = false;
    // wave w: the accepted positions 32 w + [0, 32), one per lane, and the bids of the
    // accepted nodes from that one on
    __syncthreads();
    if (wave < NT) {
      const int c = wave * kTileNodes + l32, node = node_s[c];
      KeyRows<D, DT> k;
      k.gather(keys + A.length * S::kRow, A.nodes, lane, node);
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        floatx16 x = {};
#pragma unroll
        for (int g = 0; g < S::kPieces; ++g) x = mma_piece<DT>(s.q[(u * S::kPieces + g) * 64 + lane], k.p[g], x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = u * kTileNodes + acc_row(i, h);
          const float p = fast_exp2(fmaf(x[i], A.scale, -lse_s[r]));
          if (r >= c && lse_s[r] != INFINITY) sum += p;         // no node, or an absent one: whatever its query holds
        }
      }
      sum += __shfl_xor(sum, 32, 64);
      if (h == 0 && c < A.count) crow[A.length + c] = node < 0 ? 0.f : sum;
    }
    for (void* cache : {A.k_move, A.v_move}) {
      if (moved && A.v_move == A.k_move) break;          // K and V in one buffer: once
      moved = true;
      u32x4* rows = reinterpret_cast<u32x4*>(static_cast<char*>(cache) + (slice * A.cap + A.length) * S::kRow);
      __syncthreads();
      for (int u = t; u < A.count * kUnits; u += kTreeThreads)
        if (node_s[u / kUnits] >= 0) s.rows[u] = rows[node_s[u / kUnits] * kUnits + u % kUnits];
      __syncthreads();
      for (int u = t; u < A.count * kUnits; u += kTreeThreads)
        if (node_s[u / kUnits] >= 0) rows[u] = s.rows[u];
    }
    return;
  }
  int64_t row = static_cast<int64_t>(blockIdx.x - 1) * kBlockRows + wave * 32;
  const int64_t step = static_cast<int64_t>(A.nchunk) * kBlockRows;
  KeyRows<D, DT> cur, nxt;
  cur.load(keys, row, A.length, lane);
  float lse[NT][16];
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) lse[u][i] = lse_s[u * kTileNodes + acc_row(i, h)];
  __syncthreads();
  for (; row < A.length; row += step) {
    asm volatile("" ::: "memory");                     // the queries stay in LDS (tree_apply)
    const int64_t j = row + l32;
    const float c = j < A.length ? crow[j] : 0.f;
    nxt.load(keys, row + step, A.length, lane);
    loads_go_out();
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      floatx16 x = {};
#pragma unroll
      for (int g = 0; g < S::kPieces; ++g) x = mma_piece<DT>(s.q[(u * S::kPieces + g) * 64 + lane], cur.p[g], x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // rows that are no node have zero queries and lse +inf, and count for nothing whatever k holds
        const float p = fast_exp2(fmaf(x[i], A.scale, -lse[u][i]));
        sum += lse[u][i] == INFINITY ? 0.f : p;
      }
    }
    sum += __shfl_xor(sum, 32, 64);
    if (h == 0 && j < A.length) crow[j] = c + sum;
    cur = nxt;
  }
}

// ---------------------------------------------------------------------------
// launches

// The workgroups of a slice over its cached keys: those of all slices (one more each,
// for the drafted keys) fill whole rounds of the `slots` that the GPU holds at once,
// as few rounds as fill 15/16 of their places (of 4 rounds the best).  The drafted keys'
// workgroup counts as much as the others though it ends sooner: where few workgroups a
// slice fill a round, its place is idle most of the time (384 slices of 768 places: one
// workgroup over the cached keys each, 16384 keys 499 us where 320 slices take 343).  At least
// `least` keys each: 256 (16 slices of 1000 keys, 128, 256, 512, 1024 of them: shares
// 7.2, 7.4, 10.2, 18.3 us; 15 of 5003 at head_dim 128 16, 15, 18, 27), of fp32 caches
// 128, whose tiles take four times the matrix cycles (16 of 4096 keys 16, 19, 24, 41).
constexpr int64_t least_keys(int dtype) { return dtype == DT_F32 ? kBlockRows : 2 * kBlockRows; }
int tree_split(int64_t n, int64_t length, int64_t slots, int64_t least) {
  if (length < 1) return 0;
  int64_t best = 1, best_fill = -1;
  for (int64_t rounds = (2 * n + slots - 1) / slots, i = 0; i < 4 && best_fill < 960; ++rounds, ++i) {
    const int64_t c = rounds * slots / n - 1, fill = n * (c + 1) * 1024 / (rounds * slots);
    if (fill > best_fill) {
      best = c;
      best_fill = fill;
    }
  }
  const int64_t most = (length + least - 1) / least;
  return static_cast<int>(best < most ? best : most);
}
constexpr int64_t kCUs = 256;

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

// One step's chunks and the places in its workspace.
struct TreePlan {
  int nstat, nchunk;
  size_t part, out, sum, aff, seen, total;
  TreePlan(int64_t n, int64_t length, int64_t nodes, int head_dim, int dtype, int apply_waves) {
    // The places to fill are the CUs times the workgroups that each holds, or a
    // multiple: several short rounds hide one another's start and end.  us with 3, 4, 6,
    // 8, 12, 16 places a CU, 128 slices of 65536 keys and 64 nodes (3 at once):
    // statistics 201, 245, 185, 198, 188, 205; 128 of 16384, 32 nodes (6 at once): 55, 57,
    // 53, 59, 51, 56.  Shares of the first with 2, 3, 4, 8 places (2 at once): 524, 486,
    // 472, 463; of the second with 2, 3, 4, 8 (3 at once): 89, 92, 102, 97.
    nstat = tree_split(n, length, kCUs * (nodes > kTileNodes ? 6 : 12), least_keys(dtype));
    nchunk = tree_split(n, length, kCUs * (nodes > kTileNodes && apply_waves == 2 ? 4 : apply_waves), least_keys(dtype));
    const size_t rows = static_cast<size_t>(n * (nchunk + 1) * nodes);
    part = 0;
    out = part + align_up(sizeof(float2) * n * (nstat + 1) * nodes);
    sum = out + align_up(sizeof(float) * rows * head_dim);
    aff = sum + align_up(sizeof(float) * rows);
    seen = aff + align_up(sizeof(float) * n * nodes * nodes);
    total = seen + align_up(sizeof(uint64_t) * n * kTreeMaxNodes);
  }
};

// Whether a slice's whole step runs in one workgroup (one node tile): little work, where
// two launches less count, or slices that fill the places on the GPU by themselves.
// us a call, three launches -> one, 8 nodes, bf16 64 where nothing else stands:
//   16 slices of 32, 128, 256, 512 keys 13.8 -> 11.3, 13.7 -> 11.6, 13.9 -> 13.5, 13.9 -> 16.8 (1 node
//   13.8 -> 8.5, 13.8 -> 9.0, 13.8 -> 10.7, 13.7 -> 13.9; 32 nodes, 32, 128, 256 keys 20.0 -> 19.2,
//   20.0 -> 19.6, 19.7 -> 21.3); 1, 4 and 64 slices differ by less than 0.6; head_dim 16, 512 and 768
//   keys 13.7 -> 12.6, 13.8 -> 14.5; head_dim 128, 32 and 128 keys 14.4 -> 13.2, 14.4 -> 14.4; fp32,
//   32 and 64 keys 15.2 -> 14.7, 16.1 -> 15.0
//   256 keys: 128, 192, 256, 384, 512, 768, 900 slices 14.6 -> 13.7, 16.0 -> 13.9, 16.2 -> 13.9,
//   20.2 -> 16.7, 26.4 -> 17.0, 33.5 -> 22.0, 40.1 -> 37.4
//   1024 keys: 256, 384, 512, 768, 900 slices 27.2 -> 30.8, 42.2 -> 38.8, 47.5 -> 41.3, 74.4 -> 54.7,
//   80.6 -> 86.1 (fp32 53 -> 54, 110 -> 77, 102 -> 80, 187 -> 110, 195 -> 153)
//   16384 keys: 384, 512, 640, 768, 900, 1100, 1300 slices 499 -> 503, 576 -> 557, 684 -> 699,
//   999 -> 766, 981 -> 1105, 1435 -> 1248, 1385 -> 1402 (fp32, 384 slices 1320 -> 1159; head_dim 128,
//   4096 keys: 270 -> 257, 314 -> 281, 381 -> 361, 552 -> 393, 550 -> 587, 792 -> 666, 766 -> 715)
//   head_dim 256 (256 places), 1024 keys: 256, 320, 512, 768, 900 slices 114 -> 79, 112 -> 143,
//   222 -> 159, 358 -> 269, 330 -> 347
// One threshold for all of them is off at its edges.  It takes the slower form for 900
// slices of 1024 keys and 640 and 1300 of 16384 (1 to 7%), and misses the quicker one for one
// node at 256 keys (22%), 384 and 512 slices at head_dim 128 (5 and 11%), 512 of 16384 keys
// (3%) and fp32 384 of them (12%).
template <int D, int DT>
bool tree_in_one(int64_t n, int64_t length, int64_t places) {
  constexpr int64_t kRow = Shape<D, DT>::kRow;
  if (kRow <= 128 && length * kRow <= 16384) return true;
  if (n < 192) return false;
  if (length <= 256) return true;
  if (2 * n < places) return false;
  if (D <= 128 && length <= 1024) return true;
  const int64_t rounds = (n + places - 1) / places;          // the share of the rounds' places that the slices fill
  return 100 * n >= (D <= 128 ? 70 : 95) * rounds * places;
}

template <int D, int DT, int NT>
int launch_step(const TreeArgs& a) {
  Tree A = tree_of(a);
  const TreePlan w(a.n, a.length, a.nodes, D, DT, kApplyWaves<D, DT, NT>);
  A.nstat = w.nstat;
  A.nchunk = w.nchunk;
  char* ws = static_cast<char*>(a.workspace);
  A.part = reinterpret_cast<float2*>(ws + w.part);
  A.part_out = reinterpret_cast<float*>(ws + w.out);
  A.part_sum = reinterpret_cast<float*>(ws + w.sum);
  A.aff = reinterpret_cast<float*>(ws + w.aff);
  A.seen = reinterpret_cast<uint64_t*>(ws + w.seen);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  if constexpr (NT == 1) {
    if (tree_in_one<D, DT>(a.n, a.length, kCUs * kApplyWaves<D, DT, NT>)) {
      slice_batches(a.n, [&](int64_t s0, unsigned ns) {
        A.slice0 = s0;
        DIL_TIMED("tree_one", st, (tree_apply<D, DT, NT, true><<<dim3(1, ns), kTreeThreads, 0, st>>>(A)));
      });
      return static_cast<int>(hipGetLastError());
    }
  }
  const unsigned chunks = static_cast<unsigned>(A.nchunk + 1);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    A.slice0 = s0;
    DIL_TIMED("tree_stats", st, (tree_stats<D, DT, NT><<<dim3(A.nstat + 1, ns), kTreeThreads, 0, st>>>(A)));
    DIL_TIMED("tree_apply", st,
              (tree_apply<D, DT, NT, false><<<dim3(chunks, ns, D / kApplyDV<D, DT, NT>), kTreeThreads, 0, st>>>(A)));
    DIL_TIMED("tree_finish", st, (tree_finish<D, DT><<<dim3(A.nodes, ns), kTreeThreads, 0, st>>>(A)));
  });
  return static_cast<int>(hipGetLastError());
}

template <int D, int DT, int NT>
int launch_accept(const TreeArgs& a) {
  Tree A = tree_of(a);
  // us for 128 slices of 65536 keys with 3, 4, 8, 16, 24, 32 places a CU: 263, 245, 262,
  // 244, 233, 230; 24 slices of 9001 keys 11 with any
  A.nchunk = tree_split(a.n, a.length, kCUs * 24, 2 * kBlockRows);
  A.demand = a.committed;
  A.k_move = a.k_cache;
  A.v_move = a.v_cache;
  A.path = a.path;
  A.path_sb = a.path_sb;
  A.count = a.count;
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    A.slice0 = s0;
    DIL_TIMED("tree_demand", st,
              (tree_demand<D, DT, NT><<<dim3(static_cast<unsigned>(A.nchunk + 1), ns), kTreeThreads, 0, st>>>(A)));
  });
  return static_cast<int>(hipGetLastError());
}

// f(head dim, dtype, node tiles) as integral constants
template <typename F>
int with_shape(int head_dim, int dtype, int nodes, F&& f) {
  auto by_nodes = [&](auto d, auto t) {
    return nodes <= kTileNodes ? f(d, t, std::integral_constant<int, 1>{}) : f(d, t, std::integral_constant<int, 2>{});
  };
  auto by_dtype = [&](auto d) {
    switch (dtype) {
      case DT_F32: return by_nodes(d, std::integral_constant<int, DT_F32>{});
      case DT_BF16: return by_nodes(d, std::integral_constant<int, DT_BF16>{});
      case DT_F16: return by_nodes(d, std::integral_constant<int, DT_F16>{});
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
  if (n < 1 || length < 0 || nodes < 1 || nodes > kTreeMaxNodes) return 0;
  int64_t bytes = 0;
  with_shape(head_dim, dtype, static_cast<int>(nodes), [&](auto d, auto t, auto nt) {
    bytes = static_cast<int64_t>(TreePlan(n, length, nodes, d(), t(), kApplyWaves<d(), t(), nt()>).total);
    return 0;
  });
  return bytes;
}

int tree_step(const TreeArgs& a) {
  return with_shape(a.head_dim, a.dtype, a.nodes, [&](auto d, auto t, auto nt) { return launch_step<d(), t(), nt()>(a); });
}

int tree_accept(const TreeArgs& a) {
  return with_shape(a.head_dim, a.dtype, a.count, [&](auto d, auto t, auto nt) { return launch_accept<d(), t(), nt()>(a); });
}

}  // namespace dil
