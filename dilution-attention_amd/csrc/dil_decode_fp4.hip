// The decode step over caches in 4 bits (dil_decode_step_fp4; the format is in dil_fp4.hpp):
// dil_decode_step's mathematics on the values that codes and scales stand for,
//
//   a_j = log2(e) q.k_j / sqrt(D),  p_j = 2^(a_j - m) / sum 2^(a - m),  m = max a
//   share_j = p_j / (committed_j + p_j + eps)
//   committed_j += p_j,  out = sum share_j v_j / (sum share_j + eps)
//
// in the same launches: fp4_one where one workgroup does a slice's whole step, else fp4_stats
// (affinities to scratch, chunk max and sum), fp4_apply (shares, demand, chunk sums of share v)
// and fp4_finish.
//
// A key costs D + 2 D / 32 bytes of codes and scales, 8 of demand and 8 of affinities (84 at
// D = 64, where 16-bit caches take 272), so both walks have to be short of instructions.  The
// scores come from the matrix unit, which takes codes and scales as they lie: 16 bytes of codes a
// lane go from memory into its operand.  V rows need one conversion for two elements and one fma
// each (fp32 sums); their scales stay out of the walk, since the shares go into LDS once for each
// block, times its V scale.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dil_decode_impl.hpp"
#include "dil_fp4.hpp"

namespace dil {
namespace {

// One workgroup per slice takes 1024 threads; the chunked step workgroups of 256 over chunks of
// at most 1024 keys, eight to a CU, so that some load while others reduce, and a rule as the
// decode step's (decode_chunk): as many chunks as fill whole rounds of what the GPU holds at
// once.  (At head_dim 256 a CU holds four, by fp4_stats' registers and the shares in fp4_apply's
// LDS; the chunks are the same there.)  us per step (bf16, head_dim 64: 128 slices of 16384 keys; 16 and 256 of 131072): 256 threads
// and 1024 keys 37, 38, 440; 512 and 2048 36, 37, 441 (at head_dim 32, 128 slices of 65536 keys, 77
// against 75); 128 and 512 37, 41, 450; 256 and 512 39, 46, 493; 256 and 2048 36, 39, 454.
constexpr int kOneThreads = 1024;
constexpr int kOneWaves = kOneThreads / 64;
constexpr int kQThreads = 256;
constexpr int kQWaves = kQThreads / 64;
constexpr int64_t kQResident = 2048;
constexpr int64_t kQMaxChunk = 1024;
constexpr int64_t kQMinChunk = 256;

__host__ __device__ inline int64_t fp4_target_chunks(int64_t n, int64_t length) {
  const int64_t base = (length + kQMaxChunk - 1) / kQMaxChunk;
  const int64_t rounds = (n * base + kQResident - 1) / kQResident;
  const int64_t target = rounds * kQResident / n;
  return target < base ? base : target;
}
__host__ __device__ inline int64_t fp4_chunk(int64_t n, int64_t length) {
  if (length < 1 || n < 1) return kQMinChunk;
  const int64_t target = fp4_target_chunks(n, length);
  const int64_t chunk = (length + target - 1) / target;
  return chunk < kQMinChunk ? kQMinChunk : chunk;
}
// Chunks per slice in the grid and the scratch (as decode_chunks: device_length for every live
// length up to `length`).
inline int64_t fp4_chunks(int64_t n, int64_t length, bool device_length) {
  if (length < 1) return 1;
  if (!device_length) {
    const int64_t chunk = fp4_chunk(n, length);
    return (length + chunk - 1) / chunk;
  }
  const int64_t per_min = (length + kQMinChunk - 1) / kQMinChunk;
  const int64_t target = fp4_target_chunks(n < 1 ? 1 : n, length);
  return per_min < target ? per_min : target;
}

// E elements a lane, so that D / E neighbouring lanes hold a row; W waves
template <int D, int E, int W> struct QLayout {
  static constexpr int kLanesPerRow = D / E;
  static constexpr int kRowsPerWave = 64 / kLanesPerRow;
  static constexpr int kRowsPerBlock = kRowsPerWave * W;
  static constexpr int kWords = E / 8;
};
// Elements of a V row that a lane takes: half a block, whose sums (one an element) leave the
// registers for eight workgroups of a CU (whole blocks, in the order above: 39, 42, 478 us).  At head_dim
// 256 both are the same: 64 slices of 32768 keys 120, 128 of 16384 116 us.
constexpr int kVElems = 16;

template <int W> struct CodeWords {
  uint32_t w[W];
};
template <int W>
__device__ __forceinline__ CodeWords<W> load_codes(const uint8_t* p) {
  CodeWords<W> r;
  if constexpr (W == 4) {
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = x[2]; r.w[3] = x[3];
  } else {
    static_assert(W == 2, "8 or 16 bytes");
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = x[0]; r.w[1] = x[1];
  }
  return r;
}

// The workgroup's walk over `count` rows of codes from `base` on, U rows a lane in flight; rows
// past the end are read as the last one.  A walk of three and more such blocks keeps the next one
// in flight behind the one at hand (one workgroup a slice, 8000 keys: 24 -> 21 us; below, the
// copies cost 0.3 us).
template <int D, int E, int W>
struct CodeStream {
  using L = QLayout<D, E, W>;
  static constexpr int U = 4, kRows = L::kRowsPerBlock, kStep = U * kRows;
  const uint8_t* base;
  int first, count;
  uint32_t part;                                          // this lane's bytes of a row
  CodeWords<L::kWords> r[U];
  __device__ __forceinline__ CodeStream(const uint8_t* b, int wave, int lane, int n)
      : base(b), first(wave * L::kRowsPerWave + lane / L::kLanesPerRow), count(n), part(lane % L::kLanesPerRow * (E / 2)) {}
  __device__ __forceinline__ void at(int jb) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      r[u] = load_codes<L::kWords>(base + (static_cast<uint32_t>(min(jb + u * kRows, count - 1)) * (D / 2) + part));
  }
  __device__ __forceinline__ void load() {
    if (count > 0) at(first);
  }
  template <typename F>
  __device__ __forceinline__ void each(int jb, const CodeWords<L::kWords> (&c)[U], F&& f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jb + u * kRows;
      if (j < count) f(j, c[u]);
    }
  }
  template <typename F>
  __device__ __forceinline__ void walk(F&& f) {
    if (count <= 2 * kStep) {
      for (int jb = first; jb < count; jb += kStep) {
        if (jb != first) at(jb);
        each(jb, r, f);
      }
      return;
    }
    for (int jb = first; jb < count; jb += kStep) {
      CodeWords<L::kWords> c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = r[u];
      if (jb + kStep < count) at(jb + kStep);
      each(jb, c, f);
    }
  }
};

// The scores of 64 keys by one wave, on v_mfma_scale_f32_16x16x128_f8f6f4: B holds 16 keys a
// column each (codes and scales as they lie in the cache), A the query.
//
// A query element is a sum of digits: part i is the nearest whole multiple, -16 to 16, of
// 2^(E - 3 - 5 i) to what the parts before leave, E the exponent of the largest of its 32 elements.
// fp8 (e4m3) holds these numbers, the powers are A's scales.  Within a block the unit adds
// products only down to 2^-13 of the largest one (measured; whole blocks and C in fp32), which
// whole numbers up to 16 times codes never reach: a block's sum is exact.  8 parts leave less than
// 2^-39 of the largest element, of bf16 elements next to it nothing after 4 (which would take half
// of the products: 1% less time at 128 slices of 16384 keys, and errors of 2^-19 of the largest
// element in the small ones).  The 16 rows of A hold parts 0 to 3 four times over; the second
// four parts are a product of their own into the same sums.
//
// The last part's unit is 2^(E - 38), and a scale is 2^-127 or more: a block below 2^-80 is taken 2^t up to
// it, exactly, and its keys' scales t down, so that elements down to the subnormal ones count in full against
// keys of powers up to 2^125.  A scale that would fall below 2^-127 is held there (t is 47 at most: its key
// is below 2^-78, its products with that block below 2^-158, nothing beside a bid's rounding).  A
// first part can be 2^(E + 1), past the element itself: A's scales are half of the parts' and the factor
// of the affinities twice itself, so that the sums of a score below 2^128 stay finite.
//
// A lane's 16 bytes of codes are one block of one key; the 4 blocks of K = 128 (lane group
// kb = lane / 16 holds block kb of B and both operands' scales of it) are rows of 4, 2 or 1 keys.
// fp8 operands lie otherwise: lane group g holds elements 16 (g % 2) to 16 (g % 2) + 15 of blocks
// g / 2 and 2 + g / 2.  For D <= 64 the rows of A are 0 in the blocks of keys that are not theirs, so
// that lane group g of the result (rows 4 g to 4 g + 3) gets the keys of its own set.  For
// D >= 128 each 16 keys have sums of their own and the lane group picks its.  So lane l ends with
// the score of key l.
typedef int intx8 __attribute__((ext_vector_type(8)));

template <int D> struct KeyTiles {
  static constexpr int kBlocks = Fp4Row<D>::kBlocks;
  static constexpr int kMma = kBlocks;                    // instructions for 64 keys
  static constexpr int kSets = kBlocks >= 4 ? 1 : 4 / kBlocks;        // of 16 keys in one instruction
  static constexpr int kHalves = kBlocks >= 4 ? kBlocks / 4 : 1;      // instructions of a row
  static constexpr int kWords = D < 32 ? 2 : 4;
  // block kb of K = 128 of instruction m: a key of the 64 (for column c), and a block of its row
  __device__ static __forceinline__ int key(int m, int kb, int c) {
    if constexpr (kSets == 1) return 16 * (m / kHalves) + c;
    else return 16 * (kSets * m + kb * kSets / 4) + c;
  }
  __device__ static __forceinline__ int block(int m, int kb) {
    if constexpr (kSets == 1) return 4 * (m % kHalves) + kb;
    else return kb % kBlocks;
  }
};

constexpr int kParts = 8;
template <int D> struct alignas(16) QueryShared {
  uint8_t part[kParts][D];
  int exponent[Fp4Row<D>::kBlocks];
  int up[Fp4Row<D>::kBlocks];                             // the t of a block
};
constexpr int kLeastExponent = -80;

__device__ __forceinline__ int part_exponent(int e, int i) { return e - 3 - 5 * i; }

// Element t of the query (0 past the row): loaded ahead of the keys, so that its parts do not
// wait for them (loads complete in issue order).
template <int D>
__device__ __forceinline__ float query_element(const void* q1, int64_t idx, int qdt, int t) {
  if (t >= D) return 0.f;
  if (qdt == DT_F32) return static_cast<const float*>(q1)[idx + t];
  const uint16_t x = static_cast<const uint16_t*>(q1)[idx + t];
  return qdt == DT_BF16 ? bf16_bits_to_f32(x) : f16_bits_to_f32(x);
}

// The query's parts into LDS, one element a thread (the first D threads); a barrier follows.
template <int D>
__device__ __forceinline__ void split_query(float x, QueryShared<D>& sh) {
  const int t = threadIdx.x;
  if (t >= D) return;
  uint32_t top = __float_as_uint(x) & 0x7fffffffu;
  auto with = [&](int other) { top = max(top, static_cast<uint32_t>(other)); };
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0xB1, 0xF, 0xF, true));      // quad_perm [1, 0, 3, 2]
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x4E, 0xF, 0xF, true));      // quad_perm [2, 3, 0, 1]
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x141, 0xF, 0xF, true));     // row_half_mirror
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x140, 0xF, 0xF, true));     // row_mirror
  if constexpr (Fp4Row<D>::kBlock == 32) with(__shfl_xor(static_cast<int>(top), 16, 64));
  // a query with a NaN or an infinity becomes NaN
  const bool bad = top >= 0x7f800000u;
  int e = min(static_cast<int>(top >> 23) - 127, 127);
  const int up = top != 0u ? max(kLeastExponent - e, 0) : 0;
  e = max(e, kLeastExponent);
  x *= __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
  if (t % Fp4Row<D>::kBlock == 0) {
    sh.exponent[t / Fp4Row<D>::kBlock] = e;
    sh.up[t / Fp4Row<D>::kBlock] = up;
  }
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int unit = part_exponent(e, i);
    const float digit = rintf(x * __uint_as_float(static_cast<uint32_t>(127 - unit) << 23));
    x = fmaf(-digit, __uint_as_float(static_cast<uint32_t>(127 + unit) << 23), x);
    sh.part[i][t] = bad ? 0x7f : static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(digit, 0.f, 0, false));
  }
}

// A wave's A operands: in registers, but for head_dim 256, whose 32 would leave fp4_stats three waves a
// SIMD instead of four and fp4_one without enough: there read from LDS at each use (64 slices of
// 32768 keys 120 us, held 119).
template <int D> struct QueryTiles {
  using T = KeyTiles<D>;
  static constexpr bool kHeld = T::kHalves == 1;
  const QueryShared<D>& sh;
  int lane;
  intx8 a[kHeld ? kParts / 4 : 1];
  int scale[kParts / 4][T::kHalves];
  bool any_up = false;                                    // the same in all lanes
  __device__ __forceinline__ QueryTiles(const QueryShared<D>& s, int l) : sh(s), lane(l) {
#pragma unroll
    for (int p = 0; p < kParts / 4; ++p) {
#pragma unroll
      for (int h = 0; h < T::kHalves; ++h) {
        const int b = T::block(h, lane >> 4), up = sh.up[b];
        scale[p][h] = (126 + part_exponent(sh.exponent[b], (lane & 3) + 4 * p)) | up << 8;      // the unit takes the low byte
        any_up |= __ballot(up != 0) != 0;
      }
      if constexpr (kHeld) a[p] = read(p, 0);
    }
  }
  __device__ __forceinline__ intx8 read(int p, int h) const {
    const int set = (lane & 15) >> 2, g = lane >> 4;
    intx8 x;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int kb = g / 2 + 2 * (w / 4), at = 16 * (g % 2) + 4 * (w % 4);
      const bool mine = (T::kSets == 1 || kb * T::kSets / 4 == set % T::kSets) && at < Fp4Row<D>::kBlock;
      const int y = *reinterpret_cast<const int*>(&sh.part[(lane & 3) + 4 * p][T::block(h, kb) * Fp4Row<D>::kBlock + (mine ? at : 0)]);
      x[w] = mine ? y : 0;
    }
    return x;
  }
  __device__ __forceinline__ intx8 operand(int p, int h) const {
    if constexpr (kHeld) return a[p];
    else return read(p, h);
  }
  // The keys' scales on queries with blocks that were taken up (NaN blocks stay such)
  __device__ __forceinline__ void lower(uint32_t (&s)[T::kMma]) const {
#pragma unroll
    for (int m = 0; m < T::kMma; ++m) {
      const int x = static_cast<int>(s[m]) - (scale[0][m % T::kHalves] >> 8);
      s[m] = s[m] == 255u ? 255u : static_cast<uint32_t>(max(x, 0));
    }
  }
  // Half the score of key `lane` of the 64 whose codes and scales these are
  __device__ __forceinline__ float score(const CodeWords<T::kWords> (&c)[T::kMma], const uint32_t (&s)[T::kMma]) const {
    constexpr int kOuts = 4 / T::kSets;                   // 16-key groups with sums of their own
    float out = 0.f;
#pragma unroll
    for (int g = 0; g < kOuts; ++g) {
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < T::kHalves; ++h) {
        const int m = g * T::kHalves + h;
        intx8 b = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < T::kWords; ++w) b[w] = static_cast<int>(c[m].w[w]);
#pragma unroll
        for (int p = 0; p < kParts / 4; ++p)
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(p, h), b, acc, 0, 4, 0, scale[p][h], 0,
                                                                 static_cast<int>(s[m]));
      }
      const float x = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      out = g == 0 || (lane >> 4) * kOuts / 4 == g ? x : out;
    }
    // every lane's operands count: the products must not move into a branch that some lanes leave
    asm volatile("" : "+v"(out));
    return out;
  }
};

// A wave's groups of 64 keys: `group`, group + step, ... (keys past the end are read as the last one);
// f(key, half its score) once a lane and group.
template <int D> struct KeyGroups {
  using T = KeyTiles<D>;
  // groups in flight: 4 loads of codes a lane.  The registers of 8 would leave one workgroup of
  // 1024 threads a CU instead of two, or spill (600 slices of 4000 keys 56 us, 40 with 4).
  static constexpr int U = T::kMma >= 4 ? 1 : 4 / T::kMma;
  CodeWords<T::kWords> c[U][T::kMma];
  uint32_t s[U][T::kMma];
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int count, int group, int step, int lane) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int m = 0; m < T::kMma; ++m) {
        const uint32_t j = static_cast<uint32_t>(min(64 * (group + u * step) + T::key(m, lane >> 4, lane & 15), count - 1));
        const uint32_t b = static_cast<uint32_t>(T::block(m, lane >> 4));
        c[u][m] = load_codes<T::kWords>(codes + (j * (D / 2) + b * (Fp4Row<D>::kBlock / 2)));
        s[u][m] = scales[j * T::kBlocks + b];
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(const QueryTiles<D>& q, int count, int group, int step, int lane, F&& f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = 64 * (group + u * step);
      if (j >= count) break;
      if (q.any_up) q.lower(s[u]);
      f(j + lane, q.score(c[u], s[u]));
    }
  }
};

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

// Lane moves on the vector unit: a wave's reduction by LDS shuffles is six round trips of ~100
// cycles, and the step has eight of them in a row.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ float dpp(float old, float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CTRL, ROWS, 0xF, false));
}
constexpr int kShr1 = 0x111, kShr2 = 0x112, kShr4 = 0x114, kShr8 = 0x118, kBcast15 = 0x142, kBcast31 = 0x143;
__device__ __forceinline__ float last_lane(float x) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_sum_dpp(float x) {
  x += dpp<kShr1>(0.f, x);
  x += dpp<kShr2>(0.f, x);
  x += dpp<kShr4>(0.f, x);
  x += dpp<kShr8>(0.f, x);
  x += dpp<kBcast15, 0xA>(0.f, x);
  x += dpp<kBcast31, 0xC>(0.f, x);
  return last_lane(x);
}
__device__ __forceinline__ float wave_max_dpp(float x) {
  constexpr float kNone = -INFINITY;
  x = fmaxf(x, dpp<kShr1>(kNone, x));
  x = fmaxf(x, dpp<kShr2>(kNone, x));
  x = fmaxf(x, dpp<kShr4>(kNone, x));
  x = fmaxf(x, dpp<kShr8>(kNone, x));
  x = fmaxf(x, dpp<kBcast15, 0xA>(kNone, x));
  x = fmaxf(x, dpp<kBcast31, 0xC>(kNone, x));
  return last_lane(x);
}
template <int O> __device__ __forceinline__ float from_xor(float x) {
  if constexpr (O == 1) return dpp<0xB1>(0.f, x);         // quad_perm [1, 0, 3, 2]
  else if constexpr (O == 2) return dpp<0x4E>(0.f, x);    // quad_perm [2, 3, 0, 1]
  else if constexpr (O == 8) return dpp<0x128>(0.f, x);   // row_ror:8
  else return __shfl_xor(x, O, 64);
}

// The sums of v over the lanes that differ in the bits O, O / 2, ..., LEAST: each step halves what
// a lane holds, so that it ends with the sums of its elements from `at` on alone (N - 1 moves
// and one for each step that is left then, where a sum element by element takes N moves a step).
template <int N, int O, int LEAST>
__device__ __forceinline__ void scatter_sums(float (&v)[N], int lane, int& at) {
  if constexpr (O >= LEAST) {
    if constexpr (N > 1) {
      constexpr int H = N / 2;
      const bool up = lane & O;
      float h[H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if constexpr (O >= 16) {
          // swaps the half (row) of the one with the other half (row) of the other
          u32x2 r;
          if constexpr (O == 32) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + H]), false, false);
            r = u32x2{x[0], x[1]};
          } else {
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + H]), false, false);
            r = u32x2{x[0], x[1]};
          }
          h[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        } else {
          const float keep = up ? v[i + H] : v[i], send = up ? v[i] : v[i + H];
          h[i] = keep + from_xor<O>(send);
        }
      }
      at += up ? H : 0;
      scatter_sums<H, O / 2, LEAST>(h, lane, at);
#pragma unroll
      for (int i = 0; i < H; ++i) v[i] = h[i];
    } else {
      v[0] += from_xor<O>(v[0]);
      scatter_sums<1, O / 2, LEAST>(v, lane, at);
    }
  }
}
// How many elements a lane ends with
constexpr int scattered(int n, int least) {
  for (int o = 32; o >= least && n > 1; o /= 2) n /= 2;
  return n;
}
// The workgroup's sums of share v, one row of D for each wave
template <int D, int E>
__device__ __forceinline__ void wave_sums(float (&acc)[E], int lane, float* row) {
  constexpr int kLanesPerRow = D / E;
  int at = lane % kLanesPerRow * E;
  scatter_sums<E, 32, kLanesPerRow>(acc, lane, at);
#pragma unroll
  for (int i = 0; i < scattered(E, kLanesPerRow); ++i) row[at + i] = acc[i];   // lanes with the same `at` hold the same sums
}

// Maximum and sum of 2^(a - maximum) of affinities, joined in any order of parts.  A NaN among
// them, which no maximum shows, makes the sum NaN.
struct RowStats {
  float m = -INFINITY, l = 0.f;
  bool bad = false;
  __device__ __forceinline__ void add(float a) {
    bad |= a != a;
    const float mn = fmaxf(m, a);
    if (mn > -INFINITY) {
      l = l * fast_exp2(m - mn) + fast_exp2(a - mn);
      m = mn;
    }
  }
  __device__ __forceinline__ float2 of_lane() const { return make_float2(m, bad ? NAN : l); }
};
// The same from a part a lane, in every lane (a part without a maximum, of no affinities or of NaN
// alone, adds its sum as it is)
__device__ __forceinline__ float2 join_stats(float2 p) {
  const float m = wave_max_dpp(p.x);
  return make_float2(m, wave_sum_dpp(p.x > -INFINITY ? p.y * fast_exp2(p.x - m) : p.y));
}
__device__ __forceinline__ float2 part_of_lane(const float2* p, int n, int lane) {
  return lane < n ? p[lane] : make_float2(-INFINITY, 0.f);
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
template <int D>
__device__ __forceinline__ void fp4_one_slice(const Fp4DecodeArgs& A, int64_t slice, int live, float qscale, float* s) {
  constexpr int EV = kVElems, N = Fp4Row<D>::kBlocks;
  __shared__ QueryShared<D> qs;
  __shared__ float2 part[kOneWaves];
  __shared__ float red[kOneWaves][D + 1];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row0 = slice * A.capacity;
  float* crow = A.committed + row0;
  if (A.k1 != nullptr && live > 0) {
    append_rows<D>(A, slice, live - 1);
    __syncthreads();
  }
  // group i of a wave is keys t, t + 1024, ... of its threads: what a thread leaves in s it reads back
  const uint8_t* kc = code_rows<D>(A.k_cache, row0);
  const uint8_t* ks = static_cast<const uint8_t*>(A.k_cache.scales) + row0 * N;
  const float qx = query_element<D>(A.q1, slice * D, A.q_dtype, t);
  KeyGroups<D> keys;
  const auto* vs = scale_rows<D>(A.v_cache, row0);
  // the demand and the V scales of this thread's first keys, in flight over the scores
  constexpr int kAhead = 2;
  float c0[kAhead] = {};
  typename ScaleWord<N>::type v0[kAhead] = {};
  if (live > 0) {
    keys.load(kc, ks, live, wave, kOneWaves, lane);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = min(t + u * kOneThreads, live - 1);
      c0[u] = __builtin_nontemporal_load(crow + j);
      v0[u] = vs[j];
    }
  }
  split_query<D>(qx, qs);
  __syncthreads();
  RowStats stats;
  {
    const QueryTiles<D> q(qs, lane);
    for (int g = wave; 64 * g < live; g += KeyGroups<D>::U * kOneWaves) {
      if (g != wave) keys.load(kc, ks, live, g, kOneWaves, lane);
      keys.each(q, live, g, kOneWaves, lane, [&](int j, float x) {
        if (j >= live) return;
        const float a = qscale * x;
        s[j * N] = a;
        stats.add(a);
      });
    }
  }
  CodeStream<D, EV, kOneWaves> v(code_rows<D>(A.v_cache, row0), wave, lane, live);
  v.load();                                             // in flight over the reductions
  const float2 ws = join_stats(stats.of_lane());
  if (lane == 0) part[wave] = ws;
  __syncthreads();
  const float2 all = join_stats(part_of_lane(part, kOneWaves, lane));
  const float inv = 1.f / all.y;
  float ssum = 0.f;
  auto take = [&](int j, float cm, typename ScaleWord<N>::type scale) {
    const float p = fast_exp2(s[j * N] - all.x) * inv;
    const float sh = p * fast_rcp(cm + p + kEps);
    __builtin_nontemporal_store(cm + p, crow + j);
    scaled_shares<N>(s + j * N, sh, scale);
    ssum += sh;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (t + u * kOneThreads < live) take(t + u * kOneThreads, c0[u], v0[u]);
  for (int j = t + kAhead * kOneThreads; j < live; j += kOneThreads) take(j, __builtin_nontemporal_load(crow + j), vs[j]);
  ssum = wave_sum_dpp(ssum);
  if (lane == 0) red[wave][D] = ssum;
  __syncthreads();
  const int vb = lane % (D / EV) * EV / Fp4Row<D>::kBlock;
  float acc[EV];
#pragma unroll
  for (int e = 0; e < EV; ++e) acc[e] = 0.f;
  v.walk([&](int j, const CodeWords<EV / 8>& c) { add_codes<EV>(acc, s[j * N + vb], c); });
  wave_sums<D, EV>(acc, lane, red[wave]);
  __syncthreads();
  if (t < D) {
    float x = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kOneWaves; ++w) {
      x += red[w][t];
      sum += red[w][D];
    }
    store_as(A.out, slice * D + t, A.q_dtype, x / (sum + kEps));
  }
}

template <int D>
__global__ __launch_bounds__(kOneThreads, D <= 128 ? 8 : 4) void fp4_one(Fp4DecodeArgs A, float qscale, int64_t slice0) {
  extern __shared__ float one_s[];
  fp4_one_slice<D>(A, slice0 + blockIdx.x, static_cast<int>(live_length(A.dlen, A.length)), qscale, one_s);
}

template <int D>
__global__ __launch_bounds__(kQThreads) void fp4_stats(Fp4DecodeArgs A, float* __restrict__ aff, float2* __restrict__ part,
                                                       int64_t chunk, int nchunk, float qscale, int64_t slice0,
                                                       int64_t one_max) {
  constexpr int N = Fp4Row<D>::kBlocks;
  const int64_t live = live_length(A.dlen, A.length);
  if (live <= one_max) return;                            // fp4_finish does the whole step
  const int64_t slice = slice0 + blockIdx.y;
  const int c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (A.dlen != nullptr) chunk = fp4_chunk(A.n, live);
  const int nlive = live_chunks(live, chunk);
  if (c >= nlive) return;
  const int64_t j0 = c * chunk, row0 = slice * A.capacity + j0;
  const int count = static_cast<int>(min(j0 + chunk, live) - j0);
  if (A.k1 != nullptr && c == nlive - 1) {
    append_rows<D>(A, slice, live - 1);
    __syncthreads();
  }
  const uint8_t* kc = code_rows<D>(A.k_cache, row0);
  const uint8_t* ks = static_cast<const uint8_t*>(A.k_cache.scales) + row0 * N;
  const float qx = query_element<D>(A.q1, slice * D, A.q_dtype, threadIdx.x);
  KeyGroups<D> keys;
  keys.load(kc, ks, count, wave, kQWaves, lane);
  __shared__ QueryShared<D> qs;
  split_query<D>(qx, qs);
  __syncthreads();
  const QueryTiles<D> q(qs, lane);
  float* arow = aff + slice * A.length + j0;
  RowStats stats;
  for (int g = wave; 64 * g < count; g += KeyGroups<D>::U * kQWaves) {
    if (g != wave) keys.load(kc, ks, count, g, kQWaves, lane);
    keys.each(q, count, g, kQWaves, lane, [&](int j, float x) {
      if (j >= count) return;
      const float a = qscale * x;
      arow[j] = a;
      stats.add(a);
    });
  }
  __shared__ float2 waves[kQWaves];
  const float2 ws = join_stats(stats.of_lane());
  if (lane == 0) waves[wave] = ws;
  __syncthreads();
  if (wave != 0) return;
  const float2 all = join_stats(part_of_lane(waves, kQWaves, lane));
  if (lane == 0) part[slice * nchunk + c] = all;
}

template <int D>
__global__ __launch_bounds__(kQThreads) void fp4_apply(Fp4DecodeArgs A, const float* __restrict__ aff,
                                                       const float2* __restrict__ part, float* __restrict__ part_out,
                                                       int64_t chunk, int nchunk, int64_t slice0, int64_t one_max) {
  constexpr int E = kVElems, N = Fp4Row<D>::kBlocks;
  const int64_t live = live_length(A.dlen, A.length);
  if (live <= one_max) return;                            // fp4_finish does the whole step
  const int64_t slice = slice0 + blockIdx.y;
  const int c = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (A.dlen != nullptr) chunk = fp4_chunk(A.n, live);
  const int nlive = live_chunks(live, chunk);
  if (c >= nlive) return;
  const int64_t j0 = c * chunk, row0 = slice * A.capacity + j0;
  const int count = static_cast<int>(min(j0 + chunk, live) - j0);
  const float* arow = aff + slice * A.length + j0;
  float* crow = A.committed + row0;
  const auto* vs = scale_rows<D>(A.v_cache, row0);
  // what comes first is loaded first (loads complete in issue order): the chunks' statistics, then
  // this thread's keys, then V rows.  The demand goes past the caches,
  // both ways, and leaves them to the affinities: 256 slices of 131072 keys 489 -> 440 us.
  const float2* prow = part + slice * nchunk;
  const float2 first = prow[min(lane, nlive - 1)];
  constexpr int kOwn = static_cast<int>(kQMaxChunk / kQThreads);
  float av[kOwn], cv[kOwn];
  typename ScaleWord<N>::type sv[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int j = min(static_cast<int>(threadIdx.x) + u * kQThreads, count - 1);
    av[u] = arow[j];
    cv[u] = __builtin_nontemporal_load(crow + j);
    sv[u] = vs[j];
  }
  CodeStream<D, E, kQWaves> v(code_rows<D>(A.v_cache, row0), wave, lane, count);
  v.load();
  // the slice's statistics from its chunks' (every wave by itself)
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < nlive; i += 64) {
    const float2 ps = i == lane ? first : prow[i];
    const float mn = fmaxf(m, ps.x);
    l = (m > -INFINITY ? l * fast_exp2(m - mn) : l) + (ps.x > -INFINITY ? ps.y * fast_exp2(ps.x - mn) : ps.y);
    m = mn;
  }
  const float2 all = join_stats(make_float2(m, l));
  const float inv = 1.f / all.y;

  __shared__ float s[kQMaxChunk * N];
  __shared__ float red[kQWaves][D + 1];
  float ssum = 0.f;
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const int j = threadIdx.x + u * kQThreads;
    if (j >= count) break;
    const float p = fast_exp2(av[u] - all.x) * inv;
    const float sh = p * fast_rcp(cv[u] + p + kEps);
    __builtin_nontemporal_store(cv[u] + p, crow + j);
    scaled_shares<N>(s + j * N, sh, sv[u]);
    ssum += sh;
  }
  ssum = wave_sum_dpp(ssum);
  if (lane == 0) red[wave][D] = ssum;
  __syncthreads();
  const int vb = lane % (D / E) * E / Fp4Row<D>::kBlock;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  v.walk([&](int j, const CodeWords<E / 8>& w) { add_codes<E>(acc, s[j * N + vb], w); });
  wave_sums<D, E>(acc, lane, red[wave]);
  __syncthreads();
  for (int i = threadIdx.x; i <= D; i += kQThreads) {
    float x = 0.f;
    for (int w = 0; w < kQWaves; ++w) x += red[w][i];
    part_out[(slice * nchunk + c) * (D + 1) + i] = x;
  }
}

// One workgroup per slice: the chunks' columns (D of share v, one of the shares) summed by kGroups
// threads each, every kGroups-th chunk a thread and four in flight, then over the groups; always in the
// same order.  ONE: a device-resident length that may be short: then the whole step is done here,
// and the launches before had nothing to do.
template <int D, bool ONE>
__global__ __launch_bounds__(ONE ? kOneThreads : 512, ONE && D <= 128 ? 8 : 4) void fp4_finish(Fp4DecodeArgs A, const float* __restrict__ part_out,
                                                                      int64_t chunk, int nchunk, float qscale,
                                                                      int64_t slice0, int64_t one_max) {
  constexpr int kThreads = ONE ? kOneThreads : 512;
  constexpr int kCols = D + 1, kGroups = 512 / kCols < 16 ? 512 / kCols : 16;
  const int64_t slice = slice0 + blockIdx.x, live = live_length(A.dlen, A.length);
  if constexpr (ONE) {
    extern __shared__ float one_s[];
    if (live <= one_max) {
      fp4_one_slice<D>(A, slice, static_cast<int>(live), qscale, one_s);
      return;
    }
  }
  __shared__ float sum[kGroups][kCols];
  if (A.dlen != nullptr) chunk = fp4_chunk(A.n, live);
  const int nlive = live_chunks(live, chunk);
  for (int e = threadIdx.x; e < kGroups * kCols; e += kThreads) {
    const int g = e / kCols;
    const float* p = part_out + slice * nchunk * kCols + e % kCols;
    float x = 0.f;
    int i = g;
    for (; i + 3 * kGroups < nlive; i += 4 * kGroups) {
      float y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = p[static_cast<int64_t>(i + u * kGroups) * kCols];
      x += (y[0] + y[1]) + (y[2] + y[3]);
    }
    for (; i < nlive; i += kGroups) x += p[static_cast<int64_t>(i) * kCols];
    sum[g][e % kCols] = x;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float x = 0.f, shares = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      x += sum[g][threadIdx.x];
      shares += sum[g][D];
    }
    store_as(A.out, slice * D + threadIdx.x, A.q_dtype, x / (shares + kEps));
  }
}

// The most keys of a slice that one workgroup takes whole; above, the chunked step, whose three
// launches take 9.5 us at least and whose many workgroups catch up where few slices leave CUs idle.
// us per step, one workgroup -> chunked (bf16 queries):
//   64:  1 slice 2000 keys 8.1 -> 9.6, 4000 12.2 -> 9.7; 16 slices 2000 9.0 -> 10.4, 4000 12.9 -> 10.8;
//        64 slices 4000 13.4 -> 14.6, 8000 22 -> 19; 128 slices 8100 24 -> 26, 12000 33 -> 32;
//        160 slices 8100 26 -> 29, 16000 44 -> 45; 256 slices 2000 12 -> 19, 16000 56 -> 69;
//        264 slices 8100 44 -> 42, 10000 59 -> 47; 300 slices 8100 44 -> 44; 400 slices 8100 49 -> 57,
//        12000 74 -> 76; 600 slices 8100 73 -> 79, 12000 108 -> 104; 1024 slices 16000 206 -> 235
//   128: 16 slices 1000 8.3 -> 11.7, 2000 11.7 -> 12.0; 64 slices 2000 12.0 -> 13.9, 4000 20 -> 17;
//        128 slices 4000 22 -> 24, 6000 30 -> 30; 256 slices 8000 51 -> 61; 264 slices 4000 39 -> 39,
//        6000 63 -> 52; 400 slices 4000 43 -> 49
//   256: 16 slices 500 10 -> 13, 1000 15 -> 13; 128 slices 1000 16 -> 17, 2000 25 -> 24; 256 slices 4000
//        54 -> 65; 264 slices 2000 50 -> 42; 400 slices 500 21 -> 23; 512 slices 2000 57 -> 65
//   32:  16 slices 4000 8.2 -> 11, 6000 11.4 -> 11.5; 128 slices 8000 15 -> 20, 16000 26 -> 27; 144 slices
//        16000 27 -> 32, 32000 50 -> 50; 192 slices 16000 30 -> 37, 32000 55 -> 59; 256 slices 16000 35 -> 43,
//        32000 66 -> 75; 300 slices 16000 46 -> 50; 400 slices 16000 51 -> 62, 32000 113 -> 113; 600 slices
//        16000 80 -> 86
//   16:  16 slices 4000 7.8 -> 9.9, 8000 11.9 -> 10.9; 128 slices 16000 22 -> 22, 32000 40 -> 34; 144 slices
//        16000 23 -> 28, 24000 32 -> 33, 32000 42 -> 40; 192 slices 16000 24 -> 30, 32000 44 -> 46; 256 slices
//        16000 26 -> 34, 32000 47 -> 58; 300 slices 16000 32 -> 39; 400 slices 16000 35 -> 49, 32000
//        88 -> 87; 600 slices 16000 56 -> 66
template <int D>
int64_t fp4_one_max(int64_t n) {
  constexpr int64_t kKeyBytes = D + 2 * Fp4Row<D>::kBlocks + 8;
  constexpr int64_t kMost = 32768 / Fp4Row<D>::kBlocks;               // 128 KB of LDS: one float a key and block
  if (n < 144) {
    const int64_t keys = (D == 256 ? (420 + n) << 9 : (210 + 4 * n) << 10) / kKeyBytes;
    return std::min({keys, kMost, int64_t{16384}});
  }
  if (n <= 256) return kMost;
  // more slices than CUs: up to 64 KB (and but for head_dim 256, by its registers) two of them share a
  // CU; else rounds of 256, worth it where the last one is filled
  const int64_t places = (n + 255) / 256 * 256;
  if (16 * n >= 13 * places) return kMost;
  return D == 256 ? 512 : kMost / 2;
}

struct Fp4Scratch {
  size_t part, part_out, total;
  Fp4Scratch(int64_t n, int64_t length, int head_dim, int64_t nchunk) {
    part = align_up(sizeof(float) * n * length);
    part_out = part + align_up(sizeof(float2) * n * nchunk);
    total = part_out + align_up(sizeof(float) * n * nchunk * (head_dim + 1));
  }
};

template <int D>
int launch_fp4(const Fp4DecodeArgs& a) {
  const int64_t chunk = fp4_chunk(a.n, a.length);
  const int nchunk = static_cast<int>(fp4_chunks(a.n, a.length, a.dlen != nullptr));
  const float qscale = 2.f * kLog2e / sqrtf(static_cast<float>(D));      // of half a score
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const int64_t keys = fp4_one_max<D>(a.n);
  const auto lds_of = [](int64_t k) { return sizeof(float) * static_cast<size_t>((k + 63) / 64 * 64 * Fp4Row<D>::kBlocks); };
  if (a.length <= keys) {
    slice_batches(a.n, [&](int64_t s0, unsigned ns) {
      DIL_TIMED("fp4_one", st, (fp4_one<D><<<dim3(ns), kOneThreads, lds_of(a.length), st>>>(a, qscale, s0)));
    });
    return static_cast<int>(hipGetLastError());
  }
  const int64_t one_max = a.dlen != nullptr ? keys : -1;  // a device-resident length may be short
  const Fp4Scratch w(a.n, a.length, D, nchunk);
  char* ws = static_cast<char*>(a.workspace);
  float* aff = reinterpret_cast<float*>(ws);
  float2* part = reinterpret_cast<float2*>(ws + w.part);
  float* part_out = reinterpret_cast<float*>(ws + w.part_out);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    DIL_TIMED("fp4_stats", st,
              (fp4_stats<D><<<dim3(nchunk, ns), kQThreads, 0, st>>>(a, aff, part, chunk, nchunk, qscale, s0, one_max)));
  });
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    DIL_TIMED("fp4_apply", st,
              (fp4_apply<D><<<dim3(nchunk, ns), kQThreads, 0, st>>>(a, aff, part, part_out, chunk, nchunk, s0, one_max)));
  });
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    if (one_max >= 0)
      DIL_TIMED("fp4_finish", st,
                (fp4_finish<D, true><<<dim3(ns), kOneThreads, lds_of(one_max), st>>>(a, part_out, chunk, nchunk, qscale, s0,
                                                                                        one_max)));
    else
      DIL_TIMED("fp4_finish", st,
                (fp4_finish<D, false><<<dim3(ns), 512, 0, st>>>(a, part_out, chunk, nchunk, qscale, s0, one_max)));
  });
  return static_cast<int>(hipGetLastError());
}

}  // namespace

// Sized for a device-resident length up to `length`, as the decode step's; nothing where every
// length up to it takes one workgroup a slice.
int64_t decode_fp4_workspace_bytes(int64_t n, int64_t length, int head_dim) {
  if (n < 1 || length < 1) return 0;
  const int64_t one = head_dim == 16    ? fp4_one_max<16>(n)
                      : head_dim == 32  ? fp4_one_max<32>(n)
                      : head_dim == 64  ? fp4_one_max<64>(n)
                      : head_dim == 128 ? fp4_one_max<128>(n)
                                        : fp4_one_max<256>(n);
  if (length <= one) return 0;
  return static_cast<int64_t>(Fp4Scratch(n, length, head_dim, fp4_chunks(n, length, true)).total);
}

int decode_fp4(const Fp4DecodeArgs& a) {
  switch (a.head_dim) {
    case 16: return launch_fp4<16>(a);
    case 32: return launch_fp4<32>(a);
    case 64: return launch_fp4<64>(a);
    case 128: return launch_fp4<128>(a);
    case 256: return launch_fp4<256>(a);
    default: return kErrHeadDim;
  }
}

}  // namespace dil
