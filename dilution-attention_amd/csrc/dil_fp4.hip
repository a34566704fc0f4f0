// Rows written into 4-bit caches and read back (dil_fp4_write, dil_fp4_read; the format is in
// dil_fp4.hpp).
//
// Both move bytes: a 16-bit row of 64 elements is 128 bytes on one side and 34 on the other.
// Writing, a lane takes 8 elements (16 bytes of 16-bit rows, 4 bytes of codes), so that a wave's
// accesses are contiguous on both sides; the 4 lanes of a block find its largest magnitude
// with two lane moves and its first lane stores the scale byte.  Reading, a lane gives 16 bytes of
// values.  What is used once goes past the caches: rows of 128 bytes and more as they are read
// (shorter ones are parts of lines that other heads' lanes read too), codes and values as they are
// stored.  K and V of 8 sequences x 16 heads x 16384 tokens, head_dim 64, bf16 views of a projection:
// written in 111 us (6.1 TB/s; 128 with cached accesses), read back in 107 (6.4; 116); fp32 values
// in 88 us for half of the heads (149 with two 16-byte stores a lane).
#include <hip/hip_runtime.h>

#include "dil_fp4.hpp"
#include "dil_internal.hpp"

namespace dil {
namespace {

constexpr int kFp4Threads = 256;
constexpr int kWritePasses = 4, kReadPasses = 2;      // rows of a lane, loaded together

template <int D> constexpr int kWriteRows = kFp4Threads * 8 / D;     // rows of a pass

template <int DT> using Raw8 = std::conditional_t<DT == DT_F32, floatx8, u16x8>;

// One row of K (grid z 0) or V (1) for each D / 8 lanes
template <int D, int DT>
__global__ __launch_bounds__(kFp4Threads) void fp4_write(const void* __restrict__ k, RowsView kv, const void* __restrict__ v,
                                                         RowsView vv, int64_t rows, Fp4Cache kc, Fp4Cache vc,
                                                         int64_t capacity, int64_t start,
                                                         const int64_t* __restrict__ start_dev, int64_t slice0) {
  using F = Fp4Row<D>;
  constexpr int kLanes = D / 8;
  const bool second = blockIdx.z != 0;
  const int64_t slice = slice0 + blockIdx.y;
  const void* src = second ? v : k;
  const RowsView view = second ? vv : kv;
  const Fp4Cache cache = second ? vc : kc;
  const int c = threadIdx.x % kLanes;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kWritePasses * kWriteRows<D>) + threadIdx.x / kLanes;
  const int64_t base = view.slice(slice) + 8 * c;
  Raw8<DT> r[kWritePasses];
#pragma unroll
  for (int u = 0; u < kWritePasses; ++u) {
    const int64_t row = min(row0 + u * kWriteRows<D>, rows - 1);
    const int64_t at = base + row * view.sr;
    if constexpr (DT == DT_F32) {
      const floatx4* p = reinterpret_cast<const floatx4*>(static_cast<const float*>(src) + at);
      const floatx4 a = p[0], b = p[1];
      r[u] = floatx8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
      if constexpr (D >= 64) r[u] = __builtin_nontemporal_load(reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(src) + at));
      else
        r[u] = *reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(src) + at);
    }
  }
  const int64_t pos = start_dev != nullptr ? *start_dev : start;
  uint32_t* codes = static_cast<uint32_t*>(cache.codes) + slice * capacity * kLanes + c;
  uint8_t* scales = static_cast<uint8_t*>(cache.scales) + slice * capacity * F::kBlocks + c * 8 / F::kBlock;
#pragma unroll
  for (int u = 0; u < kWritePasses; ++u) {
    const uint32_t s = fp4_scale(block_top<D>(top_bits<DT>(r[u])));
    const uint32_t word = fp4_codes8<DT>(r[u], s);
    const int64_t row = row0 + u * kWriteRows<D>;
    // a position outside the cache is never written (a device-resident start is not checked)
    if (row < rows && pos >= -row && pos < capacity - row) {
      __builtin_nontemporal_store(word, codes + (pos + row) * kLanes);
      if (c * 8 % F::kBlock == 0) scales[(pos + row) * F::kBlocks] = static_cast<uint8_t>(s);
    }
  }
}

template <int DT> constexpr int kReadElems = DT == DT_F32 ? 4 : 8;      // 16 bytes of values a lane

template <int D, int DT>
__global__ __launch_bounds__(kFp4Threads) void fp4_read(Fp4Cache kc, Fp4Cache vc, int64_t capacity, int64_t start,
                                                        int64_t rows, void* __restrict__ k, void* __restrict__ v,
                                                        int64_t slice0) {
  using F = Fp4Row<D>;
  constexpr int E = kReadElems<DT>, kLanes = D / E, kPass = kFp4Threads / kLanes;
  using Word = std::conditional_t<E == 8, uint32_t, uint16_t>;
  const bool second = blockIdx.z != 0;
  const int64_t slice = slice0 + blockIdx.y;
  void* dst = second ? v : k;
  const Fp4Cache cache = second ? vc : kc;
  const int c = threadIdx.x % kLanes;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kReadPasses * kPass) + threadIdx.x / kLanes;
  const Word* codes = static_cast<const Word*>(cache.codes) + (slice * capacity + start) * kLanes + c;
  const uint8_t* scales =
      static_cast<const uint8_t*>(cache.scales) + (slice * capacity + start) * F::kBlocks + c * E / F::kBlock;
  uint32_t word[kReadPasses], s[kReadPasses];
#pragma unroll
  for (int u = 0; u < kReadPasses; ++u) {
    const int64_t row = min(row0 + u * kPass, rows - 1);
    word[u] = codes[row * kLanes];
    s[u] = scales[row * F::kBlocks];
  }
#pragma unroll
  for (int u = 0; u < kReadPasses; ++u) {
    const int64_t row = row0 + u * kPass;
    float x[8];
    fp4_values8(word[u], x);
    const float factor = fp4_factor(s[u]);
    if (row >= rows) continue;
    if constexpr (DT == DT_F32) {
      __builtin_nontemporal_store(floatx4{x[0] * factor, x[1] * factor, x[2] * factor, x[3] * factor},
                                  reinterpret_cast<floatx4*>(static_cast<float*>(dst) + (slice * rows + row) * D) + c);
    } else {
      u16x8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = DT == DT_BF16 ? f32_to_bf16_bits(x[e] * factor) : f32_to_f16_bits(x[e] * factor);
      __builtin_nontemporal_store(y, reinterpret_cast<u16x8*>(static_cast<uint16_t*>(dst) + (slice * rows + row) * D) + c);
    }
  }
}

template <int D, int DT>
int launch_write(const Fp4WriteArgs& a) {
  constexpr int64_t kRows = kWritePasses * kWriteRows<D>;
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows), ns, 2);
    DIL_TIMED("fp4_write", st,
              (fp4_write<D, DT><<<grid, kFp4Threads, 0, st>>>(a.k, a.kv, a.v, a.vv, a.rows, a.k_cache, a.v_cache, a.capacity,
                                                              a.start, a.start_dev, s0)));
  });
  return static_cast<int>(hipGetLastError());
}

template <int D, int DT>
int launch_read(const Fp4ReadArgs& a) {
  constexpr int64_t kRows = kReadPasses * kFp4Threads * kReadElems<DT> / D;
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  slice_batches(a.n, [&](int64_t s0, unsigned ns) {
    const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows), ns, 2);
    DIL_TIMED("fp4_read", st,
              (fp4_read<D, DT><<<grid, kFp4Threads, 0, st>>>(a.k_cache, a.v_cache, a.capacity, a.start, a.rows, a.k, a.v, s0)));
  });
  return static_cast<int>(hipGetLastError());
}

// f(head_dim, dtype) as constants
template <typename F>
int with_type(int head_dim, int dtype, F&& f) {
  auto typed = [&](auto d) {
    switch (dtype) {
      case DT_F32: return f(d, std::integral_constant<int, DT_F32>{});
      case DT_BF16: return f(d, std::integral_constant<int, DT_BF16>{});
      case DT_F16: return f(d, std::integral_constant<int, DT_F16>{});
      default: return kErrDtype;
    }
  };
  switch (head_dim) {
    case 16: return typed(std::integral_constant<int, 16>{});
    case 32: return typed(std::integral_constant<int, 32>{});
    case 64: return typed(std::integral_constant<int, 64>{});
    case 128: return typed(std::integral_constant<int, 128>{});
    case 256: return typed(std::integral_constant<int, 256>{});
    default: return kErrHeadDim;
  }
}

}  // namespace

int fp4_write(const Fp4WriteArgs& a) {
  return with_type(a.head_dim, a.dtype, [&](auto d, auto t) { return launch_write<d(), t()>(a); });
}

int fp4_read(const Fp4ReadArgs& a) {
  return with_type(a.head_dim, a.dtype, [&](auto d, auto t) { return launch_read<d(), t()>(a); });
}

}  // namespace dil
