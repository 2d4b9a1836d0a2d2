// Block quantisation to e4m3 (fp8.cuh) and reading it back.
//
//   rows      x [M,K] -> data [M,K], scale [M,ceil(K/128)]: one scale for 128 values of a row
//   permuted  the same rows written to the expert-major places of their tokens: x is read and quantised
//             once and stored k times
//   weight    w [G,N,K] -> data [G,N,K], scale [G,ceil(N/128),ceil(K/128)]: one scale for 128 x 128 values, so
//             the same tensor serves the product with w and, read the other way, with its transpose
//   read      data, scale -> bf16 rows: an e4m3 number times a power of two, exact within bf16's range (below
//             2^-133 results are rounded, from 2^128 on they are infinite)
//
// All four only move bytes; K is a multiple of 16, so that a thread holds 16
// values (one 16-byte store) and eight lanes a block. The values stay packed
// as they were loaded between the maximum and the conversion (the weight
// kernel with unpacked fp32 and a filter on every value: 438 us instead of
// 204). Measured: 8192 x 7168 rows to 8 places each 101 us, 5.9 TB/s; weight
// 16 x 4096 x 7168 bf16 204 us, 6.9 TB/s; 16384 x 2048 read back 18 us,
// 5.7 TB/s.
#include "fp8.cuh"

namespace moe {
namespace {

using namespace fp8;

constexpr int kUnit = 16;  // values of one thread

// 16 values as they lie in memory. amax() is one instruction a value: the
// largest magnitude, and not finite if any value is not; amax_finite() and
// pack(.., true) then treat such a block as fp8.cuh says.
struct Bf16Unit {
  using T = __nv_bfloat16;
  uint4 q[2];
  MOE_DEVICE void load(const T* p) {
    q[0] = __ldg(reinterpret_cast<const uint4*>(p));
    q[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  MOE_DEVICE void zero() { q[0] = q[1] = make_uint4(0u, 0u, 0u, 0u); }
  MOE_DEVICE uint32_t word(int i) const {
    const uint4& v = q[i >> 2];
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
  }
  MOE_DEVICE float value(int i) const {
    return (i & 1) ? bf16_hi(word(i >> 1)) : bf16_lo(word(i >> 1));
  }
  MOE_DEVICE float amax() const {
    uint32_t a = word(0) & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < 8; ++i)
      asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(word(i) & 0x7FFF7FFFu));
    return max_nan(bf16_lo(a), bf16_hi(a));
  }
  MOE_DEVICE static float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
  }
};
struct Fp32Unit {
  using T = float;
  float v[kUnit];
  MOE_DEVICE void load(const T* p) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(p) + h);
      v[4 * h] = q.x;
      v[4 * h + 1] = q.y;
      v[4 * h + 2] = q.z;
      v[4 * h + 3] = q.w;
    }
  }
  MOE_DEVICE void zero() {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] = 0.f;
  }
  MOE_DEVICE float value(int i) const { return v[i]; }
  MOE_DEVICE float amax() const {
    float a = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < kUnit; ++i) a = Bf16Unit::max_nan(a, fabsf(v[i]));
    return a;
  }
};

template <typename U>
MOE_DEVICE float amax_finite(const U& u) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < kUnit; ++i) a = fmaxf(a, finite_abs(u.value(i)));
  return a;
}

// `odd`: the block holds a value that is not finite.
template <typename U>
MOE_DEVICE uint4 pack(const U& u, float inv, bool odd) {
  uint32_t w[4];
  if (!odd) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = pack4(u.value(4 * i) * inv, u.value(4 * i + 1) * inv, u.value(4 * i + 2) * inv,
                   u.value(4 * i + 3) * inv);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = pack4(scaled(u.value(4 * i), inv), scaled(u.value(4 * i + 1), inv),
                   scaled(u.value(4 * i + 2), inv), scaled(u.value(4 * i + 3), inv));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

MOE_DEVICE float max8(float a) {  // over the eight lanes of a block
#pragma unroll
  for (int off = 4; off > 0; off >>= 1)
    a = Bf16Unit::max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
  return a;
}

constexpr int kMaxRowThreads = 512;
constexpr int kMaxTopk = 32;

// One CTA per row (grid-stride over rows), a thread for every unit of it as far
// as 512 reach, so that a row's loads are all under way at once. kPermute: the row goes to its
// token's k destinations instead of its own place.
template <typename U, bool kPermute>
__global__ void __launch_bounds__(kMaxRowThreads) quantize_rows_kernel(
    const typename U::T* __restrict__ x, int64_t rows, int units, int kb, const int64_t* __restrict__ map,
    const int64_t* __restrict__ experts, int k, int64_t E, int64_t num_out,
    uint4* __restrict__ data, uint8_t* __restrict__ scale) {
  __shared__ int64_t s_dst[kMaxTopk];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    if (kPermute) {
      __syncthreads();
      if (threadIdx.x < k) {
        const int64_t e = __ldg(experts + r * k + threadIdx.x);
        int64_t d = -1;
        if (e >= 0 && e < E) d = __ldg(map + r * E + e);
        s_dst[threadIdx.x] = d < num_out ? d : -1;
      }
      __syncthreads();
    }
    for (int u0 = 0; u0 < units; u0 += blockDim.x) {
      const int u = u0 + threadIdx.x;
      const bool in = u < units;
      U v;
      v.zero();
      if (in) v.load(x + (r * units + u) * kUnit);
      float a = max8(v.amax());
      const bool odd = !(a < INFINITY);
      if (__any_sync(0xffffffffu, odd)) {
        const float f = max8(amax_finite(v));
        if (odd) a = f;
      }
      const uint32_t b = scale_byte(a);
      const uint4 q = pack(v, inverse_scale(b), odd);
      if (!in) continue;
      if (kPermute) {
        for (int j = 0; j < k; ++j) {
          const int64_t d = s_dst[j];
          if (d < 0) continue;
          data[d * units + u] = q;
          if ((u & 7) == 0) scale[d * kb + (u >> 3)] = static_cast<uint8_t>(b);
        }
      } else {
        data[r * units + u] = q;
        if ((u & 7) == 0) scale[r * kb + (u >> 3)] = static_cast<uint8_t>(b);
      }
    }
  }
}

// One CTA per 128 x 128 block of one weight matrix; a thread holds kUnits
// units (bf16: 4, 256 threads; fp32: 2, 512 threads: 32 registers of data
// either way, so that enough blocks are resident to overlap one's loads with
// another's stores).
template <typename U, int kUnits>
__global__ void __launch_bounds__(1024 / kUnits) quantize_weight_kernel(
    const typename U::T* __restrict__ w, int64_t N, int units, int kb, uint4* __restrict__ data,
    uint8_t* __restrict__ scale) {
  constexpr int kThreads = 1024 / kUnits, kRows = kThreads / 8;
  __shared__ float s_amax[kThreads / 32];
  const int u = blockIdx.x * 8 + (threadIdx.x & 7);
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kBlock + (threadIdx.x >> 3);
  const int64_t base = static_cast<int64_t>(blockIdx.z) * N;
  U v[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int64_t n = n0 + kRows * i;
    v[i].zero();
    if (u < units && n < N) v[i].load(w + ((base + n) * units + u) * kUnit);
  }
  // the block's amax, of the finite values alone if there are others
  auto block_max = [&](float a) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      a = Bf16Unit::max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
    if (lane_id() == 0) s_amax[warp_id()] = a;
    __syncthreads();
    a = s_amax[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) a = Bf16Unit::max_nan(a, s_amax[i]);
    return a;
  };
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) a = Bf16Unit::max_nan(a, v[i].amax());
  a = block_max(a);
  const bool odd = !(a < INFINITY);
  if (odd) {  // the whole block takes this branch
    __syncthreads();
    a = 0.f;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) a = fmaxf(a, amax_finite(v[i]));
    a = block_max(a);
  }
  const uint32_t b = scale_byte(a);
  const float inv = inverse_scale(b);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int64_t n = n0 + kRows * i;
    if (u < units && n < N) data[(base + n) * units + u] = pack(v[i], inv, odd);
  }
  if (threadIdx.x == 0)
    scale[(static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * kb + blockIdx.x] =
        static_cast<uint8_t>(b);
}

// One CTA per kReadRows rows, 8 values of each per thread: consecutive lanes
// store consecutive 16 bytes, a thread has four loads under way, and nothing
// is divided (with a 64-bit quotient in every thread 20 against 18 us for
// 16384 x 2048).
constexpr int kReadRows = 4;
__global__ void __launch_bounds__(kMaxRowThreads) dequantize_rows_kernel(
    const uint2* __restrict__ data, const uint8_t* __restrict__ scale, int64_t rows, int units, int kb,
    uint4* __restrict__ out) {
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kReadRows; r0 < rows;
       r0 += static_cast<int64_t>(gridDim.x) * kReadRows) {
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      uint2 q[kReadRows];
      uint32_t b[kReadRows];
#pragma unroll
      for (int h = 0; h < kReadRows; ++h)
        if (r0 + h < rows) {
          q[h] = __ldg(data + (r0 + h) * units + u);
          b[h] = __ldg(scale + (r0 + h) * kb + (u >> 4));
        }
#pragma unroll
      for (int h = 0; h < kReadRows; ++h)
        if (r0 + h < rows) {
          const float s = scale_value(b[h]);
          const float2 v0 = unpack2(q[h].x), v1 = unpack2(q[h].x >> 16);
          const float2 v2 = unpack2(q[h].y), v3 = unpack2(q[h].y >> 16);
          out[(r0 + h) * units + u] =
              make_uint4(pack_bf16x2(v0.x * s, v0.y * s), pack_bf16x2(v1.x * s, v1.y * s),
                         pack_bf16x2(v2.x * s, v2.y * s), pack_bf16x2(v3.x * s, v3.y * s));
        }
    }
  }
}

bool aligned16(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

// Threads of a CTA for a row of `units` units: all in one pass, or in equal passes.
int row_threads(int units) {
  const int passes = (units + kMaxRowThreads - 1) / kMaxRowThreads;
  return ((units + passes - 1) / passes + 31) / 32 * 32;
}

template <bool kPermute, typename U>
int launch_rows(const void* x, int64_t M, int64_t K, const int64_t* map, const int64_t* experts, int k,
                int64_t E, int64_t num_out, void* data, void* scale, cudaStream_t s,
                const char* who) {
  const int64_t grid = M < (1 << 20) ? M : (1 << 20);
  const int units = static_cast<int>(K / kUnit);
  quantize_rows_kernel<U, kPermute><<<static_cast<unsigned>(grid), row_threads(units), 0, s>>>(
      static_cast<const typename U::T*>(x), M, units, static_cast<int>((K + kBlock - 1) / kBlock), map, experts,
      k, E, num_out, static_cast<uint4*>(data), static_cast<uint8_t*>(scale));
  MOE_CUDA_CHECK_LAUNCH(who);
  return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_quantize_fp8(const void* x, int32_t src_type, int64_t M, int64_t K, void* data,
                                void* scale, moe_stream_t stream) {
  MOE_REQUIRE(src_type == 0 || src_type == 1, "quantize_fp8: src_type must be 0 (bf16) or 1 (fp32)");
  MOE_REQUIRE(M >= 0 && K >= 16 && K % 16 == 0 && K < (1ll << 31),
              "quantize_fp8: M=%lld K=%lld (K must be a positive multiple of 16)", (long long)M,
              (long long)K);
  if (M == 0) return MOE_OK;
  MOE_REQUIRE(x && data && scale, "quantize_fp8: null pointer");
  MOE_REQUIRE(aligned16(x, data), "quantize_fp8: x and data must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (src_type == 1)
    return launch_rows<false, Fp32Unit>(x, M, K, nullptr, nullptr, 0, 0, 0, data,
                              scale, s, "quantize_fp8 launch");
  return launch_rows<false, Bf16Unit>(x, M, K, nullptr, nullptr, 0, 0, 0,
                            data, scale, s, "quantize_fp8 launch");
}

extern "C" int moe_permute_fp8(const void* x, const int64_t* row_id_map_te,
                               const int64_t* topk_experts, int32_t k, void* data, void* scale,
                               int64_t T, int64_t H, int64_t E, int64_t num_out,
                               moe_stream_t stream) {
  MOE_REQUIRE(T >= 0 && E >= 1 && num_out >= 0, "permute_fp8: bad shape T=%lld E=%lld rows=%lld",
              (long long)T, (long long)E, (long long)num_out);
  MOE_REQUIRE(H >= 16 && H % 16 == 0 && H < (1ll << 31),
              "permute_fp8: H=%lld must be a positive multiple of 16", (long long)H);
  MOE_REQUIRE(k >= 1 && k <= kMaxTopk, "permute_fp8: k=%d out of [1,%d]", k, kMaxTopk);
  if (T == 0 || num_out == 0) return MOE_OK;
  MOE_REQUIRE(x && row_id_map_te && topk_experts && data && scale, "permute_fp8: null pointer");
  MOE_REQUIRE(aligned16(x, data), "permute_fp8: x and data must be 16-byte aligned");
  return launch_rows<true, Bf16Unit>(x, T, H, row_id_map_te, topk_experts,
                           k, E, num_out, data, scale, reinterpret_cast<cudaStream_t>(stream),
                           "permute_fp8 launch");
}

extern "C" int moe_quantize_fp8_weight(const void* w, int32_t src_type, int64_t G, int64_t N,
                                       int64_t K, void* data, void* scale, moe_stream_t stream) {
  MOE_REQUIRE(src_type == 0 || src_type == 1,
              "quantize_fp8_weight: src_type must be 0 (bf16) or 1 (fp32)");
  MOE_REQUIRE(G >= 0 && G <= 65535, "quantize_fp8_weight: G=%lld out of [0,65535]", (long long)G);
  MOE_REQUIRE(N >= 1 && (N + kBlock - 1) / kBlock <= 65535, "quantize_fp8_weight: N=%lld out of range",
              (long long)N);
  MOE_REQUIRE(K >= 16 && K % 16 == 0 && K < (1ll << 31),
              "quantize_fp8_weight: K=%lld must be a positive multiple of 16", (long long)K);
  if (G == 0) return MOE_OK;
  MOE_REQUIRE(w && data && scale, "quantize_fp8_weight: null pointer");
  MOE_REQUIRE(aligned16(w, data), "quantize_fp8_weight: w and data must be 16-byte aligned");
  const int units = static_cast<int>(K / kUnit);
  const int kb = static_cast<int>((K + kBlock - 1) / kBlock);
  const dim3 grid(kb, static_cast<unsigned>((N + kBlock - 1) / kBlock), static_cast<unsigned>(G));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (src_type == 1)
    quantize_weight_kernel<Fp32Unit, 2><<<grid, 512, 0, s>>>(
        static_cast<const float*>(w), N, units, kb, static_cast<uint4*>(data),
        static_cast<uint8_t*>(scale));
  else
    quantize_weight_kernel<Bf16Unit, 4><<<grid, 256, 0, s>>>(
        static_cast<const __nv_bfloat16*>(w), N, units, kb, static_cast<uint4*>(data),
        static_cast<uint8_t*>(scale));
  MOE_CUDA_CHECK_LAUNCH("quantize_fp8_weight launch");
  return MOE_OK;
}

extern "C" int moe_dequantize_fp8(const void* data, const void* scale, int64_t M, int64_t K,
                                  void* out, moe_stream_t stream) {
  MOE_REQUIRE(M >= 0 && K >= 16 && K % 16 == 0 && K < (1ll << 31),
              "dequantize_fp8: M=%lld K=%lld (K must be a positive multiple of 16)", (long long)M,
              (long long)K);
  if (M == 0) return MOE_OK;
  MOE_REQUIRE(data && scale && out, "dequantize_fp8: null pointer");
  MOE_REQUIRE(aligned16(data, out), "dequantize_fp8: data and out must be 16-byte aligned");
  const int units = static_cast<int>(K / 8);
  const int64_t blocks = (M + kReadRows - 1) / kReadRows;
  dequantize_rows_kernel<<<static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20)),
                           row_threads(units), 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint2*>(data), static_cast<const uint8_t*>(scale), M, units,
      static_cast<int>((K + kBlock - 1) / kBlock), static_cast<uint4*>(out));
  MOE_CUDA_CHECK_LAUNCH("dequantize_fp8 launch");
  return MOE_OK;
}
