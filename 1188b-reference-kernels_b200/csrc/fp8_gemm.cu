// Grouped GEMM of e4m3 operands with one power-of-two scale for 128 values.
//
//   out[r, n] = sum over k of (xq[r,k] 2^ex[r,k/128]) (wq[n,k] 2^ew[n/128,k/128])   for the rows r of group g
//
// The scales are E8M0 bytes, which tcgen05.mma.kind::mxf8f6f4.block_scale
// multiplies in itself, so the fp32 accumulation in TMEM needs no pass of its
// own over partial sums. The unit's scale granularity is 32 along K: the four
// K=32 instructions of a 128-block name the same byte. Scales sit in TMEM, a
// 32-bit cell per row holding the bytes of four consecutive 128-blocks; the
// instruction descriptor selects the byte (k-block index & 3).
//
// One persistent CTA per SM, 224 threads:
//   warp 0     TMA producer: 128 x 128 A tile and two 128 x 128 B tiles (48 KB) per stage and 128-block of K
//   warp 1     TMEM owner; one thread copies scales to TMEM (tcgen05.cp) and issues the MMAs (M=128, N=256, K=32)
//   warps 2-5  epilogue, one row per thread
//   warp 6     scales: global memory -> shared memory in the layout of tcgen05.cp, one 512-deep K group ahead
// Rows are described by the group table of moe_grouped_gemm_plan_*. Every
// wait is bounded (2 s): on timeout the kernel records an error word, drains
// its copies and MMAs, frees TMEM and returns.
#include <mutex>

#include "fp8.cuh"
#include "group_table.cuh"
#include "swiglu.cuh"

namespace moe {
namespace g8 {

using fp8::kBlock;

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int kStages = 4;
constexpr int kThreads = 224;
constexpr uint32_t kTileBytes = 128 * 128;             // 128 rows (or reduction rows) x 128 bytes
constexpr uint32_t kStageBytes = 3 * kTileBytes;       // A, B columns 0..127, B columns 128..255
constexpr int kSfStages = 2;
constexpr uint32_t kSfBytes = 512 + 1024;              // 128 A rows and 256 B rows, one 32-bit cell each
constexpr size_t kSmemBytes = 1024 + kStages * kStageBytes + kSfStages * kSfBytes + 256;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSfCol = 480;                       // TMEM columns of the scales: 4 for A, 8 for B per stage

constexpr int kErrProducer = 1;
constexpr int kErrMma = 2;
constexpr int kErrEpilogue = 3;
constexpr int kErrScales = 5;

struct Params {
  const int32_t* row_start;
  const int32_t* rows;
  const int32_t* widx;
  int32_t* err;
  const uint8_t* xs;   // [x_rows, num_kb]
  const uint8_t* ws;   // NK: [num_w, n_blocks, num_kb]; KN: [num_w, num_kb, n_blocks]
  void* out;           // bf16 [x_rows, N], or e4m3 [x_rows, F]
  uint8_t* out_scale;  // [x_rows, F / 128] (epilogue 1)
  __nv_bfloat16* pre;  // bf16 [x_rows, N] gate|up (epilogue 1, nullable)
  int64_t x_rows;
  int G;
  int num_w;
  int n;         // columns of the product (2F for epilogue 1)
  int f_half;    // F for epilogue 1
  int num_kb;    // 128-blocks along K
  int n_blocks;  // 128-blocks along N
  int n_tiles;
  int b_mn;      // weight is [num_w, K, N]: B staged MN-major
  int epilogue;  // 0 bf16 out; 1 SwiGLU -> e4m3 rows
};

// Instruction descriptor, kind::mxf8f6f4: D fp32, A and B e4m3, E8M0 scales;
// sf_id selects the byte of a scale cell, the same for A and B.
__host__ __device__ constexpr uint32_t idesc_mxf8(int m, int n, bool b_mn) {
  return (b_mn ? 1u << 16 : 0u)                    // B MN-major
         | (static_cast<uint32_t>(n >> 3) << 17)   // N / 8
         | (1u << 23)                              // scale type E8M0
         | (static_cast<uint32_t>(m >> 7) << 27);  // M / 128
}
MOE_DEVICE uint32_t with_sf_id(uint32_t idesc, uint32_t id) {
  return idesc | (id << 4) | (id << 29);
}

// Shared-memory descriptor of a scale tile for tcgen05.cp: 32 rows of 16
// bytes, unswizzled, 8-row groups 128 bytes apart.
MOE_DEVICE uint64_t sf_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 16;
  d |= static_cast<uint64_t>(128u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  return d;
}

MOE_DEVICE void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

MOE_DEVICE void umma_mxf8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], "
      "[%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

MOE_DEVICE void tma_load_3d(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z,
                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

MOE_DEVICE bool wait_drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitTimeoutNs) return false;
  return true;
}

MOE_DEVICE void raise_abort(volatile int* abort_flag, int32_t* err, int code) {
  atomicCAS(err, 0, code);
  *abort_flag = 1;
  __threadfence_block();
}

// Tile t of the launch: group, then N-tile by N-tile with the group's M-tiles
// innermost (they share the weight tile). Indices only grow, so the walk only
// moves forward.
struct Tile {
  int g, m, n;
};
struct Walker {
  const int32_t* rows;
  int G, n_tiles;
  int g = 0, mt = -1;
  long long base = 0;
  __device__ bool locate(long long t, Tile& tile) {
    while (g < G) {
      if (mt < 0) mt = (max(rows[g], 0) + BM - 1) / BM;
      const long long cnt = static_cast<long long>(mt) * n_tiles;
      if (t < base + cnt) break;
      base += cnt;
      ++g;
      mt = -1;
    }
    if (g >= G) return false;
    const int local = static_cast<int>(t - base);
    tile.g = g;
    tile.n = local / mt;
    tile.m = local % mt;
    return true;
  }
};

// Four scale bytes kb0..kb0+3 of a row of `num_kb` bytes at p (1.0 past its
// end), `step` bytes apart.
MOE_DEVICE uint32_t scale_cell(const uint8_t* p, int64_t step, int kb0, int num_kb) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = kb0 + i < num_kb ? __ldg(p + (kb0 + i) * step) : fp8::kOne;
    w |= b << (8 * i);
  }
  return w;
}

__global__ void __launch_bounds__(kThreads, 1)
    grouped_gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a,
                            const __grid_constant__ CUtensorMap tmap_b, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_addr);
  uint8_t* sf_ptr = base_ptr + kStages * kStageBytes;
  const uint32_t sf_base = base + kStages * kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sf_ptr + kSfStages * kSfBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto sf_full = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
  auto sf_empty = [&](int s) { return bar0 + 8u * (2 * kStages + kSfStages + s); };
  const uint32_t acc_full = bar0 + 8u * (2 * kStages + 2 * kSfStages);
  const uint32_t acc_empty = acc_full + 8u;
  const uint32_t drain_bar = acc_full + 16u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 2 * kSfStages + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id();
  const int lane = lane_id();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < kSfStages; ++s) {
      mbar_init(sf_full(s), 1);
      mbar_init(sf_empty(s), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 4);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int groups4 = (p.num_kb + 3) / 4;  // 512-deep K groups, one scale cell each

  Walker walker{p.rows, p.G, p.n_tiles};
  Tile tile;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued[kStages];
#pragma unroll
      for (int s = 0; s < kStages; ++s) issued[s] = -1;
      bool ok = true;
      for (long long t = blockIdx.x; ok && walker.locate(t, tile); t += gridDim.x) {
        const int row0 = p.row_start[tile.g] + tile.m * BM;
        const int wi = p.widx[tile.g];
        const int n0 = p.epilogue == 1 ? tile.n * 128 : tile.n * BN;
        const int n1 = p.epilogue == 1 ? p.f_half + n0 : n0 + 128;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t sa = base + stage * kStageBytes;
          mbar_arrive_expect_tx(full_bar(stage), kStageBytes);
          tma_load_3d(sa, &tmap_a, kb * 128, row0, 0, full_bar(stage));
          if (p.b_mn) {
            tma_load_3d(sa + kTileBytes, &tmap_b, n0, kb * 128, wi, full_bar(stage));
            tma_load_3d(sa + 2 * kTileBytes, &tmap_b, n1, kb * 128, wi, full_bar(stage));
          } else {
            tma_load_3d(sa + kTileBytes, &tmap_b, kb * 128, n0, wi, full_bar(stage));
            tma_load_3d(sa + 2 * kTileBytes, &tmap_b, kb * 128, n1, wi, full_bar(stage));
          }
          issued[stage] = static_cast<int>(phase);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        raise_abort(abort_flag, p.err, kErrProducer);
        for (int s = 0; s < kStages; ++s)
          if (issued[s] >= 0) wait_drain(full_bar(s), static_cast<uint32_t>(issued[s]));
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      const uint32_t idesc = idesc_mxf8(BM, BN, p.b_mn != 0);
      // +32 values along K: 32 bytes inside a K-major swizzle row; 32 reduction
      // rows (four 1024-byte groups of 8) of an MN-major tile.
      const uint64_t bstep = p.b_mn ? 4096ull >> 4 : 32ull >> 4;
      int stage = 0, sf = 0;
      uint32_t phase = 0, sf_phase = 0, acc_phase = 0;
      bool ok = true, issued_any = false;
      for (long long t = blockIdx.x; ok && walker.locate(t, tile); t += gridDim.x) {
        if (!mbar_wait(acc_empty, acc_phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kg = 0; kg < groups4 && ok; ++kg) {
          if (!mbar_wait(sf_full(sf), sf_phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfa = tmem + kSfCol + static_cast<uint32_t>(sf) * 12u;
          const uint32_t sfb = sfa + 4u;
          const uint32_t src = sf_base + static_cast<uint32_t>(sf) * kSfBytes;
          tmem_copy_scales(sfa, sf_desc(src));
          tmem_copy_scales(sfb, sf_desc(src + 512u));
          tmem_copy_scales(sfb + 4u, sf_desc(src + 1024u));
          issued_any = true;
          const int kb1 = min(kg * 4 + 4, p.num_kb);
          for (int kb = kg * 4; kb < kb1; ++kb) {
            if (!mbar_wait(full_bar(stage), phase, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = base + stage * kStageBytes;
            const uint64_t ad = umma_desc_k_sw128(sa);
            const uint64_t bd = p.b_mn ? umma_desc_mn_sw128(sa + kTileBytes, kTileBytes)
                                       : umma_desc_k_sw128(sa + kTileBytes);
            const uint32_t id = with_sf_id(idesc, static_cast<uint32_t>(kb & 3));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_mxf8(tmem, ad + 2ull * k, bd + bstep * k, id, sfa, sfb, (kb | k) != 0 ? 1u : 0u);
            umma_commit(empty_bar(stage));
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          umma_commit(sf_empty(sf));
          if (++sf == kSfStages) {
            sf = 0;
            sf_phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(acc_full);
        acc_phase ^= 1u;
      }
      if (!ok) {
        raise_abort(abort_flag, p.err, kErrMma);
        if (issued_any) {
          umma_commit(drain_bar);
          wait_drain(drain_bar, 0);
        }
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    // ---------------------------------------------------------------- scales
    int sf = 0;
    uint32_t sf_phase = 0;
    bool ok = true;
    for (long long t = blockIdx.x; ok && walker.locate(t, tile); t += gridDim.x) {
      const int64_t row0 = static_cast<int64_t>(p.row_start[tile.g]) + tile.m * BM;
      const int64_t wi = p.widx[tile.g];
      const int nb0 = p.epilogue == 1 ? tile.n : tile.n * 2;
      const int nb1 = p.epilogue == 1 ? p.f_half / 128 + tile.n : nb0 + 1;
      for (int kg = 0; kg < groups4; ++kg) {
        uint32_t a[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t r = row0 + c * 32 + lane;
          a[c] = r < p.x_rows ? scale_cell(p.xs + r * p.num_kb, 1, kg * 4, p.num_kb) : 0x7F7F7F7Fu;
        }
        uint32_t b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nb = h ? nb1 : nb0;
          const int64_t w0 = p.b_mn ? wi * p.num_kb * p.n_blocks + nb
                                    : (wi * p.n_blocks + nb) * p.num_kb;
          b[h] = nb < p.n_blocks && wi < p.num_w
                     ? scale_cell(p.ws + w0, p.b_mn ? p.n_blocks : 1, kg * 4, p.num_kb)
                     : 0x7F7F7F7Fu;
        }
        if (!mbar_wait(sf_empty(sf), sf_phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        uint4* dst = reinterpret_cast<uint4*>(sf_ptr + sf * kSfBytes) + lane;
        dst[0] = make_uint4(a[0], a[1], a[2], a[3]);
        dst[32] = make_uint4(b[0], b[0], b[0], b[0]);
        dst[64] = make_uint4(b[1], b[1], b[1], b[1]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(sf_full(sf));
        if (++sf == kSfStages) {
          sf = 0;
          sf_phase ^= 1u;
        }
      }
    }
    if (!ok && lane == 0) raise_abort(abort_flag, p.err, kErrScales);
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    const int quad = warp & 3;  // TMEM lanes 32*quad .. of this warp
    uint32_t acc_phase = 0;
    bool ok = true;
    for (long long t = blockIdx.x; walker.locate(t, tile); t += gridDim.x) {
      if (!mbar_wait(acc_full, acc_phase, abort_flag)) {
        ok = false;
        break;
      }
      acc_phase ^= 1u;
      tc_fence_after();
      const int m_local = tile.m * BM + quad * 32 + lane;
      const int64_t row = static_cast<int64_t>(p.row_start[tile.g]) + m_local;
      const bool rvalid = m_local < p.rows[tile.g] && row < p.x_rows;
      const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16);
      if (p.epilogue == 0) {
        const int n0 = tile.n * BN;
        __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.out) + row * p.n;
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tbase + c * 32, r);
          tmem_ld_wait();
          if (rvalid) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const int col = n0 + c * 32 + v * 8;
              if (col + 8 <= p.n) {
                uint32_t o[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  o[q] = pack_bf16x2(__uint_as_float(r[v * 8 + 2 * q]),
                                     __uint_as_float(r[v * 8 + 2 * q + 1]));
                *reinterpret_cast<uint4*>(orow + col) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          }
        }
      } else {
        // gate in columns 0..127, up in 128..255; the 128 results of a row
        // are one block of the quantised output
        float h[128];
        float amax = 0.f;
        __nv_bfloat16* prow = p.pre == nullptr ? nullptr : p.pre + row * p.n + tile.n * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t gr[32], ur[32];
          tmem_ld_32x32b_x32(tbase + c * 32, gr);
          tmem_ld_32x32b_x32(tbase + 128 + c * 32, ur);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 v = swiglu2_f32(
                make_float2(__uint_as_float(gr[2 * q]), __uint_as_float(gr[2 * q + 1])),
                make_float2(__uint_as_float(ur[2 * q]), __uint_as_float(ur[2 * q + 1])));
            h[c * 32 + 2 * q] = v.x;
            h[c * 32 + 2 * q + 1] = v.y;
            amax = fmaxf(amax, fmaxf(fp8::finite_abs(v.x), fp8::finite_abs(v.y)));
          }
          if (prow != nullptr && rvalid) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t o[4], u[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                o[q] = pack_bf16x2(__uint_as_float(gr[v * 8 + 2 * q]),
                                   __uint_as_float(gr[v * 8 + 2 * q + 1]));
                u[q] = pack_bf16x2(__uint_as_float(ur[v * 8 + 2 * q]),
                                   __uint_as_float(ur[v * 8 + 2 * q + 1]));
              }
              *reinterpret_cast<uint4*>(prow + c * 32 + v * 8) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(prow + p.f_half + c * 32 + v * 8) =
                  make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        }
        if (rvalid) {
          const uint32_t sb = fp8::scale_byte(amax);
          const float inv = fp8::inverse_scale(sb);
          uint4* orow = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + row * p.f_half +
                                                 tile.n * 128);
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int j = v * 16 + q * 4;
              o[q] = fp8::pack4(fp8::scaled(h[j], inv), fp8::scaled(h[j + 1], inv),
                                fp8::scaled(h[j + 2], inv), fp8::scaled(h[j + 3], inv));
            }
            orow[v] = make_uint4(o[0], o[1], o[2], o[3]);
          }
          p.out_scale[row * (p.f_half / 128) + tile.n] = static_cast<uint8_t>(sb);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
    }
    if (!ok && lane == 0) raise_abort(abort_flag, p.err, kErrEpilogue);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// 3-D tensor map over bytes [d2, d1, d0] (d0 contiguous), box 128 x 128 x 1,
// 128-byte swizzle; reads outside give zeros.
int make_tmap(CUtensorMap* m, const void* ptr, uint64_t d0, uint64_t d1, uint64_t d2) {
  auto encode = gg::get_encode_fn();
  if (encode == nullptr) {
    set_last_error("grouped_gemm_fp8: cuTensorMapEncodeTiled unavailable");
    return MOE_ERR_CUDA;
  }
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {d0, d0 * d1};
  cuuint32_t box[3] = {128u, 128u, 1u};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUresult r =
      encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("grouped_gemm_fp8: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return MOE_ERR_CUDA;
  }
  return MOE_OK;
}

int ensure_smem_attr(int dev) {
  static std::mutex mu;
  static bool done[64] = {};
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && dev < 64 && done[dev]) return MOE_OK;
  MOE_CUDA_CALL(cudaFuncSetAttribute(grouped_gemm_fp8_kernel,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(kSmemBytes)),
                "cudaFuncSetAttribute(grouped_gemm_fp8)");
  if (dev >= 0 && dev < 64) done[dev] = true;
  return MOE_OK;
}

}  // namespace g8
}  // namespace moe

using namespace moe;

extern "C" int moe_grouped_gemm_fp8(const void* x, const void* x_scale, const void* w,
                                    const void* w_scale, void* out, void* out_scale, void* pre,
                                    int64_t x_rows, int64_t G, int64_t num_w, int64_t N, int64_t K,
                                    int32_t w_kn, int32_t epilogue, const void* workspace,
                                    size_t workspace_bytes, moe_stream_t stream) {
  MOE_REQUIRE(epilogue == 0 || epilogue == 1, "grouped_gemm_fp8: epilogue must be 0 or 1");
  MOE_REQUIRE(G >= 1 && num_w >= 1, "grouped_gemm_fp8: G=%lld num_w=%lld", (long long)G,
              (long long)num_w);
  MOE_REQUIRE(x_rows >= 0 && x_rows < (1ll << 31), "grouped_gemm_fp8: x_rows=%lld out of range",
              (long long)x_rows);
  MOE_REQUIRE(K >= 16 && K % 16 == 0 && K < (1ll << 31),
              "grouped_gemm_fp8: K=%lld must be a positive multiple of 16", (long long)K);
  MOE_REQUIRE(N >= 8 && N % 8 == 0 && N < (1ll << 30),
              "grouped_gemm_fp8: N=%lld must be a positive multiple of 8", (long long)N);
  MOE_REQUIRE(!w_kn || N % 16 == 0, "grouped_gemm_fp8: w [G,K,N] needs N %% 16 == 0, N=%lld",
              (long long)N);
  MOE_REQUIRE(epilogue == 0 || !w_kn, "grouped_gemm_fp8: the SwiGLU epilogue needs w [G,N,K]");
  MOE_REQUIRE(epilogue == 0 || N % 256 == 0,
              "grouped_gemm_fp8: the SwiGLU epilogue needs N = 2F with F %% 128 == 0, N=%lld",
              (long long)N);
  MOE_REQUIRE(num_w < (1ll << 31), "grouped_gemm_fp8: num_w too large");
  MOE_REQUIRE(epilogue == 1 || pre == nullptr, "grouped_gemm_fp8: pre needs the SwiGLU epilogue");
  MOE_REQUIRE(workspace != nullptr && workspace_bytes >= gg::ws_bytes(G),
              "grouped_gemm_fp8: workspace too small (%zu < %zu)", workspace_bytes, gg::ws_bytes(G));
  MOE_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
              "grouped_gemm_fp8: workspace must be 256-byte aligned");
  if (x_rows == 0) return MOE_OK;
  MOE_REQUIRE(x && x_scale && w && w_scale && out, "grouped_gemm_fp8: null pointer");
  MOE_REQUIRE(epilogue == 0 || out_scale != nullptr, "grouped_gemm_fp8: null out_scale");
  MOE_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) |
                reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pre)) &
               15) == 0,
              "grouped_gemm_fp8: x, w, out and pre must be 16-byte aligned");
  int dev = 0;
  MOE_CUDA_CALL(cudaGetDevice(&dev), "cudaGetDevice");
  int st = g8::ensure_smem_attr(dev);
  if (st) return st;

  CUtensorMap ta, tb;
  st = g8::make_tmap(&ta, x, static_cast<uint64_t>(K), static_cast<uint64_t>(x_rows), 1);
  if (st) return st;
  st = w_kn ? g8::make_tmap(&tb, w, static_cast<uint64_t>(N), static_cast<uint64_t>(K),
                            static_cast<uint64_t>(num_w))
            : g8::make_tmap(&tb, w, static_cast<uint64_t>(K), static_cast<uint64_t>(N),
                            static_cast<uint64_t>(num_w));
  if (st) return st;

  const gg::WsLayout l = gg::ws_layout(workspace, G);
  g8::Params p;
  p.row_start = l.row_start;
  p.rows = l.rows;
  p.widx = l.widx;
  p.err = l.err;
  p.xs = static_cast<const uint8_t*>(x_scale);
  p.ws = static_cast<const uint8_t*>(w_scale);
  p.out = out;
  p.out_scale = static_cast<uint8_t*>(out_scale);
  p.pre = static_cast<__nv_bfloat16*>(pre);
  p.x_rows = x_rows;
  p.G = static_cast<int>(G);
  p.num_w = static_cast<int>(num_w);
  p.n = static_cast<int>(N);
  p.f_half = epilogue == 1 ? static_cast<int>(N / 2) : 0;
  p.num_kb = static_cast<int>((K + 127) / 128);
  p.n_blocks = static_cast<int>((N + 127) / 128);
  p.n_tiles = epilogue == 1 ? p.f_half / 128 : static_cast<int>((N + g8::BN - 1) / g8::BN);
  p.b_mn = w_kn ? 1 : 0;
  p.epilogue = epilogue;
  g8::grouped_gemm_fp8_kernel<<<num_sms(dev), g8::kThreads, g8::kSmemBytes,
                                reinterpret_cast<cudaStream_t>(stream)>>>(ta, tb, p);
  MOE_CUDA_CHECK_LAUNCH("grouped_gemm_fp8 launch");
  return MOE_OK;
}
