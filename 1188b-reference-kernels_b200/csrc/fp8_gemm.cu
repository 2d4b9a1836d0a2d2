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
// Three forms of one kernel, persistent, 224 threads a CTA:
//   pair    clusters of two CTAs (cta_group::2) on 256 x 256 tiles, for groups of more than 128 rows: each CTA
//           stages its own 128 A rows and half of the B tile (32 KB a 128-block of K, six stages), the leader
//           issues M=256, N=256 MMAs over both shared memories into both TMEMs
//   single  128 x 256 tiles (48 KB a 128-block, four stages) for smaller groups, where the weight stream is
//           what takes the time
//   few     the same for calls of at most 32 rows in all: A tiles of 32 rows, so that six stages fit and half as
//           much weight again is on its way (K 7168, N 4096, 32 rows over 20 groups: 133 -> 119 us; one row: 38 ->
//           32 us). The MMAs read 128 rows from the A tile's place all the same; what lies behind it only enters
//           rows that nobody stores. As a launch of its own beside the single form it gave nothing (512 rows over
//           32 groups 181 against 183 us, 768 rows of which half in larger groups 193 against 183)
// Warps:
//   warp 0     TMA producer
//   warp 1     TMEM owner; copies scales to TMEM (tcgen05.cp) and issues the MMAs (K=32)
//   warps 2-5  epilogue, one row per thread
//   warp 6     scales: global memory -> shared memory in the layout of tcgen05.cp, ahead of the MMAs. Every CTA
//              keeps the scales of its own 128 rows and of all 256 columns
// TMEM: two accumulators of 256 columns and two scale buffers of 12 would need
// 536 of 512 columns, so accumulator 1 starts at column 224 and the two share
// the 32 columns 224..255. The epilogue reads those first and hands them over
// on a barrier of their own (`shared`), which the next tile's MMAs wait for;
// the rest of a tile's epilogue overlaps the next tile's mainloop.
// Measured (one B200 at its 1000 W, 1.2 to 1.5 GHz): 32 groups of 1024 rows,
// K 7168, N 4096 with SwiGLU 0.88-0.92 ms, K 2048, N 7168 0.48-0.51 ms (2150
// and 1950 TFLOP/s, at the power limit with the tensor pipe busy 68 to 72 %: it
// stands still at the hand-over between tiles and for the scale copies); 20
// groups of one or two rows 103-129 us by box, 4.6-5.7 TB/s of weights.
// Rows are described by the group table of moe_grouped_gemm_plan_*. Every
// wait is bounded (2 s): on timeout the kernel records an error word, drains
// its copies and MMAs, frees TMEM and returns.
#include <algorithm>
#include <mutex>

#include "fp8.cuh"
#include "group_table.cuh"
#include "swiglu.cuh"

namespace moe {
namespace g8 {

using fp8::kBlock;
using gg::Tile;
using gg::raise_abort;
using gg::wait_drain;

constexpr int BN = 256;
constexpr int kThreads = 224;
constexpr uint32_t kTileBytes = 128 * 128;  // 128 rows (or reduction rows) x 128 bytes
constexpr int kFewRows = 32;   // rows of the small A box, and of a call of the few form
constexpr int kSfStages = 6;   // scale buffers in shared memory
constexpr int kSfTmem = 2;     // and in TMEM
constexpr uint32_t kSfBytes = 512 + 1024;    // 128 A rows and 256 B rows, one 32-bit cell each
constexpr uint32_t kEpiWarpBytes = 4096;     // per epilogue warp: two 32 x 64-byte boxes or one 32 x 128-byte box

enum Form { kPairForm, kSingleForm, kFewForm };

template <Form kForm>
struct Shape {
  static constexpr int kTileM = kForm == kPairForm ? 256 : 128;
  static constexpr int kStages = kForm == kSingleForm ? 4 : 6;
  static constexpr uint32_t kABytes = kForm == kFewForm ? kFewRows * 128u : kTileBytes;
  static constexpr uint32_t kStageBytes = kABytes + (kForm == kPairForm ? 1 : 2) * kTileBytes;  // of one CTA
  static constexpr uint32_t kEpiBytes = kForm == kFewForm ? 0u : 4 * kEpiWarpBytes;
  static constexpr size_t kSmemBytes =
      1024 + kStages * kStageBytes + kEpiBytes + kSfStages * kSfBytes + 512;
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kAccCol1 = 224;  // first column of accumulator 1
constexpr uint32_t kSfCol = 480;    // TMEM columns of the scales: 4 for A, 8 for B per buffer

// Groups of at most so many rows go to the single form, which keeps more of the
// weight in flight; above, one pair tile does for two single ones. 32 groups of
// 100 rows (K 7168, N 4096): 183 us single, 217 pair; 40 of 200 ([K,N], K 4096,
// N 5120): 253 single, 229 pair.
constexpr int kSingleRows = 128;
// Calls of at least so many rows a group on average leave small groups to the
// pairs as well, and make one launch (K 2048, N 7168: 32 groups of 1024 rows 430
// -> 418 us, 16 of 100 and 924 in turn 157 -> 141, 30 of 4 rows beside 2 of 8132
// 298 and 300; K 7168, N 4096: one of 1024 42 -> 39, 16 of 100 and 924 252 -> 255).
constexpr int64_t kOneLaunchRows = 512;
constexpr int64_t kSlabBytes = 32ll << 20;  // weight bytes walked per pass: they stay in L2 beside the rows

constexpr int kErrProducer = 1;
constexpr int kErrMma = 2;
constexpr int kErrEpilogue = 3;
constexpr int kErrScales = 5;

// Scale bytes at 4 kg .. 4 kg + 3 of row `row` of a [rows, num_kb] byte matrix
// of `total` bytes, 1.0 past the row's end. Rows that are whole words take one
// load, other rows of a word-aligned matrix two neighbouring words.
struct ScaleRows {
  const uint8_t* p;
  int64_t total;
  int num_kb;
  bool aligned;  // p is a multiple of 4
};

struct Params {
  const int32_t* row_start;
  const int32_t* rows;
  const int32_t* widx;
  int32_t* err;
  ScaleRows xs;        // [x_rows, num_kb]
  ScaleRows ws;        // NK: [num_w, n_blocks, num_kb]; KN: [num_w, num_kb, n_blocks] (by bytes)
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
  int above, most;  // rows of the groups that this launch takes: (above, most]
  int n_chunk;   // pair kernel: N-tiles walked per pass over a group's rows
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

// The same in every lane, and known to be so by the compiler.
MOE_DEVICE uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
MOE_DEVICE bool all_lanes(bool v) { return __all_sync(0xffffffffu, v) != 0; }

// Bytes of A that a CTA loads of `rows` rows.
MOE_DEVICE uint32_t a_bytes(int rows) {
  return rows <= 0 ? 0u : rows <= kFewRows ? kFewRows * 128u : kTileBytes;
}

// Tile load into this CTA's shared memory; a pair counts the bytes on the
// leader's barrier.
template <bool kPair>
MOE_DEVICE void tma_load_3d(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z,
                            uint32_t bar, uint64_t policy) {
  if constexpr (kPair)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        ".L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        ".L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
}

MOE_DEVICE uint32_t scale_cell(const ScaleRows& m, int64_t row, int kg) {
  const int64_t at = row * m.num_kb + kg * 4;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(m.p) + (at >> 2);
  if (m.aligned && m.num_kb % 4 == 0) return __ldg(words);
  uint32_t w = 0;
  if (m.aligned && (at & ~3ll) + 8 <= m.total) {
    w = __funnelshift_r(__ldg(words), __ldg(words + 1), static_cast<uint32_t>(at & 3) * 8u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < m.total) w |= static_cast<uint32_t>(__ldg(m.p + at + i)) << (8 * i);
  }
  const int live = m.num_kb - kg * 4;  // bytes before the row's end
  if (live < 4) {
    const uint32_t mask = (1u << (8 * live)) - 1u;
    w = (w & mask) | (0x7F7F7F7Fu & ~mask);
  }
  return w;
}

// This lane's scale cells of one 512-deep K group: rows row0 + lane + 32 c of
// x, and weight row blocks nb0, nb1 (the same cell for all 128 of a block).
MOE_DEVICE void load_scale_cells(const Params& p, int64_t row0, int64_t wi, int nb0, int nb1, int kg,
                                 int lane, uint32_t (&a)[4], uint32_t (&b)[2]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int64_t r = row0 + c * 32 + lane;
    a[c] = static_cast<uint64_t>(r) < static_cast<uint64_t>(p.x_rows) ? scale_cell(p.xs, r, kg) : 0x7F7F7F7Fu;
  }
  if (p.b_mn) {  // bytes of one block lie a row of blocks apart: a lane loads each
    const int nb = lane & 4 ? nb1 : nb0;
    const int kb = kg * 4 + (lane & 3);
    uint32_t v = fp8::kOne;
    if (lane < 8 && nb < p.n_blocks && wi < p.num_w && kb < p.num_kb)
      v = __ldg(p.ws.p + (wi * p.num_kb + kb) * p.n_blocks + nb);
    v <<= 8 * (lane & 3);
    v |= __shfl_xor_sync(0xffffffffu, v, 1);
    v |= __shfl_xor_sync(0xffffffffu, v, 2);
    b[0] = __shfl_sync(0xffffffffu, v, 0);
    b[1] = __shfl_sync(0xffffffffu, v, 4);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int nb = h ? nb1 : nb0;
    b[h] = nb < p.n_blocks && wi < p.num_w
               ? scale_cell(p.ws, wi * p.n_blocks + nb, kg)
               : 0x7F7F7F7Fu;
  }
}

MOE_DEVICE void tmem_copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}

MOE_DEVICE void umma_mxf8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                               uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], "
      "[%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

MOE_DEVICE void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// What the two forms do differently around the same instruction.
template <bool kPair>
struct Op {
  static MOE_DEVICE bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if constexpr (kPair) return mbar_wait_cluster(bar, parity, abort_flag);
    return mbar_wait(bar, parity, abort_flag);
  }
  static MOE_DEVICE bool try_wait(uint32_t bar, uint32_t parity) {
    if constexpr (kPair) return mbar_try_wait_cluster(bar, parity);
    return mbar_try_wait(bar, parity);
  }
  // a commit that both CTAs see / that the issuing CTA alone needs
  static MOE_DEVICE void commit(uint32_t bar) {
    if constexpr (kPair)
      umma_commit_pair(bar, 0x3);
    else
      umma_commit(bar);
  }
  static MOE_DEVICE void commit_own(uint32_t bar) {
    if constexpr (kPair)
      umma_commit_pair(bar, 0x1);
    else
      umma_commit(bar);
  }
  static MOE_DEVICE uint32_t leader(uint32_t bar) {
    if constexpr (kPair) return map_to_rank(bar, 0);
    return bar;
  }
  static MOE_DEVICE void arrive(uint32_t leader_bar) {
    if constexpr (kPair)
      mbar_arrive_cluster(leader_bar);
    else
      mbar_arrive(leader_bar);
  }
  static MOE_DEVICE void copy_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (kPair)
      tmem_copy_scales_pair(taddr, desc);
    else
      tmem_copy_scales(taddr, desc);
  }
  static MOE_DEVICE void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                             uint32_t sfb, uint32_t accumulate) {
    if constexpr (kPair)
      umma_mxf8_pair(d, a, b, idesc, sfa, sfb, accumulate);
    else
      umma_mxf8(d, a, b, idesc, sfa, sfb, accumulate);
  }
};

template <Form kForm>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a,
                            const __grid_constant__ CUtensorMap tmap_a_few,
                            const __grid_constant__ CUtensorMap tmap_b,
                            const __grid_constant__ CUtensorMap tmap_out,
                            const __grid_constant__ CUtensorMap tmap_pre, const Params p) {
  constexpr bool kPair = kForm == kPairForm;
  constexpr bool kFew = kForm == kFewForm;
  using O = Op<kPair>;
  constexpr int kTileM = Shape<kForm>::kTileM;
  constexpr int kS = Shape<kForm>::kStages;
  constexpr uint32_t kSB = Shape<kForm>::kStageBytes;
  constexpr uint32_t kAB = Shape<kForm>::kABytes;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_addr);
  const uint32_t epi_base = base + kS * kSB;
  const uint32_t sf_base = epi_base + Shape<kForm>::kEpiBytes;
  uint8_t* sf_ptr = base_ptr + kS * kSB + Shape<kForm>::kEpiBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sf_ptr + kSfStages * kSfBytes);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kS + s); };
  auto sf_full = [&](int s) { return bar0 + 8u * (2 * kS + s); };
  auto sf_empty = [&](int s) { return bar0 + 8u * (2 * kS + kSfStages + s); };
  auto sf_used = [&](int b) { return bar0 + 8u * (2 * kS + 2 * kSfStages + b); };
  auto acc_full = [&](int a) { return bar0 + 8u * (2 * kS + 2 * kSfStages + kSfTmem + a); };
  auto acc_empty = [&](int a) { return bar0 + 8u * (2 * kS + 2 * kSfStages + kSfTmem + 2 + a); };
  const uint32_t shared_bar = bar0 + 8u * (2 * kS + 2 * kSfStages + kSfTmem + 4);
  const uint32_t drain_bar = shared_bar + 8u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kS + 2 * kSfStages + kSfTmem + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t rank = kPair ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const long long cid = kPair ? cluster_id_x() : blockIdx.x;
  const long long ncl = kPair ? num_clusters_x() : gridDim.x;
  const int warp = static_cast<int>(uniform(static_cast<uint32_t>(warp_id())));
  const int lane = lane_id();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kS; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < kSfStages; ++s) {
      mbar_init(sf_full(s), kPair ? 2 : 1);  // the scale warp of each CTA
      mbar_init(sf_empty(s), 1);
    }
    for (int b = 0; b < kSfTmem; ++b) mbar_init(sf_used(b), 1);
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), kPair ? 8 : 4);  // four epilogue warps in each CTA
    }
    mbar_init(shared_bar, kPair ? 8 : 4);
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();  // barriers of both CTAs initialised before any remote use
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  // The single form's launch behind this one works on other groups: its CTAs
  // start where this one's have left ([K,N], K 4096, N 5120, 40 groups of 20 to
  // 380 rows: 291 -> 278 us).
  if constexpr (kPair) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int groups4 = (p.num_kb + 3) / 4;

  gg::WalkerRT<kTileM> walker{p.rows, p.G, p.n_tiles, 1 << 20, p.n_chunk, p.above, p.most};
  Tile tile;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      for (long long t = cid; ok && walker.locate(t, tile); t += ncl) {
        const int row0 = p.row_start[tile.g] + tile.m_idx * kTileM + static_cast<int>(rank) * 128;
        const int wi = p.widx[tile.g];
        // first weight row (KN: column) of the two halves of the B tile; a
        // pair's CTA loads its own
        const int n0 = p.epilogue == 1 ? tile.n_idx * 128 : tile.n_idx * BN;
        const int n1 = p.epilogue == 1 ? p.f_half + n0 : n0 + 128;
        // This CTA's A rows: none, few (a box of that height) or a whole box.
        // The rest of the tile keeps what an earlier one left there: an MMA
        // row depends on no other.
        const int rows = p.rows[tile.g];
        const int left = rows - tile.m_idx * kTileM;
        const int mine = left - static_cast<int>(rank) * 128;
        const CUtensorMap* map_a = kFew || mine <= kFewRows ? &tmap_a_few : &tmap_a;
        // (the few form has room for the small box alone, whatever the table names)
        const uint32_t bytes = a_bytes(kFew ? min(left, kFewRows) : left) + (kPair ? a_bytes(left - 128) + 2 * kTileBytes : 2 * kTileBytes);
        // A weight that one M-tile reads is not read again: it leaves L2
        // first (32 groups of 100 rows, K 2048: 122 -> 114 us).
        const uint64_t policy = rows <= kTileM ? l2_policy_evict_first() : l2_policy_evict_normal();
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t sa = base + stage * kSB;
          const uint32_t leader_full = O::leader(full_bar(stage));
          if (leader) mbar_arrive_expect_tx(full_bar(stage), bytes);
          if (mine > 0)
            tma_load_3d<kPair>(sa, map_a, kb * 128, row0, 0, leader_full, l2_policy_evict_normal());
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (kPair && h != static_cast<int>(rank)) continue;
            const int n = h ? n1 : n0;
            tma_load_3d<kPair>(sa + kAB + (kPair ? 0 : h) * kTileBytes, &tmap_b, p.b_mn ? n : kb * 128,
                               p.b_mn ? kb * 128 : n, wi, leader_full, policy);
          }
          ++issued;
          if (++stage == kS) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (ok) {
        // every stage's release lands in this CTA's shared memory: wait for the last ones
        for (long long i = issued > kS ? issued - kS : 0; i < issued; ++i)
          wait_drain(empty_bar(static_cast<int>(i % kS)), static_cast<uint32_t>(i / kS) & 1u);
      } else {
        raise_abort(abort_flag, p.err, kErrProducer);
        if (leader) {
          for (long long i = issued > kS ? issued - kS : 0; i < issued; ++i)
            wait_drain(full_bar(static_cast<int>(i % kS)), static_cast<uint32_t>(i / kS) & 1u);
        } else {
          // copies count on the leader's barrier; give them a bounded time to land
          const unsigned long long t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 200000ull) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (leader)
    // The whole warp runs the loop in step (every wait's answer is a vote) and
    // one lane issues: the operands of an MMA are then warp-uniform registers.
    // With the loop in one lane's branch an MMA took 240 clocks to issue,
    // against the unit's own 128.
    if (leader) {
      const bool issuer = lane == 0;
      const uint32_t idesc = idesc_mxf8(kTileM, BN, p.b_mn != 0);
      // +32 values along K: 32 bytes inside a K-major swizzle row; 32 reduction
      // rows (four 1024-byte groups of 8) of an MN-major tile.
      const uint64_t bstep = p.b_mn ? 4096ull >> 4 : 32ull >> 4;
      int stage = 0, sf = 0, copied = 0, used = 0, it = 0;
      uint32_t phase = 0, sf_phase = 0;
      bool ok = true, issued_any = false, ready = false;
      // Scales of the next K group (the pair's groups in order, across tiles) to the
      // TMEM buffer that the group before the current one has used. Called in
      // the middle of a group, so that neither wait is for work just issued.
      auto scales_ready = [&]() {  // without waiting
        return all_lanes(mbar_try_wait(sf_used(copied & 1), static_cast<uint32_t>((copied >> 1) & 1) ^ 1u) &&
                         O::try_wait(sf_full(sf), sf_phase));
      };
      auto copy_scales = [&](bool are_ready) {
        const uint32_t b = static_cast<uint32_t>(copied & 1);
        if (!are_ready &&
            !all_lanes(mbar_wait(sf_used(b), static_cast<uint32_t>((copied >> 1) & 1) ^ 1u, abort_flag) &&
                       O::wait(sf_full(sf), sf_phase, abort_flag)))
          return false;
        tc_fence_after();
        const uint32_t sfa = tmem + kSfCol + b * 12u;
        const uint32_t src = sf_base + static_cast<uint32_t>(sf) * kSfBytes;
        if (issuer) {
          O::copy_scales(sfa, sf_desc(src));
          O::copy_scales(sfa + 4u, sf_desc(src + 512u));
          O::copy_scales(sfa + 8u, sf_desc(src + 1024u));
          O::commit(sf_empty(sf));
        }
        __syncwarp();
        issued_any = true;
        ++copied;
        if (++sf == kSfStages) {
          sf = 0;
          sf_phase ^= 1u;
        }
        return true;
      };
      long long t = cid;
      bool more = all_lanes(walker.locate(t, tile));
      if (more) ok = copy_scales(false);
      while (ok && more) {
        t += ncl;
        more = all_lanes(walker.locate(t, tile));  // whether another tile follows
        const int acc = it & 1;
        const uint32_t d_tmem = tmem + (acc ? kAccCol1 : 0u);
        // the accumulator's last epilogue (two tiles ago) and the columns
        // shared with the other accumulator's (the last tile)
        if (!all_lanes(
                O::wait(acc_empty(acc), static_cast<uint32_t>((it >> 1) & 1) ^ 1u, abort_flag) &&
                O::wait(shared_bar, static_cast<uint32_t>(it & 1) ^ 1u, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kg = 0; kg < groups4 && ok; ++kg, ++used) {
          const uint32_t sfa = tmem + kSfCol + static_cast<uint32_t>(used & 1) * 12u;
          const int n = min(4, p.num_kb - kg * 4);
          for (int i = 0; i < n; ++i) {
            if (!ready && !all_lanes(mbar_wait(full_bar(stage), phase, abort_flag))) {
              ok = false;
              break;
            }
            // the next stage is looked at before this one's MMAs are issued,
            // so that the answer's latency does not stand between the two
            const int next = stage + 1 == kS ? 0 : stage + 1;
            ready = all_lanes(mbar_try_wait(full_bar(next), next == 0 ? phase ^ 1u : phase));
            const bool copy = i == min(2, n - 1) && (kg + 1 < groups4 || more);
            const bool sf_ready = copy && scales_ready();
            tc_fence_after();
            const uint32_t sa = base + stage * kSB;
            const uint64_t ad = umma_desc_k_sw128(sa);
            const uint64_t bd = p.b_mn ? umma_desc_mn_sw128(sa + kAB, kTileBytes)
                                       : umma_desc_k_sw128(sa + kAB);
            const uint32_t id = with_sf_id(idesc, static_cast<uint32_t>(i));
            if (issuer) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                O::mma(d_tmem, ad + 2ull * k, bd + bstep * k, id, sfa, sfa + 4u,
                      (kg | i | k) != 0 ? 1u : 0u);
              O::commit(empty_bar(stage));
            }
            __syncwarp();
            if (++stage == kS) {
              stage = 0;
              phase ^= 1u;
            }
            if (copy && !copy_scales(sf_ready)) {
              ok = false;
              break;
            }
          }
          if (!ok) break;
          if (issuer) O::commit_own(sf_used(used & 1));
        }
        if (!ok) break;
        if (issuer) O::commit(acc_full(acc));
        ++it;
      }
      if (!ok && issuer) {
        raise_abort(abort_flag, p.err, kErrMma);
        if (issued_any) {
          O::commit_own(drain_bar);
          wait_drain(drain_bar, 0);
        }
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    // ---------------------------------------------------------------- scales
    int sf = 0;
    uint32_t sf_phase = 0;
    int filled[kSfStages];
#pragma unroll
    for (int s = 0; s < kSfStages; ++s) filled[s] = -1;
    bool ok = true;
    for (long long t = cid; ok && walker.locate(t, tile); t += ncl) {
      const int64_t row0 = static_cast<int64_t>(p.row_start[tile.g]) + tile.m_idx * kTileM + rank * 128;
      const int64_t wi = p.widx[tile.g];
      const int nb0 = p.epilogue == 1 ? tile.n_idx : tile.n_idx * 2;
      const int nb1 = p.epilogue == 1 ? p.f_half / 128 + tile.n_idx : nb0 + 1;
      // One group at a time: four groups' loads at once take 7 % longer, the
      // burst of scattered words holds up the tile loads.
      for (int kg = 0; kg < groups4; ++kg) {
        uint32_t a[4], b[2];
        load_scale_cells(p, row0, wi, nb0, nb1, kg, lane, a, b);
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
        if (lane == 0) O::arrive(O::leader(sf_full(sf)));
        filled[sf] = static_cast<int>(sf_phase);
        if (++sf == kSfStages) {
          sf = 0;
          sf_phase ^= 1u;
        }
      }
    }
    if (!ok) {
      if (lane == 0) raise_abort(abort_flag, p.err, kErrScales);
    } else if (lane == 0) {
      // the releases land in this CTA's shared memory: wait for the last ones
      for (int s = 0; s < kSfStages; ++s)
        if (filled[s] >= 0) wait_drain(sf_empty(s), static_cast<uint32_t>(filled[s]));
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue (both CTAs)
    const int quad = warp & 3;
    const uint32_t leader_empty0 = O::leader(acc_empty(0));
    const uint32_t leader_empty1 = O::leader(acc_empty(1));
    const uint32_t leader_shared = O::leader(shared_bar);
    const uint32_t epi = epi_base + static_cast<uint32_t>(quad) * kEpiWarpBytes;
    uint32_t box_no = 0;
    int it = 0;
    bool ok = true;
    for (long long t = cid; walker.locate(t, tile); t += ncl, ++it) {
      const int acc = it & 1;
      if (!mbar_wait(acc_full(acc), static_cast<uint32_t>((it >> 1) & 1), abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int m_local = tile.m_idx * kTileM + static_cast<int>(rank) * 128 + quad * 32 + lane;
      const int64_t row = static_cast<int64_t>(p.row_start[tile.g]) + m_local;
      const bool rvalid =
          m_local < p.rows[tile.g] && static_cast<uint64_t>(row) < static_cast<uint64_t>(p.x_rows);
      // a warp whose 32 rows all belong to the group stores them with TMA
      const bool tma = !kFew && __all_sync(0xffffffffu, rvalid);
      const int warp_row0 = static_cast<int>(row) - lane;
      const uint32_t tbase =
          tmem + (static_cast<uint32_t>(quad * 32) << 16) + (acc ? kAccCol1 : 0u);
      // 32 columns of bf16 of this lane's row through a 64-byte-swizzled box
      auto emit = [&](const CUtensorMap* map, __nv_bfloat16* orow, const uint32_t (&o)[16], int col) {
        if (tma) {
          const uint32_t buf = epi + (box_no & 1u) * 2048u;
          ++box_no;
          if (lane == 0) bulk_wait_read<1>();  // the store that used this box has read it
          __syncwarp();
          const uint32_t sw = static_cast<uint32_t>((lane >> 1) & 3);
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            st_shared_v4(buf + static_cast<uint32_t>(lane) * 64u + ((j ^ sw) << 4), o[4 * j],
                         o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(map, col, warp_row0, buf);
            bulk_commit();
          }
        } else if (rvalid) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (col + (v + 1) * 8 <= p.n)
              *reinterpret_cast<uint4*>(orow + col + v * 8) =
                  make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
      };
      auto release_shared = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) O::arrive(leader_shared);
      };
      if (p.epilogue == 0) {
        // accumulator 0 shares its last 32 columns, accumulator 1 its first
        const int n0 = tile.n_idx * BN;
        __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(p.out) + row * p.n;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int c = acc ? i : (i + 7) & 7;
          uint32_t r[32];
          tmem_ld_32x32b_x32(tbase + c * 32, r);
          tmem_ld_wait();
          if (i == 0) release_shared();
          const int col = n0 + c * 32;
          if (col >= p.n) continue;  // warp-uniform
          uint32_t o[16];
#pragma unroll
          for (int q = 0; q < 16; ++q)
            o[q] = pack_bf16x2(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
          emit(&tmap_out, orow, o, col);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) O::arrive(acc ? leader_empty1 : leader_empty0);
      } else {
        // gate in columns 0..127, up in 128..255, 32 of each at a time; the
        // shared columns lie in the chunk that comes first. h[] is indexed in
        // the order of the chunks, so that it stays in registers.
        float h[128];
        float amax = 0.f;
        __nv_bfloat16* prow = p.pre == nullptr ? nullptr : p.pre + row * p.n;
        if (tma) {  // the last tile's box has been read before its bytes are used again
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = acc ? i : (i + 3) & 3;
          uint32_t gr[32], ur[32];
          tmem_ld_32x32b_x32(tbase + c * 32, gr);
          tmem_ld_32x32b_x32(tbase + 128 + c * 32, ur);
          tmem_ld_wait();
          if (i == 0) release_shared();
          if (i == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) O::arrive(acc ? leader_empty1 : leader_empty0);
          }
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 v = swiglu2_f32(
                make_float2(__uint_as_float(gr[2 * q]), __uint_as_float(gr[2 * q + 1])),
                make_float2(__uint_as_float(ur[2 * q]), __uint_as_float(ur[2 * q + 1])));
            h[i * 32 + 2 * q] = v.x;
            h[i * 32 + 2 * q + 1] = v.y;
            amax = fmaxf(amax, fmaxf(fp8::finite_abs(v.x), fp8::finite_abs(v.y)));
          }
          if (prow != nullptr) {
            uint32_t o[16];
#pragma unroll
            for (int q = 0; q < 16; ++q)
              o[q] = pack_bf16x2(__uint_as_float(gr[2 * q]), __uint_as_float(gr[2 * q + 1]));
            emit(&tmap_pre, prow, o, tile.n_idx * 128 + c * 32);
#pragma unroll
            for (int q = 0; q < 16; ++q)
              o[q] = pack_bf16x2(__uint_as_float(ur[2 * q]), __uint_as_float(ur[2 * q + 1]));
            emit(&tmap_pre, prow, o, p.f_half + tile.n_idx * 128 + c * 32);
          }
        }
        const uint32_t sb = fp8::scale_byte(amax);
        const float inv = fp8::inverse_scale(sb);
        if (tma) {
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        uint8_t* orow = static_cast<uint8_t*>(p.out) + row * p.f_half + tile.n_idx * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = acc ? i : (i + 3) & 3;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int j = i * 32 + v * 16 + q * 4;
              o[q] = fp8::pack4(fp8::scaled(h[j], inv), fp8::scaled(h[j + 1], inv),
                                fp8::scaled(h[j + 2], inv), fp8::scaled(h[j + 3], inv));
            }
            const uint32_t chunk = static_cast<uint32_t>(c * 2 + v);
            if (tma)  // 128-byte-swizzled box of 32 rows
              st_shared_v4(epi + static_cast<uint32_t>(lane) * 128u +
                               ((chunk ^ static_cast<uint32_t>(lane & 7)) << 4),
                           o[0], o[1], o[2], o[3]);
            else if (rvalid)
              *reinterpret_cast<uint4*>(orow + chunk * 16) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        if (rvalid)
          p.out_scale[row * (p.f_half / 128) + tile.n_idx] = static_cast<uint8_t>(sb);
        if (tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmap_out, tile.n_idx * 128, warp_row0, epi);
            bulk_commit();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();  // every tile store has finished
    __syncwarp();
    if (!ok && lane == 0) raise_abort(abort_flag, p.err, kErrEpilogue);
  }

  if constexpr (kPair) {
    pair_teardown(tmem, kTmemCols, warp == 1);
  } else {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, kTmemCols);
    }
    // What follows in the stream waits for this launch alone, so it ends after the pairs'.
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
}

// 3-D tensor map over bytes [d2, d1, d0] (d0 contiguous), box 128 x box_rows x 1,
// 128-byte swizzle; reads outside give zeros.
int make_tmap(CUtensorMap* m, const void* ptr, uint64_t d0, uint64_t d1, uint64_t d2,
              uint32_t box_rows = 128u) {
  auto encode = gg::get_encode_fn();
  if (encode == nullptr) {
    set_last_error("grouped_gemm_fp8: cuTensorMapEncodeTiled unavailable");
    return MOE_ERR_CUDA;
  }
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {d0, d0 * d1};
  cuuint32_t box[3] = {128u, box_rows, 1u};
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

// 2-D map over a row-major [rows, cols] output for 32-row tile stores: boxes
// of 32 bf16 columns (64-byte swizzle) or 128 bytes (128-byte swizzle).
int make_store_tmap(CUtensorMap* m, void* ptr, uint64_t cols, uint64_t rows, bool bf16) {
  auto encode = gg::get_encode_fn();
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {cols * (bf16 ? 2 : 1)};
  cuuint32_t box[2] = {bf16 ? 32u : 128u, 32u};
  cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = encode(
      m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, ptr, dims,
      strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      bf16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("grouped_gemm_fp8: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return MOE_ERR_CUDA;
  }
  return MOE_OK;
}

// Launch attributes of both kernels, once per device; `clusters` gets the CTA
// pairs that can be resident at once (0: none, the single-CTA kernel serves).
int prepare_device(int dev, int* clusters) {
  static std::mutex mu;
  static int pairs[64];
  static bool done[64] = {};
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && dev < 64 && done[dev]) {
    *clusters = pairs[dev];
    return MOE_OK;
  }
  MOE_CUDA_CALL(cudaFuncSetAttribute(grouped_gemm_fp8_kernel<kPairForm>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(Shape<kPairForm>::kSmemBytes)),
                "cudaFuncSetAttribute(grouped_gemm_fp8 pair)");
  MOE_CUDA_CALL(cudaFuncSetAttribute(grouped_gemm_fp8_kernel<kSingleForm>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(Shape<kSingleForm>::kSmemBytes)),
                "cudaFuncSetAttribute(grouped_gemm_fp8 single)");
  MOE_CUDA_CALL(cudaFuncSetAttribute(grouped_gemm_fp8_kernel<kFewForm>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(Shape<kFewForm>::kSmemBytes)),
                "cudaFuncSetAttribute(grouped_gemm_fp8 few)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * 74);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shape<kPairForm>::kSmemBytes;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, grouped_gemm_fp8_kernel<kPairForm>, &cfg) != cudaSuccess) n = 0;
  cudaGetLastError();  // clear a non-sticky error of the query
  if (dev >= 0 && dev < 64) {
    pairs[dev] = n;
    done[dev] = true;
  }
  *clusters = n;
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
  MOE_REQUIRE(x_rows >= 0 && x_rows < (1ll << 31) - 256, "grouped_gemm_fp8: x_rows=%lld out of range",
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
  int clusters = 0;
  int st = g8::prepare_device(dev, &clusters);
  if (st) return st;

  CUtensorMap ta, taf, tb;
  st = g8::make_tmap(&ta, x, static_cast<uint64_t>(K), static_cast<uint64_t>(x_rows), 1);
  if (st) return st;
  st = g8::make_tmap(&taf, x, static_cast<uint64_t>(K), static_cast<uint64_t>(x_rows), 1,
                     g8::kFewRows);
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
  p.n_chunk = 0;
  p.above = 0;
  p.most = 0x7fffffff;
  p.b_mn = w_kn ? 1 : 0;
  p.epilogue = epilogue;
  p.xs = {static_cast<const uint8_t*>(x_scale), x_rows * p.num_kb, p.num_kb,
          (reinterpret_cast<uintptr_t>(x_scale) & 3) == 0};
  p.ws = {static_cast<const uint8_t*>(w_scale), num_w * p.n_blocks * p.num_kb, p.num_kb,
          (reinterpret_cast<uintptr_t>(w_scale) & 3) == 0};
  CUtensorMap to, tp;
  st = g8::make_store_tmap(&to, out, static_cast<uint64_t>(epilogue == 1 ? p.f_half : p.n),
                           static_cast<uint64_t>(x_rows), epilogue == 0);
  if (st) return st;
  tp = to;
  if (pre != nullptr) {
    st = g8::make_store_tmap(&tp, pre, static_cast<uint64_t>(N), static_cast<uint64_t>(x_rows), true);
    if (st) return st;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Calls of few rows stay with the one launch, which then takes every group (a
  // table may name more rows than there are: those that are there count).
  const bool pairs = clusters > 0 && x_rows > g8::kSingleRows;
  const bool one_launch = pairs && x_rows >= g8::kOneLaunchRows * G;
  if (pairs) {
    p.most = g8::kSingleRows;
    g8::Params pb = p;
    pb.above = one_launch ? 0 : g8::kSingleRows;
    pb.most = 0x7fffffff;
    pb.n_chunk = static_cast<int>(
        std::min<int64_t>(p.n_tiles, std::max<int64_t>(1, g8::kSlabBytes / (g8::BN * K))));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * clusters);
    cfg.blockDim = dim3(g8::kThreads);
    cfg.dynamicSmemBytes = g8::Shape<g8::kPairForm>::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MOE_CUDA_CALL(
        cudaLaunchKernelEx(&cfg, g8::grouped_gemm_fp8_kernel<g8::kPairForm>, ta, taf, tb, to, tp, pb),
        "grouped_gemm_fp8 pair launch");
    if (one_launch) return MOE_OK;
  }
  if (x_rows <= g8::kFewRows) {
    g8::grouped_gemm_fp8_kernel<g8::kFewForm>
        <<<num_sms(dev), g8::kThreads, g8::Shape<g8::kFewForm>::kSmemBytes, s>>>(ta, taf, tb, to, tp, p);
    MOE_CUDA_CHECK_LAUNCH("grouped_gemm_fp8 few launch");
    return MOE_OK;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(num_sms(dev));
  cfg.blockDim = dim3(g8::kThreads);
  cfg.dynamicSmemBytes = g8::Shape<g8::kSingleForm>::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pairs ? 1 : 0;  // a launch that follows another's kernel waits for its end
  MOE_CUDA_CALL(
      cudaLaunchKernelEx(&cfg, g8::grouped_gemm_fp8_kernel<g8::kSingleForm>, ta, taf, tb, to, tp, p),
      "grouped_gemm_fp8 launch");
  return MOE_OK;
}
