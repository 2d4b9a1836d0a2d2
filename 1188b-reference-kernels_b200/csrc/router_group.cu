// Group-limited router with a balance bias, and the gradient of routing weights.
//
//   s = sigmoid(x) or softmax(x) over the experts; c = s + bias (the bias
//   steers the selection alone); the E experts form num_groups equal groups,
//   a group is worth its largest c or the sum of its two largest; the best
//   topk_groups groups stay and the k experts with the largest c inside them
//   are taken. Weights w = s of the taken experts, divided by their sum if
//   renorm, times scale. Ties go to the lower group and the lower expert.
//
// The selection hangs on the last bits of c wherever two experts come close
// (16384 tokens x 256 experts always hold such pairs), so it is that of c and
// group values formed and compared in 64 bits. A first pass in fp32 with an
// error bound settles the rows where no decision is that close; the others are
// ordered or selected in 64 bits. Of 16384 rows of 256 normal logits, top-8,
// that is 0.05 % with sigmoid and 0.2 % with softmax scores, mostly only to be
// ordered; of the same logits rounded to bf16, where equal scores are common,
// 39 % (20 us more for one group).
//
// One warp per token: a row is a kilobyte, its group maxima and its selection
// are exchanges between lanes, and nothing has to leave the warp. A lane
// holds consecutive columns of one group, so that a group is a few lanes.
// Bound by instruction issue, and at the end by the latency of a row that
// needs 64 bits (16384 x 256, 8 groups of which 4 stay, top-8: selected by a
// copy of c in shared memory 10 us of 34, in registers 3 of 24; rows where the
// order of the taken experts alone is open, most of them, evaluate only
// those): 23.3 us on the device against 6.0 us of bytes (4 us more with __expf
// and __fdividef, which cover subnormal numbers, and with checks of every
// column); 8192 x 1024, one group: 44 us from a sigmoid, 49 from a softmax; 4
// tokens: 3.9 us.
// The gradient reads what a row needs and writes it once: 16384 x 256 from a
// sigmoid 9.2 us (2.9 us of bytes; a warp a token took 2 us more), from a
// softmax without renorm, which reads its row twice, 17 to 19.
#include <math.h>

#include <type_traits>

#include "moe_common.cuh"

namespace moe {
namespace {

constexpr int kMaxK = 16;
constexpr int kMaxE = 1024;
constexpr int kWarps = 4;

// Order-preserving bits of a double: NaN above everything, -0 equal to +0.
MOE_DEVICE uint64_t order_key(double v) {
  if (isnan(v)) return ~0ull;
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// Larger key wins, then the lower index; every lane gets the winner.
MOE_DEVICE void warp_argmax(uint64_t& key, int& idx) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const uint64_t k2 = __shfl_xor_sync(0xffffffffu, key, off);
    const int i2 = __shfl_xor_sync(0xffffffffu, idx, off);
    if (k2 > key || (k2 == key && i2 < idx)) {
      key = k2;
      idx = i2;
    }
  }
}

MOE_DEVICE double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
MOE_DEVICE float warp_sumf(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
MOE_DEVICE float warp_maxf(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// A token's logits as 64-bit scores.
struct Scores64 {
  const float* x;
  const float* bias;
  double m, z;
  bool softmax, none;
  // s of expert e; a softmax row whose every logit is -inf has s = 0
  __device__ double s(int e) const {
    const double v = __ldg(x + e);
    if (!softmax) return 1.0 / (1.0 + exp(-v));
    return none ? (isnan(v) ? v : 0.0) : exp(v - m) / z;
  }
  __device__ double c(int e) const { return s(e) + (bias ? static_cast<double>(__ldg(bias + e)) : 0.0); }
};

// Softmax normaliser in 64 bits (all lanes).
MOE_DEVICE double softmax_sum64(const float* x, int E, double m) {
  double sum = 0.0;
  for (int e = lane_id(); e < E; e += 32) sum += exp(static_cast<double>(__ldg(x + e)) - m);
  return warp_sum(sum);
}

// Selection in 64 bits, the definition as it stands: returns lane r's (r < k)
// expert. c: E doubles of this warp in shared memory.
MOE_DEVICE int select64(const Scores64& sc, double* c, int E, int k, int groups, int keep, int top2) {
  const int lane = lane_id();
  for (int e = lane; e < E; e += 32) c[e] = sc.c(e);
  __syncwarp();
  const int size = E / groups;
  uint32_t kept = 0xffffffffu;  // bit g: group g stays
  if (keep < groups) {
    uint64_t key = 0;
    if (lane < groups) {
      double a = -INFINITY, b = -INFINITY;  // the two largest; a NaN counts as the largest
      bool nan = false;
      for (int i = 0; i < size; ++i) {
        const double v = c[lane * size + i];
        nan |= isnan(v);
        if (v > a) {
          b = a;
          a = v;
        } else if (v > b) {
          b = v;
        }
      }
      key = nan ? ~0ull : order_key(top2 && size > 1 ? a + b : a);
    }
    kept = 0;
    for (int r = 0; r < keep; ++r) {
      // a live key is never 0 (the smallest is that of -inf), so taken and
      // absent groups lose
      uint64_t w = lane < groups && !(kept >> lane & 1u) ? key : 0;
      int wi = lane < groups ? lane : 1 << 20;
      warp_argmax(w, wi);
      kept |= 1u << wi;
    }
  }
  int mine = 0;
  uint32_t taken = 0;  // bit j: column lane + 32 j
  for (int r = 0; r < k; ++r) {
    uint64_t w = 0;
    int wi = 1 << 20;
    for (int e = lane, j = 0; e < E; e += 32, ++j) {
      if ((taken >> j & 1u) || !(kept >> (e / size) & 1u)) continue;
      const uint64_t key = order_key(c[e]);
      if (key > w) {
        w = key;
        wi = e;
      }
    }
    warp_argmax(w, wi);
    if ((wi & 31) == lane) taken |= 1u << (wi >> 5);
    if (lane == r) mine = wi;
  }
  return mine;
}

// Order-preserving bits of a float that is neither NaN nor -0; never 0.
MOE_DEVICE uint32_t order_key32(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
MOE_DEVICE float key32_value(uint32_t key) {
  return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}

// One instruction each; subnormal results are 0.
MOE_DEVICE float fast_exp(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t * 1.4426950408889634f));
  return r;
}
MOE_DEVICE float fast_rcp(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
MOE_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct RouteArgs {
  const float* logits;
  const float* bias;
  int64_t T;
  int E, k, softmax, groups, keep, top2, renorm;
  float scale;
  int lanes;  // lanes that share a group (a power of two)
  int vpl;    // columns of a lane
  float* vals;
  int64_t* idx;
  uint8_t* rmap;
  float* probs;
};

enum Settled { kOpen, kOrder, kAll };

// Fast selection in fp32 with an error bound. Each lane holds vpl consecutive
// columns of one group, `lanes` lanes a group. c in fp32 is off by at most
// `err` (below), so an order of fp32 values is the true one where neighbours
// differ by more than 2 err. Where a decision hangs on less than that, every lane
// gets what is open: kOpen, which experts are taken (or a NaN is there); kOrder,
// only their order.
// kFull: every lane holds VPL columns, a multiple of 4, and the rows are
// 16-byte aligned.
template <int VPL, bool kFull>
MOE_DEVICE Settled select32(const RouteArgs& a, const float* x, int* s_mine, int& mine) {
  const int lane = lane_id();
  const int size = a.E / a.groups;
  const int g = lane / a.lanes;
  const int first = (lane & (a.lanes - 1)) * a.vpl;  // inside the group
  const int n = kFull ? VPL : g < a.groups ? max(0, min(a.vpl, size - first)) : 0;
  const int col0 = g * size + first;
  float v[VPL], c[VPL], add[VPL];
  auto load = [&](const float* p, float none, float (&r)[VPL]) {
    if constexpr (kFull) {
#pragma unroll
      for (int j = 0; j < VPL; j += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + col0 + j));
        r[j] = q.x;
        r[j + 1] = q.y;
        r[j + 2] = q.z;
        r[j + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j) r[j] = j < n ? __ldg(p + col0 + j) : none;
    }
  };
  load(x, -INFINITY, v);
  if (a.bias != nullptr) load(a.bias, 0.f, add);
  // fp32 scores and what they may be off by, in units of 2^-23.
  // fast_exp(t) is off by 2 + 1.18 |t| of itself (the CUDA C++ Programming
  // Guide's bound of __expf, these two steps: 2 + 1.173 |t| ulp), fast_rcp by 1
  // (PTX ISA, rcp.approx), its use by 1.
  // sigmoid: of exp's error s (1 - s) arrives, at most 1/4 * 2 + 1.18 * 0.23;
  //   the sum 1 + e adds 1/2, the quotient 2: together below 4.
  // softmax: t = x - m adds |t| / 2 to exp's; s |t| <= rz / e, so that
  //   s (2 + 1.68 |t|) <= 2.62 rz. z inherits the mean of 2 + 1.68 |t| under s;
  //   that of |t| is s's entropy less ln z, at most ln E, E <= 32 VPL. Its own
  //   sums, VPL terms in a row and five steps between lanes, add (VPL + 5) / 2,
  //   quotient and product 2.5. With s <= rz the total is
  //   (9.7 + 1.68 ln(32 VPL) + VPL / 2) rz: 37.3 for 32 columns (23.0 for 8),
  //   in the code 1 + (22 + VPL / 2) rz, 38 (26).
  // Adding the bias rounds once more, 2^-24 |c|.
  float m = 0.f, rz = 1.f, err;
  if (a.softmax) {
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) m = fmaxf(m, v[j]);
    m = warp_maxf(m);
    float z = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) z += kFull || j < n ? fast_exp(v[j] - m) : 0.f;
    rz = fast_rcp(warp_sumf(z));
    err = (1.f + (22 + VPL / 2) * rz) * 1.1920929e-7f;
  } else {
    err = 4.f * 1.1920929e-7f;
  }
  bool odd = a.softmax && !(fabsf(m) < INFINITY);  // no maximum to subtract
  float big = 0.f;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    c[j] = a.softmax ? fast_exp(v[j] - m) * rz : fast_rcp(1.0f + fast_exp(-v[j]));
    if (a.bias != nullptr) c[j] += add[j];
    big = max_nan(big, fabsf(c[j]));
  }
  // (columns that are not there have c = 0). Of a y above 2^126 the reciprocal
  // is 0, as sigmoid of such x is to within 2^-126.
  big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
  if (!(big < INFINITY)) {
    odd |= isnan(big);
    big = 0.f;  // a bias of -inf is exact
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (c[j] > -INFINITY) big = fmaxf(big, fabsf(c[j]));
    big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
  }
  err += 5.9604645e-8f * big;
  const float gap = 2.f * err;

  bool in = n > 0;
  if (a.keep < a.groups) {
    float hi = -INFINITY, lo = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (kFull || j < n) {
        lo = fmaxf(lo, fminf(hi, c[j]));
        hi = fmaxf(hi, c[j]);
      }
    for (int off = 1; off < a.lanes; off <<= 1) {
      const float h2 = __shfl_xor_sync(0xffffffffu, hi, off);
      const float l2 = __shfl_xor_sync(0xffffffffu, lo, off);
      lo = fmaxf(fminf(hi, h2), fmaxf(lo, l2));
      hi = fmaxf(hi, h2);
    }
    const float rank = a.top2 && size > 1 ? hi + lo : hi;
    int better = 0;
    for (int q = 0; q < a.groups; ++q)
      better += __shfl_sync(0xffffffffu, rank, q * a.lanes) > rank;
    const bool stays = g < a.groups && better < a.keep;
    // worst group that stays against the best that goes: two sums of two
    const uint32_t kept_min = __reduce_min_sync(0xffffffffu, stays ? order_key32(rank) : 0xffffffffu);
    const uint32_t gone_max =
        __reduce_max_sync(0xffffffffu, g < a.groups && !stays ? order_key32(rank) : 0u);
    const int staying = __popc(__ballot_sync(0xffffffffu, stays && (lane & (a.lanes - 1)) == 0));
    odd |= staying != a.keep || gone_max == 0u ||
           !(key32_value(kept_min) - key32_value(gone_max) > 4.f * err + 4.f * 5.9604645e-8f * big);
    in &= stays;
  }
  uint32_t key[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) key[j] = in && (kFull || j < n) && !odd ? order_key32(c[j]) : 0u;
  // A lane offers its best column; its second best stands ready, and only a
  // lane that wins a second time looks through its columns again. It passes
  // over those it has given, not over their keys: others may have equal ones.
  uint32_t b1 = 0, b2 = 0;
  int c1 = 0, c2 = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const bool first = key[j] > b1, second = key[j] > b2;
    b2 = first ? b1 : second ? key[j] : b2;
    c2 = first ? c1 : second ? j : c2;
    b1 = first ? key[j] : b1;
    c1 = first ? j : c1;
  }
  bool spare = true;
  uint32_t wins = 0;
  uint32_t given = 0;               // bit j: column j has been taken
  uint32_t won = 0;                 // lane r: the key of round r
  for (int r = 0; r <= a.k; ++r) {  // one more than is taken: the border below
    const uint32_t w = __reduce_max_sync(0xffffffffu, b1);
    if (lane == r) won = w;
    if (w == 0u || r == a.k) break;  // nothing left (all taken, or a NaN: odd)
    if (b1 == w) {  // one lane, or several of equal keys: the wins then add up to more than k
      ++wins;
      s_mine[r] = col0 + c1;
      given |= 1u << c1;
      if (spare) {
        b1 = b2;
        c1 = c2;
        spare = false;
      } else {
        b1 = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          const bool next = !(given >> j & 1u) && key[j] > b1;
          b1 = next ? key[j] : b1;
          c1 = next ? j : c1;
        }
      }
    }
  }
  __syncwarp();
  mine = lane < a.k ? s_mine[lane] : 0;
  odd |= __reduce_add_sync(0xffffffffu, wins) != static_cast<uint32_t>(a.k);
  // Rounds whose keys lie too close (equal ones of one lane come up one round
  // after the other) leave their order open, the last of them against the
  // border also the choice; so does an empty round.
  const uint32_t before = __shfl_up_sync(0xffffffffu, won, 1);
  const bool close =
      lane >= 1 && lane <= a.k && won != 0u && !(key32_value(before) - key32_value(won) > gap);
  odd |= (lane < a.k && won == 0u) || (lane == a.k && close);
  if (__any_sync(0xffffffffu, odd)) return kOpen;
  return __any_sync(0xffffffffu, close) ? kOrder : kAll;
}

// The taken experts in the order of their 64-bit scores.
MOE_DEVICE int order64(const Scores64& sc, int k, int mine, int* s_mine) {
  const int lane = lane_id();
  const uint64_t key = lane < k ? order_key(sc.c(mine)) : 0;
  int rank = 0;
  for (int j = 0; j < k; ++j) {
    const uint64_t other = __shfl_sync(0xffffffffu, key, j);
    const int e = __shfl_sync(0xffffffffu, mine, j);
    rank += other > key || (other == key && e < mine);
  }
  if (lane < k) s_mine[rank] = mine;
  __syncwarp();
  return lane < k ? s_mine[lane] : 0;
}

// The larger of two 64-bit keys over the warp, as two 32-bit maxima; `owners`
// gets the lanes that hold it.
MOE_DEVICE uint64_t warp_max_key(uint64_t key, uint32_t& owners) {
  const uint32_t hi = static_cast<uint32_t>(key >> 32), lo = static_cast<uint32_t>(key);
  const uint32_t mhi = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t mlo = __reduce_max_sync(0xffffffffu, hi == mhi ? lo : 0u);
  owners = __ballot_sync(0xffffffffu, hi == mhi && lo == mlo);
  return static_cast<uint64_t>(mhi) << 32 | mlo;
}

// Selection in 64 bits in the lane layout of select32 (columns rise with the
// lane, so the lowest owner of a key has the lowest column).
template <int VPL>
MOE_DEVICE int select64_lanes(const RouteArgs& a, const Scores64& sc, int* s_mine) {
  const int lane = lane_id();
  const int size = a.E / a.groups;
  const int g = lane / a.lanes;
  const int first = (lane & (a.lanes - 1)) * a.vpl;
  const int n = g < a.groups ? max(0, min(a.vpl, size - first)) : 0;
  const int col0 = g * size + first;
  uint64_t key[VPL];
  double hi = -INFINITY, lo = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    key[j] = 0;
    if (j < n) {
      const double c = sc.c(col0 + j);
      nan |= isnan(c);
      lo = fmax(lo, fmin(hi, c));
      hi = fmax(hi, c);
      key[j] = order_key(c);
    }
  }
  if (a.keep < a.groups) {
    for (int off = 1; off < a.lanes; off <<= 1) {
      const double h2 = __shfl_xor_sync(0xffffffffu, hi, off);
      const double l2 = __shfl_xor_sync(0xffffffffu, lo, off);
      nan |= __shfl_xor_sync(0xffffffffu, static_cast<int>(nan), off) != 0;
      lo = fmax(fmin(hi, h2), fmax(lo, l2));
      hi = fmax(hi, h2);
    }
    // a NaN counts as the largest value of its group
    const uint64_t rank = nan ? ~0ull : order_key(a.top2 && size > 1 ? hi + lo : hi);
    int better = 0;
    for (int q = 0; q < a.groups; ++q) {
      const uint64_t other = __shfl_sync(0xffffffffu, rank, q * a.lanes);
      better += other > rank || (other == rank && q < g);
    }
    if (better >= a.keep) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) key[j] = 0;
    }
  }
  for (int r = 0; r < a.k; ++r) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (key[j] > best) {
        best = key[j];
        at = j;
      }
    uint32_t owners;
    warp_max_key(best, owners);
    if (lane == __ffs(owners) - 1) {
      s_mine[r] = col0 + at;
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (j == at) key[j] = 0;
    }
  }
  __syncwarp();
  return lane < a.k ? s_mine[lane] : 0;
}

// One warp per token. VPL 0: 64 bits throughout, the scores in shared memory
// (shapes whose lanes would hold more than 32 columns, where a number of groups
// that is no power of two leaves lanes without any: 3 groups of 341, 9 of 113,
// 17 of 60).
template <int VPL, bool kFull>
__global__ void __launch_bounds__(32 * kWarps) router_group_kernel(const RouteArgs a) {
  extern __shared__ double s_c[];
  const int lane = lane_id();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp_id();
  if (t >= a.T) return;
  const float* x = a.logits + t * a.E;
  // the dense outputs are 0 outside the selection
  if (a.probs) {
    float* row = a.probs + t * a.E;
    if (a.E % 4 == 0 && (reinterpret_cast<uintptr_t>(a.probs) & 15) == 0)
      for (int e = lane; e < a.E / 4; e += 32) reinterpret_cast<float4*>(row)[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    else
      for (int e = lane; e < a.E; e += 32) row[e] = 0.f;
  }
  if (a.rmap) {
    uint8_t* row = a.rmap + t * a.E;
    if (a.E % 4 == 0 && (reinterpret_cast<uintptr_t>(a.rmap) & 3) == 0)
      for (int e = lane; e < a.E / 4; e += 32) reinterpret_cast<uint32_t*>(row)[e] = 0u;
    else
      for (int e = lane; e < a.E; e += 32) row[e] = 0;
  }
  int mine = 0;
  Settled settled = kOpen;
  __shared__ int s_mine[kWarps][kMaxK];
  if constexpr (VPL > 0) settled = select32<VPL, kFull>(a, x, s_mine[warp_id()], mine);
  Scores64 sc{x, a.bias, 0.0, 1.0, a.softmax != 0, false};
  // The softmax's normaliser cancels in renormalised weights, so that only
  // the 64-bit selection and plain softmax weights need it.
  if (a.softmax) {
    float m = -INFINITY;
    for (int e = lane; e < a.E; e += 32) m = fmaxf(m, __ldg(x + e));
    sc.m = warp_maxf(m);
    sc.none = sc.m == -INFINITY;
    if (settled != kAll || !a.renorm) sc.z = softmax_sum64(x, a.E, sc.m);
  }
  if (settled == kOrder) mine = order64(sc, a.k, mine, s_mine[warp_id()]);
  if (settled == kOpen) {
    if constexpr (VPL > 0)
      mine = select64_lanes<VPL>(a, sc, s_mine[warp_id()]);
    else
      mine = select64(sc, s_c + warp_id() * a.E, a.E, a.k, a.groups, a.keep, a.top2);
  }
  double weight = lane < a.k ? sc.s(mine) : 0.0;
  if (a.renorm) {
    const double sum = warp_sum(weight);
    weight = sum == 0.0 ? 0.0 : weight / sum;
  }
  const float w = static_cast<float>(weight * static_cast<double>(a.scale));
  __syncwarp();  // the zeros above come first
  if (lane < a.k) {
    if (a.vals) a.vals[t * a.k + lane] = w;
    if (a.idx) a.idx[t * a.k + lane] = mine;
    if (a.rmap) a.rmap[t * a.E + mine] = 1;
    if (a.probs) a.probs[t * a.E + mine] = w;
  }
}

template <int VPL>
void launch_route(const RouteArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((a.T + kWarps - 1) / kWarps);
  if constexpr (VPL >= 4 && VPL % 4 == 0) {
    // every lane full: no column is asked whether it is there, and loads are of 16 bytes (8 groups of 32:
    // 24.8 against 27.2 us, 16 of 32: 36 against 51)
    if (a.E == 32 * VPL && 32 / a.lanes == a.groups && a.vpl == VPL &&
        ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.bias)) & 15) == 0) {
      router_group_kernel<VPL, true><<<grid, 32 * kWarps, 0, s>>>(a);
      return;
    }
  }
  router_group_kernel<VPL, false>
      <<<grid, 32 * kWarps, VPL > 0 ? 0 : kWarps * a.E * sizeof(double), s>>>(a);
}

// kLanes lanes per token, of which lane j < k holds the j-th selected expert.
// With renorm the weights are w_j = s_j / S, S = sum_i s_i, and
//   sigmoid: dx_j = scale * w_j (1 - s_j) (g_j - sum_i g_i w_i)
//   softmax: dx_j = scale * w_j (g_j - sum_i g_i w_i): its normaliser cancels, w is a softmax of the selected
//            logits alone and the rest of the row is not read
//   logits:  dx_j = scale * (g_j - sum_i g_i w_i) / S
// and 0 elsewhere; nothing is divided by S twice, whose square leaves fp32's
// range long before the weights do. Without:
//   sigmoid: dx_j = scale * g_j s_j (1 - s_j)     logits: dx_j = scale * g_j
//   softmax: dx_e = s_e (ds_e - sum_j ds_j s_j), ds_j = scale * g_j, 0 outside the selection
// Of a sigmoid, q = e^-|x| gives s and 1 - s as 1 / (1 + q) and q / (1 + q),
// neither by a difference. Its w_j come from numerators e^min(x,0) relative to
// the list's largest, so that a list of tiny scores keeps its weights.
// What a token waits for is its list, then the gathers; with as few lanes a
// token as its list needs, a warp has those of several under way.
// 64-bit sigmoid scores of logits at or below this are 0, and so are the
// forward's weights of a list that holds no other.
constexpr float kNoScore = -709.7827f;

template <int kLanes>
MOE_DEVICE float group_sum(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
template <int kLanes>
MOE_DEVICE float group_max(float v) {
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

template <int kLanes>
__global__ void __launch_bounds__(32 * kWarps) router_backward_kernel(
    const float* __restrict__ logits, const float* __restrict__ bias,
    const int32_t* __restrict__ perm, const int64_t* __restrict__ idx,
    const float* __restrict__ grad_vals, const float* __restrict__ grad_probs, int64_t T, int E,
    int k, int mode, int renorm, float scale, float* __restrict__ out) {
  constexpr int kTokens = 32 / kLanes;  // of a warp
  const int lane = lane_id();
  const int l = lane % kLanes;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kWarps + warp_id()) * kTokens;
  if (t0 >= T) return;
  const int64_t t = t0 + lane / kLanes;
  const float* x = logits + t * E;
  float* o = out + t * E;
  const bool list_softmax = mode == 1 && renorm;
  const bool row_softmax = kLanes == 32 && mode == 1 && !renorm;
  float m = 0.f, z = 1.f;
  if (row_softmax) {
    m = -INFINITY;
    for (int e = lane; e < E; e += 32) m = fmaxf(m, __ldg(x + e) + (bias ? __ldg(bias + e) : 0.f));
    m = warp_maxf(m);
    float sum = 0.f;
    if (m > -INFINITY)
      for (int e = lane; e < E; e += 32)
        sum += expf(__ldg(x + e) + (bias ? __ldg(bias + e) : 0.f) - m);
    z = warp_sumf(sum);
  }
  auto logit = [&](int e) { return __ldg(x + e) + (bias ? __ldg(bias + e) : 0.f); };
  auto row_score = [&](int e) { return m > -INFINITY ? expf(logit(e) - m) / z : 0.f; };
  int col = -1;  // this lane's expert, as a column of the logits
  float v = 0.f, g = 0.f;
  if (l < k && t < T) {
    const int64_t slot = __ldg(idx + t * k + l);
    if (slot >= 0 && slot < E) col = perm ? __ldg(perm + slot) : static_cast<int>(slot);
    if (col >= 0 && col < E) {
      g = scale * (grad_vals ? __ldg(grad_vals + t * k + l) : __ldg(grad_probs + t * E + slot));
      v = logit(col);
    } else {
      col = -1;  // named by neither the list nor the placement: no gradient
    }
  }
  // dx_j = ds * factor
  float ds = g, factor = 1.f;
  float dot = 0.f;  // of a softmax over the row
  if (mode == 2) {
    const float q = expf(-fabsf(v));
    const float r = 1.0f / (1.0f + q);
    const bool up = v >= 0.f;
    factor = up ? q * r : r;  // 1 - s
    if (renorm) {
      const float top = fminf(v, 0.f);
      m = group_max<kLanes>(col >= 0 ? top : -INFINITY);
      float w = col >= 0 && m > kNoScore ? expf(top - m) * r : 0.f;
      const float S = group_sum<kLanes>(w);
      w = S == 0.f ? 0.f : w / S;
      ds = w * (g - group_sum<kLanes>(g * w));
    } else {
      ds = g * (up ? r : q * r);
    }
  } else if (list_softmax) {
    m = group_max<kLanes>(col >= 0 ? v : -INFINITY);
    float w = col >= 0 && m > -INFINITY ? expf(v - m) : 0.f;
    const float S = group_sum<kLanes>(w);
    w = S == 0.f ? 0.f : w / S;
    ds = w * (g - group_sum<kLanes>(g * w));
  } else if (row_softmax) {
    factor = col >= 0 ? row_score(col) : 0.f;
    dot = warp_sumf(ds * factor);
  } else if (renorm) {
    const float S = group_sum<kLanes>(v);
    const float mean = group_sum<kLanes>(S == 0.f ? 0.f : g * (v / S));
    ds = S == 0.f ? 0.f : (g - mean) / S;
  }
  // an expert named twice gets the sum of its gradients
  float dsum = 0.f;
  for (int j = 0; j < k; ++j) {
    const int cj = __shfl_sync(0xffffffffu, col, j, kLanes);
    const float dj = __shfl_sync(0xffffffffu, ds, j, kLanes);
    if (cj == col) dsum += dj;
  }
  if (row_softmax) {
    for (int e = lane; e < E; e += 32) o[e] = -row_score(e) * dot;
  } else {  // the warp's rows lie one behind the other
    float* first = out + t0 * E;
    const int64_t values = (T - t0 < kTokens ? T - t0 : kTokens) * E;
    if (E % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0)
      for (int64_t e = lane; e < values / 4; e += 32)
        reinterpret_cast<float4*>(first)[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    else
      for (int64_t e = lane; e < values; e += 32) first[e] = 0.f;
  }
  __syncwarp();
  if (col >= 0) o[col] = (dsum - dot) * factor;
}

template <int kLanes, typename... Args>
void launch_backward(int64_t T, cudaStream_t s, Args... args) {
  const int64_t tokens = kWarps * (32 / kLanes);  // of a CTA
  router_backward_kernel<kLanes>
      <<<static_cast<unsigned>((T + tokens - 1) / tokens), 32 * kWarps, 0, s>>>(args...);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_router_group_topk(const float* logits, const float* bias, int64_t T, int64_t E,
                                     int32_t k, int32_t score_mode, int32_t num_groups,
                                     int32_t topk_groups, int32_t group_score, int32_t renorm,
                                     float scale, float* topk_vals, int64_t* topk_idx,
                                     uint8_t* routing_map, float* probs, moe_stream_t stream) {
  MOE_REQUIRE(T >= 0 && E >= 1, "router_group_topk: bad shape T=%lld E=%lld", (long long)T,
              (long long)E);
  MOE_REQUIRE(score_mode == 1 || score_mode == 2,
              "router_group_topk: score_mode must be 1 (softmax) or 2 (sigmoid)");
  MOE_REQUIRE(group_score == 0 || group_score == 1,
              "router_group_topk: group_score must be 0 (max) or 1 (sum of the two largest)");
  MOE_REQUIRE(num_groups >= 1 && E % num_groups == 0,
              "router_group_topk: E=%lld is no multiple of num_groups=%d", (long long)E, num_groups);
  MOE_REQUIRE(topk_groups >= 1 && topk_groups <= num_groups,
              "router_group_topk: topk_groups=%d out of [1,%d]", topk_groups, num_groups);
  MOE_REQUIRE(k >= 1 && k <= E / num_groups * topk_groups,
              "router_group_topk: k=%d out of range for %d groups of %lld experts", k, topk_groups,
              (long long)(E / num_groups));
  if (k > kMaxK || E > kMaxE || num_groups > 32) {
    set_last_error("router_group_topk: k=%d E=%lld num_groups=%d exceeds this build (k <= %d, E <= "
                   "%d, num_groups <= 32)",
                   k, (long long)E, num_groups, kMaxK, kMaxE);
    return MOE_ERR_UNSUPPORTED;
  }
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(topk_vals || topk_idx || routing_map || probs, "router_group_topk: no output requested");
  MOE_REQUIRE(logits != nullptr, "router_group_topk: null logits");
  MOE_REQUIRE(T <= (int64_t)0x7fffffff * kWarps, "router_group_topk: T too large");
  RouteArgs a;
  a.logits = logits;
  a.bias = bias;
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = k;
  a.softmax = score_mode == 1;
  a.groups = num_groups;
  a.keep = topk_groups;
  a.top2 = group_score;
  a.renorm = renorm;
  a.scale = scale;
  a.vals = topk_vals;
  a.idx = topk_idx;
  a.rmap = routing_map;
  a.probs = probs;
  a.lanes = 32;
  while (32 / a.lanes < num_groups) a.lanes >>= 1;
  a.vpl = (a.E / num_groups + a.lanes - 1) / a.lanes;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.vpl <= 1)
    launch_route<1>(a, s);
  else if (a.vpl <= 2)
    launch_route<2>(a, s);
  else if (a.vpl <= 4)
    launch_route<4>(a, s);
  else if (a.vpl <= 8)
    launch_route<8>(a, s);
  else if (a.vpl <= 12)
    launch_route<12>(a, s);
  else if (a.vpl <= 16)
    launch_route<16>(a, s);
  else if (a.vpl <= 32)
    launch_route<32>(a, s);
  else
    launch_route<0>(a, s);
  MOE_CUDA_CHECK_LAUNCH("router_group_topk launch");
  return MOE_OK;
}

extern "C" int moe_router_topk_backward(const float* logits, const float* bias,
                                        const int32_t* placement, const int64_t* topk_idx,
                                        const float* grad_vals, const float* grad_probs, int64_t T,
                                        int64_t E, int32_t k, int32_t score_mode, int32_t renorm,
                                        float scale, float* grad_logits, moe_stream_t stream) {
  MOE_REQUIRE(T >= 0 && E >= 1 && E <= (1 << 24), "router_topk_backward: bad shape T=%lld E=%lld",
              (long long)T, (long long)E);
  MOE_REQUIRE(k >= 1 && k <= 32 && k <= E, "router_topk_backward: k=%d out of [1,min(E,32)]", k);
  MOE_REQUIRE(score_mode >= 0 && score_mode <= 2,
              "router_topk_backward: score_mode must be 0 (logits), 1 (softmax) or 2 (sigmoid)");
  MOE_REQUIRE((grad_vals != nullptr) != (grad_probs != nullptr) || T == 0,
              "router_topk_backward: exactly one of grad_vals and grad_probs");
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(logits && topk_idx && grad_logits, "router_topk_backward: null pointer");
  MOE_REQUIRE(T <= (int64_t)0x7fffffff * kWarps, "router_topk_backward: T too large");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto launch = [&](auto lanes) {
    launch_backward<decltype(lanes)::value>(T, s, logits, bias, placement, topk_idx, grad_vals, grad_probs,
                                            T, static_cast<int>(E), k, score_mode, renorm, scale, grad_logits);
  };
  if (k > 16 || (score_mode == 1 && !renorm))  // or the whole row is read
    launch(std::integral_constant<int, 32>());
  else if (k > 8)
    launch(std::integral_constant<int, 16>());
  else
    launch(std::integral_constant<int, 8>());
  MOE_CUDA_CHECK_LAUNCH("router_topk_backward launch");
  return MOE_OK;
}
