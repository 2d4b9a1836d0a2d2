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
// (16384 tokens x 256 experts always hold such pairs), so c and the group
// values are formed and compared in 64 bits.
#include <math.h>

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

// One warp per token, its c in shared memory as doubles.
__global__ void __launch_bounds__(32 * kWarps) router_group_kernel(
    const float* __restrict__ logits, const float* __restrict__ bias, int64_t T, int E, int k,
    int softmax, int groups, int keep, int top2, int renorm, float scale, float* __restrict__ vals,
    int64_t* __restrict__ idx_out, uint8_t* __restrict__ rmap, float* __restrict__ probs) {
  extern __shared__ double s_c[];
  const int lane = lane_id();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp_id();
  if (t >= T) return;
  double* c = s_c + warp_id() * E;
  const float* x = logits + t * E;
  double m = 0.0, z = 1.0;
  if (softmax) {
    float mf = -INFINITY;
    for (int e = lane; e < E; e += 32) mf = fmaxf(mf, __ldg(x + e));
    m = warp_maxf(mf);
    double sum = 0.0;
    for (int e = lane; e < E; e += 32) sum += exp(static_cast<double>(__ldg(x + e)) - m);
    z = warp_sum(sum);
  }
  // A row without any score (every logit -inf) has softmax 0, not 0/0.
  const bool none = softmax && m == -INFINITY;
  auto score = [&](int e) -> double {
    const double v = __ldg(x + e);
    if (!softmax) return 1.0 / (1.0 + exp(-v));
    return none ? (isnan(v) ? v : 0.0) : exp(v - m) / z;
  };
  for (int e = lane; e < E; e += 32) c[e] = score(e) + (bias ? static_cast<double>(__ldg(bias + e)) : 0.0);
  __syncwarp();
  const int size = E / groups;
  uint32_t kept = 0xffffffffu;  // bit g: group g stays
  if (keep < groups) {
    uint64_t key = 0;
    int g = lane;
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
      uint64_t w = key;
      int wi = lane < groups ? g : 1 << 20;
      if (kept >> lane & 1u) w = 0;
      if (lane >= groups) w = 0;
      // a live key is never 0 (the smallest is that of -inf), so taken and
      // absent groups lose
      warp_argmax(w, wi);
      kept |= 1u << wi;
    }
  }
  int mine = 0;
  double my_s = 0.0;
  uint32_t taken = 0;  // bit j: column lane + 32 j
  for (int r = 0; r < k; ++r) {
    uint64_t w = 0;
    int wi = 1 << 20;
    for (int e = lane, j = 0; e < E; e += 32, ++j) {
      if (taken >> j & 1u) continue;
      if (!(kept >> (e / size) & 1u)) continue;
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
  if (lane < k) my_s = score(mine);
  double weight = my_s;
  if (renorm) {
    const double sum = warp_sum(my_s);
    weight = sum == 0.0 ? 0.0 : my_s / sum;
  }
  const float w = static_cast<float>(weight * static_cast<double>(scale));
  if (lane < k) {
    if (vals) vals[t * k + lane] = w;
    if (idx_out) idx_out[t * k + lane] = mine;
  }
  if (rmap)
    for (int e = lane, j = 0; e < E; e += 32, ++j) rmap[t * E + e] = taken >> j & 1u;
  if (probs) {
    for (int e = lane; e < E; e += 32) probs[t * E + e] = 0.f;
    __syncwarp();
    if (lane < k) probs[t * E + mine] = w;
  }
}

// One warp per token; lane j < k holds the j-th selected expert.
//   renorm: ds_j = scale * (g_j / S - (sum_i g_i s_i) / S^2), S = sum_i s_i;  else ds_j = scale * g_j
//   sigmoid: dx_j = ds_j s_j (1 - s_j), 0 elsewhere; logits: dx_j = ds_j
//   softmax: dx_e = s_e (ds_e - sum_j ds_j s_j), ds 0 outside the selection
// With renorm the softmax's normaliser cancels: the weights are a softmax w of
// the selected logits alone, dx_j = w_j (g_j - sum_i g_i w_i), exactly 0
// elsewhere, and the rest of the row is not read.
__global__ void __launch_bounds__(32 * kWarps) router_backward_kernel(
    const float* __restrict__ logits, const float* __restrict__ bias,
    const int32_t* __restrict__ perm, const int64_t* __restrict__ idx,
    const float* __restrict__ grad_vals, const float* __restrict__ grad_probs, int64_t T, int E,
    int k, int mode, int renorm, float scale, float* __restrict__ out) {
  const int lane = lane_id();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp_id();
  if (t >= T) return;
  const float* x = logits + t * E;
  float* o = out + t * E;
  const bool list_softmax = mode == 1 && renorm;
  const bool row_softmax = mode == 1 && !renorm;
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
  auto score = [&](int e) {
    const float v = __ldg(x + e) + (bias ? __ldg(bias + e) : 0.f);
    if (mode == 2) return 1.0f / (1.0f + expf(-v));
    if (row_softmax) return m > -INFINITY ? expf(v - m) / z : 0.f;
    return v;  // list_softmax: the exponential follows once the list's maximum is known
  };
  int col = -1;  // this lane's expert, as a column of the logits
  float s = 0.f, g = 0.f;
  if (lane < k) {
    const int64_t slot = __ldg(idx + t * k + lane);
    if (slot >= 0 && slot < E) {
      col = perm ? __ldg(perm + slot) : static_cast<int>(slot);
      g = scale * (grad_vals ? __ldg(grad_vals + t * k + lane) : __ldg(grad_probs + t * E + slot));
      s = score(col);
    }
  }
  if (list_softmax) {
    m = warp_maxf(col >= 0 ? s : -INFINITY);
    s = col >= 0 && m > -INFINITY ? expf(s - m) : 0.f;
    const float S = warp_sumf(s);
    s = S == 0.f ? 0.f : s / S;
  }
  float ds = g;
  if (list_softmax) {
    ds = g - warp_sumf(g * s);
  } else if (renorm) {
    const float S = warp_sumf(s);
    const float dot = warp_sumf(g * s);
    ds = S == 0.f ? 0.f : g / S - dot / (S * S);
  }
  const float dot = row_softmax ? warp_sumf(ds * s) : 0.f;
  // an expert named twice gets the sum of its gradients
  float dsum = 0.f;
  for (int j = 0; j < k; ++j) {
    const int cj = __shfl_sync(0xffffffffu, col, j);
    const float dj = __shfl_sync(0xffffffffu, ds, j);
    if (cj == col) dsum += dj;
  }
  for (int e = lane; e < E; e += 32) o[e] = row_softmax ? -score(e) * dot : 0.f;
  __syncwarp();
  if (col >= 0) {
    float d = dsum;
    if (mode == 2) d = dsum * s * (1.0f - s);
    if (row_softmax) d = s * (dsum - dot);
    if (list_softmax) d = s * dsum;
    o[col] = d;
  }
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
  router_group_kernel<<<static_cast<unsigned>((T + kWarps - 1) / kWarps), 32 * kWarps,
                        kWarps * E * sizeof(double), reinterpret_cast<cudaStream_t>(stream)>>>(
      logits, bias, T, static_cast<int>(E), k, score_mode == 1, num_groups, topk_groups,
      group_score, renorm, scale, topk_vals, topk_idx, routing_map, probs);
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
  router_backward_kernel<<<static_cast<unsigned>((T + kWarps - 1) / kWarps), 32 * kWarps, 0,
                           reinterpret_cast<cudaStream_t>(stream)>>>(
      logits, bias, placement, topk_idx, grad_vals, grad_probs, T, static_cast<int>(E), k,
      score_mode, renorm, scale, grad_logits);
  MOE_CUDA_CHECK_LAUNCH("router_topk_backward launch");
  return MOE_OK;
}
