// Balance loss of a router with the experts' counts, and its gradient.
//
//   s_te = softmax over e of l_te, or sigmoid(l_te) / sum over e' of sigmoid(l_te')
//   loss = E / (K N^2) * sum_e c_e S_e,   S_e = sum over live t of s_te,   c_e = choices of e by live tokens (no gradient)
//   dl_te = g E / (K N^2) * s_te (c_e - sum_e' s_te' c_e')                         softmax
//   dl_te = g E / (K N^2) * sigmoid'(l_te) / sum_e' sigmoid(l_te') * (c_e - sum_e' s_te' c_e')   sigmoid
//
// A token's scores sum to one, so any constant may be taken from all counts: the gradient uses E c_e - sum of all counts, exact in whole
// numbers. Taken as they are, counts that are nearly equal (what the loss is for) cancel all but a few bits of an fp32 difference.
// What bounds it: HBM and instructions for many tokens (65536 x 256 in fp32, softmax: forward 19 us and the sums' 9, backward 25, where the bytes take 10 and 20),
// launches for few. A token's logits are spread over up to 32 lanes (a power of two), which keep their
// experts' sums over all their tokens in registers; a block leaves its sums, a cluster of blocks adds them in a fixed order, so that the loss
// does not change from run to run. Up to kOneBlock token groups a single block does it all in one launch.
#include <cooperative_groups.h>

#include <algorithm>

#include "api.h"
#include "early_start.cuh"

namespace fastb {

namespace {

using bf16 = __nv_bfloat16;
constexpr int kFoldCtas = 8, kFoldThreads = 1024;
constexpr int kOneBlock = 4;     // rounds of the one-block launch

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const bf16* p) { return __bfloat162float(__ldg(p)); }

// Sum and maximum over the G neighbouring lanes of a token.
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// 1 / sum of a token's scores; none: 0, so that its scores are 0.
__device__ __forceinline__ float inverse(float total) { return total > 0.0f ? 1.0f / total : 0.0f; }

// l: logits of my experts (-inf past the last) -> their shares of the token, to be multiplied by what is returned: 1 / their sum. slope, if wanted:
// sigmoid'(l), by the same factor (softmax: the share). Every value is taken through a maximum with 0, which turns NaN, a NaN logit's or that of -inf - -inf, into 0.
template <int G, int P, bool SIGMOID, bool SLOPE>
__device__ __forceinline__ float shares(float (&l)[P], float (&slope)[SLOPE ? P : 1]) {
  float total = 0.0f;
  if (SIGMOID) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float e = __expf(-fabsf(l[i])), d = 1.0f / (1.0f + e);   // exact towards both ends
      if (SLOPE) slope[i] = fmaxf(e * d * d, 0.0f);
      l[i] = fmaxf(l[i] >= 0.0f ? d : e * d, 0.0f);
      total += l[i];
    }
  } else {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < P; ++i) top = fmaxf(top, l[i]);
    top = lanes_max<G>(top);
    if (top == INFINITY) {   // the infinite ones share the token
#pragma unroll
      for (int i = 0; i < P; ++i) l[i] = l[i] == INFINITY ? 0.0f : -INFINITY;
      top = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      l[i] = fmaxf(__expf(l[i] - top), 0.0f);
      if (SLOPE) slope[i] = l[i];
      total += l[i];
    }
  }
  return inverse(lanes_sum<G>(total));
}

// Column sums and counts of a part of the tokens. A lane's experts are g, g + G, ..., P of them.
template <class T, int G, int P, bool SIGMOID>
__global__ void __launch_bounds__(P >= 16 ? 512 : 1024, 1) balance_kernel(const BalanceArgs a) {
  extern __shared__ int s_mem[];               // counts [E], then sums [warps][E]
  __shared__ int s_live;
  __shared__ float s_loss[32];
  int* s_count = s_mem;
  float* s_sum = reinterpret_cast<float*>(s_mem + a.E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane % G;
  constexpr int kTokens = 32 / G;              // of a warp at a time
  grid_dependency_wait();
  launch_dependents();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) s_count[e] = 0;
  if (threadIdx.x == 0) s_live = 0;
  __syncthreads();
  float acc[P], unused[1];
#pragma unroll
  for (int i = 0; i < P; ++i) acc[i] = 0.0f;
  int live = 0;
  const long long step = static_cast<long long>(gridDim.x) * warps * kTokens;
  long long t0 = (static_cast<long long>(blockIdx.x) * warps + warp) * kTokens;
  float next[P];
  bool next_on = false;
  int next_e = -1;                             // of the token's choices, mine
  const auto request = [&](long long first) {   // the next token is under way while this one is worked on
    const long long t = first + lane / G;
    const bool in = t < a.T;
    const T* row = static_cast<const T*>(a.logits) + (in ? t : 0) * a.stride;
#pragma unroll
    for (int i = 0; i < P; ++i) next[i] = in && g + i * G < a.E ? load_logit(row + g + i * G) : -INFINITY;
    next_e = in && g < a.K ? __ldg(a.topk_idx + t * a.K + g) : -1;
    next_on = in && (a.mask == nullptr || a.mask[t] != 0);
  };
  const auto count = [&](int e) { if (e >= 0 && e < a.E) atomicAdd(s_count + e, 1); };
  if (t0 < a.T) request(t0);
  for (; t0 < a.T; t0 += step) {   // all lanes of a warp alike
    const long long t = t0 + lane / G;
    const bool on = next_on;
    const int mine = next_e;
    float l[P];
#pragma unroll
    for (int i = 0; i < P; ++i) l[i] = next[i];
    if (t0 + step < a.T) request(t0 + step);
    if (on) {
      live += g == 0 ? 1 : 0;
      count(mine);
      for (int j = g + G; j < a.K; j += G) count(__ldg(a.topk_idx + t * a.K + j));
    }
    const float inv = shares<G, P, SIGMOID, false>(l, unused), factor = on ? inv : 0.0f;   // a padded token's logits have no part, whatever they are
#pragma unroll
    for (int i = 0; i < P; ++i) acc[i] = fmaf(l[i], factor, acc[i]);
  }
  if (live) atomicAdd(&s_live, live);
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (lane < G && g + i * G < a.E) s_sum[warp * a.E + g + i * G] = acc[i];
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      float v = 0.0f;
      for (int w = 0; w < warps; ++w) v += s_sum[w * a.E + e];
      a.sums[static_cast<size_t>(blockIdx.x) * a.E + e] = v;
      a.chosen[static_cast<size_t>(blockIdx.x) * (a.E + 1) + e] = s_count[e];
    }
    if (threadIdx.x == 0) a.chosen[static_cast<size_t>(blockIdx.x) * (a.E + 1) + a.E] = s_live;
    return;
  }
  float part = 0.0f;
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float v = 0.0f;
    for (int w = 0; w < warps; ++w) v += s_sum[w * a.E + e];
    a.counts[e] = a.kept[e] = s_count[e];
    part = fmaf(static_cast<float>(s_count[e]), v, part);
  }
  part = lanes_sum<32>(part);
  if (lane == 0) s_loss[warp] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < warps; ++w) part += s_loss[w];
    const float n = static_cast<float>(max(s_live, 1));
    *a.loss = part / n * (static_cast<float>(a.E) / (static_cast<float>(a.K) * n));
    a.kept[a.E] = s_live;
  }
}

// The blocks' sums and counts, added up by a cluster: CTA r takes every eighth block's, all experts side by side; then an eighth of the experts, from
// the CTAs' shared memory. Always in the same order. (An expert a warp, its lanes a row apart in memory, took 15 us for 296 blocks of 256 experts.)
__global__ void __cluster_dims__(kFoldCtas, 1, 1) __launch_bounds__(kFoldThreads) balance_fold_kernel(const BalanceArgs a, int blocks, int across) {
  namespace cg = cooperative_groups;
  __shared__ float s_v[kFoldThreads], s_sum[kBalanceMaxExperts], s_part[kFoldThreads / 32], s_all[kFoldCtas];
  __shared__ int s_n[kFoldThreads], s_count[kBalanceMaxExperts], s_live;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = kFoldThreads / across, slice = threadIdx.x / across;   // across: a power of two, as many experts as fit side by side
  grid_dependency_wait();
  launch_dependents();
  for (int e0 = 0; e0 < a.E; e0 += across) {
    const int e = e0 + threadIdx.x % across;
    float v = 0.0f;
    int n = 0;
    if (e < a.E) {
#pragma unroll 8
      for (int b = rank + kFoldCtas * slice; b < blocks; b += kFoldCtas * slices) {
        v += __ldcg(a.sums + static_cast<size_t>(b) * a.E + e);
        n += __ldcg(a.chosen + static_cast<size_t>(b) * (a.E + 1) + e);
      }
    }
    s_v[threadIdx.x] = v;
    s_n[threadIdx.x] = n;
    __syncthreads();
    if (slice == 0 && e < a.E) {
      for (int q = 1; q < slices; ++q) { v += s_v[threadIdx.x + q * across]; n += s_n[threadIdx.x + q * across]; }
      s_sum[e] = v;
      s_count[e] = n;
    }
    __syncthreads();
  }
  if (warp == 0) {
    int n = 0;
    for (int b = rank + kFoldCtas * lane; b < blocks; b += kFoldCtas * 32) n += __ldcg(a.chosen + static_cast<size_t>(b) * (a.E + 1) + a.E);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_live = n;
  }
  cluster.sync();
  float part = 0.0f;
  for (int e = rank + kFoldCtas * threadIdx.x; e < a.E; e += kFoldCtas * kFoldThreads) {
    float v = 0.0f;
    int n = 0;
#pragma unroll
    for (int r = 0; r < kFoldCtas; ++r) {
      v += *cluster.map_shared_rank(s_sum + e, r);
      n += *cluster.map_shared_rank(s_count + e, r);
    }
    a.counts[e] = a.kept[e] = n;
    part = fmaf(static_cast<float>(n), v, part);
  }
  part = lanes_sum<32>(part);
  if (lane == 0) s_part[warp] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kFoldThreads / 32; ++w) part += s_part[w];
    *cluster.map_shared_rank(s_all + rank, 0) = part;
  }
  int live = 0;
  if (rank == 0 && threadIdx.x == 0)
    for (int r = 0; r < kFoldCtas; ++r) live += *cluster.map_shared_rank(&s_live, r);
  cluster.sync();   // nobody leaves while its shared memory is read
  if (rank == 0 && threadIdx.x == 0) {
    part = 0.0f;
    for (int r = 0; r < kFoldCtas; ++r) part += s_all[r];
    const float n = static_cast<float>(max(live, 1));
    *a.loss = part / n * (static_cast<float>(a.E) / (static_cast<float>(a.K) * n));
    a.kept[a.E] = live;
  }
}

template <class T, int G, int P, bool SIGMOID>
__global__ void __launch_bounds__(256) balance_bwd_kernel(const BalanceBwdArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane % G;
  constexpr int kTokens = 32 / G;
  grid_dependency_wait();
  launch_dependents();
  // E c_e - sum of all counts, and g / (K N^2)
  float d[P];
  long long all = 0;
  int c[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    c[i] = g + i * G < a.E ? __ldg(a.kept + g + i * G) : 0;
    all += c[i];
  }
#pragma unroll
  for (int o = G / 2; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll
  for (int i = 0; i < P; ++i) d[i] = g + i * G < a.E ? static_cast<float>(static_cast<long long>(a.E) * c[i] - all) : 0.0f;
  const float n = static_cast<float>(max(__ldg(a.kept + a.E), 1)), factor = __ldg(a.dloss) / n / (static_cast<float>(a.K) * n);
  const long long step = static_cast<long long>(gridDim.x) * warps * kTokens;
  for (long long t0 = (static_cast<long long>(blockIdx.x) * warps + warp) * kTokens; t0 < a.T; t0 += step) {
    const long long t = t0 + lane / G;
    const bool on = t < a.T && (a.mask == nullptr || a.mask[t] != 0);
    const T* row = static_cast<const T*>(a.logits) + (on ? t : 0) * a.stride;
    float l[P], slope[P];
#pragma unroll
    for (int i = 0; i < P; ++i) l[i] = on && g + i * G < a.E ? load_logit(row + g + i * G) : -INFINITY;
    const float inv = shares<G, P, SIGMOID, true>(l, slope);
    float mean = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) mean = fmaf(l[i], d[i], mean);
    mean = lanes_sum<G>(mean) * inv;
    if (t >= a.T) continue;
    T* out = static_cast<T*>(a.dlogits) + t * a.E;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (g + i * G >= a.E) continue;
      const float v = on ? slope[i] * inv * (d[i] - mean) * factor : 0.0f;   // the small factor last: slopes may be tiny
      if constexpr (sizeof(T) == 2) out[g + i * G] = __float2bfloat16_rn(v);
      else out[g + i * G] = v;
    }
  }
}

// Lanes of a token and experts of a lane.
int lanes_for(int E) { int g = 2; while (g < 32 && g < E) g *= 2; return g; }

template <class F>
cudaError_t with_shape(int E, bool is_bf16, bool sigmoid, F f) {
  const auto go = [&](auto g, auto p) {
    if (is_bf16) return sigmoid ? f(bf16{}, g, p, std::true_type()) : f(bf16{}, g, p, std::false_type());
    return sigmoid ? f(float{}, g, p, std::true_type()) : f(float{}, g, p, std::false_type());
  };
  using one = std::integral_constant<int, 1>;
  if (E <= 2) return go(std::integral_constant<int, 2>(), one());
  if (E <= 4) return go(std::integral_constant<int, 4>(), one());
  if (E <= 8) return go(std::integral_constant<int, 8>(), one());
  if (E <= 16) return go(std::integral_constant<int, 16>(), one());
  if (E <= 32) return go(std::integral_constant<int, 32>(), one());
  if (E <= 64) return go(std::integral_constant<int, 32>(), std::integral_constant<int, 2>());
  if (E <= 128) return go(std::integral_constant<int, 32>(), std::integral_constant<int, 4>());
  if (E <= 256) return go(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
  if (E <= 512) return go(std::integral_constant<int, 32>(), std::integral_constant<int, 16>());
  return go(std::integral_constant<int, 32>(), std::integral_constant<int, 32>());
}

// Threads of a block. Large ones: every block leaves sums that have to be added up (256 experts: 592 blocks of 256 threads took 7.7 + 11.5 us).
int block_for(int E) { return E > 256 ? 512 : 1024; }

}  // namespace

int balance_blocks(const BalanceArgs& a, int sms) {
  const int per_warp = 32 / lanes_for(a.E);
  const int per_block = block_for(a.E) / 32 * per_warp;
  if (a.T <= kOneBlock * per_block) return 1;
  return std::min(1024 / block_for(a.E) * sms, (a.T + per_block - 1) / per_block);
}

cudaError_t launch_balance(const BalanceArgs& a, int blocks, cudaStream_t stream) {
  if (a.T < 0 || a.E < 1 || a.E > kBalanceMaxExperts || a.K < 1 || blocks < 1 || (blocks > 1 && (a.sums == nullptr || a.chosen == nullptr))) return cudaErrorInvalidValue;
  const int threads = block_for(a.E);
  const size_t smem = static_cast<size_t>(a.E) * 4 * (1 + threads / 32);
  cudaError_t e = with_shape(a.E, a.logits_bf16 != 0, a.sigmoid != 0, [&](auto t, auto g, auto p, auto s) {
    auto kern = balance_kernel<decltype(t), decltype(g)::value, decltype(p)::value, decltype(s)::value>;
    const cudaError_t err = allow_smem(kern, smem);
    return err != cudaSuccess ? err : launch_early(kern, dim3(blocks), threads, smem, stream, a);
  });
  note_launch();
  if (e != cudaSuccess || blocks == 1) return e;
  int across = 1;
  while (across < a.E && across < kFoldThreads) across *= 2;
  e = launch_early(balance_fold_kernel, dim3(kFoldCtas), kFoldThreads, 0, stream, a, blocks, across);
  note_launch();
  return e;
}

cudaError_t launch_balance_bwd(const BalanceBwdArgs& a, int sms, cudaStream_t stream) {
  if (a.T < 0 || a.E < 1 || a.E > kBalanceMaxExperts || a.K < 1) return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  const int per_block = 8 * (32 / lanes_for(a.E));
  const int blocks = std::min(8 * sms, (a.T + per_block - 1) / per_block);
  const cudaError_t e = with_shape(a.E, a.logits_bf16 != 0, a.sigmoid != 0, [&](auto t, auto g, auto p, auto s) {
    return launch_early(balance_bwd_kernel<decltype(t), decltype(g)::value, decltype(p)::value, decltype(s)::value>, dim3(blocks), 256, 0, stream, a);
  });
  note_launch();
  return e;
}

}  // namespace fastb
