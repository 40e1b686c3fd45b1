// A linear layer on a few tokens: out = act(x W^T + bias) + residual, or SwiGLU, in tiles of 128 rows of the weight by up to kFewTokens tokens; and
// its data gradient, x W, in tiles of 128 of its columns.
//
// What bounds it: the weight's bytes. A cluster of CTAs has a tile and shares out the reduction; a CTA streams its part of the weight's
// rows through shared memory (TMA) as operand A of M = 128 MMAs, the tokens are N (rounded up to 16), so a decode step does no more work
// than its tokens are. Each CTA finishes an equal share of the tile's features: the others send it their fp32 sums through distributed shared memory, it
// adds them up in the order of the reduction (bias, activation, residual, store): no counters, no scratch in global memory, nothing to
// clear beforehand, one launch. 1 token, weight from HBM: 4096 -> 14336 21 us (5.6 TB/s), 14336 -> 4096 21.6 us, 4096 -> 4096 9.0 us (3.7 TB/s; 3 us of a launch are setting up,
// the first loads and the sums' way). A launch of no more CTAs than SMs has all their shared memory for stages; a larger one, half: two CTAs an SM. With
// hundreds of tokens the bound is a CTA's way from L2: 32 KiB in 0.23 us, whether or not two CTAs share the tokens in one MMA of M = 256 (512 x 4096 -> 4096 17.8 and 17.7 us).
// SwiGLU: the 128 rows are 64 gate rows and the 64 up rows of the same features.
#include <algorithm>

#include "early_start.cuh"
#include "gemm_common.cuh"

namespace fastb {

namespace {

using namespace ptx;
using namespace gemm;

constexpr int kRows = 128;                       // of the weight, a tile
constexpr int kThreads = 256;                    // two warps for every quarter of tensor memory
constexpr int kMaxStages = 12;
constexpr int kFewABytes = kRows * BK * 2;       // 16 KiB
constexpr int kFewSmem = 110 * 1024, kFewDeepSmem = 220 * 1024;   // of an SM's two CTAs each, or of its only one
__host__ __device__ constexpr int few_stage(int n) { return kFewABytes + n * BK * 2; }

struct __align__(8) FewCtl {
  uint64_t full[kMaxStages], empty[kMaxStages], done, products;
  uint32_t tmem_base;
  int abort_flag, issued;   // blocks whose loads were requested, where the launch gave up
};
// The fp32 sums: where the stages were, or, where they are few and of several CTAs, beside them: a peer's may come while this CTA still multiplies.
__host__ __device__ constexpr int few_sums(int n) { return n * kRows * 4; }
__host__ __device__ constexpr bool few_beside(int n, int parts) { return parts > 1 && n <= 64; }
__host__ __device__ constexpr int few_room(int n, int parts, int stages) {
  const int operands = stages * few_stage(n);
  return few_beside(n, parts) ? operands + few_sums(n) : operands > few_sums(n) ? operands : few_sums(n);
}
constexpr int kFewOther = 1024 + static_cast<int>(sizeof(FewCtl));
constexpr int few_stages(int n, int parts, int smem) { return std::min(kMaxStages, (smem - kFewOther - (few_beside(n, parts) ? few_sums(n) : 0)) / few_stage(n)); }
constexpr int few_smem(int n, int parts, int stages) { return few_room(n, parts, stages) + kFewOther; }
constexpr int few_most(int n, int parts, int smem) { return few_smem(n, parts, few_stages(n, parts, smem)); }
static_assert(few_stages(16, 8, kFewSmem) >= 5 && few_stages(kFewTokens, 1, kFewSmem) >= 3 && few_most(kFewTokens, 1, kFewSmem) <= kFewSmem && few_most(16, 8, kFewSmem) <= kFewSmem &&
              few_most(64, 4, kFewDeepSmem) <= kFewDeepSmem && few_most(kFewTokens, 4, kFewDeepSmem) <= kFewDeepSmem, "stages at both ends of the range");

__device__ __forceinline__ float4 ld_sums(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void st_own(uint32_t addr, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint2 pack4(const float4& v) { return make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)); }
__device__ __forceinline__ uint2 rest4(const float4& v) { return make_uint2(pack_rest(v.x, v.y), pack_rest(v.z, v.w)); }
__device__ __forceinline__ float4 unpack4(const __nv_bfloat16* at) {
  const uint2 v = *reinterpret_cast<const uint2*>(at);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <Activation ACT>
__device__ __forceinline__ float activated(float z) {
  return ACT == Activation::kRelu ? relu(z) : ACT == Activation::kSilu ? silu(z) : ACT == Activation::kGelu ? gelu(z) : z;
}

// DGRAD: out = x W, the weight's columns are the features (operand A MN-major).
template <Activation ACT, bool SWIGLU, bool DGRAD, int PARTS>
__global__ void __launch_bounds__(kThreads) linear_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const FewArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int n = p.n, stage_size = few_stage(n), stages = p.stages;
  const uint32_t sums = smem_u32(tiles) + (few_beside(n, PARTS) ? stages * stage_size : 0);
  FewCtl* ctl = reinterpret_cast<FewCtl*>(tiles + few_room(n, PARTS, stages));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = static_cast<int>(cluster_cta_rank());
  const int tile = blockIdx.x / PARTS, t0 = blockIdx.y * n, T = min(n, p.T - t0);   // rows of the weight, tokens
  constexpr int F = SWIGLU ? kRows / 2 : kRows, MINE = F / PARTS;   // features of a tile, and those that I finish
  const uint32_t columns = n <= 32 ? 32 : n <= 64 ? 64 : 128;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&ctl->full[s], 1); mbar_init(&ctl->empty[s], 1); }
    mbar_init(&ctl->done, 1);
    mbar_init(&ctl->products, 1);
    ctl->abort_flag = ctl->issued = 0;
    mbar_fence_init();
    prefetch_tmap(&map_w);
    prefetch_tmap(&map_x);
  }
  if (warp == 1) { tmem_alloc(&ctl->tmem_base, columns); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  if (few_beside(n, PARTS)) cluster_arrive();
  tc_fence_after_sync();
  const uint32_t tmem = ctl->tmem_base;
  volatile int* abort_flag = &ctl->abort_flag;
  grid_dependency_wait();
  launch_dependents();
  // This CTA's blocks of 64 of the reduction; a part has one at least.
  const int kb0 = static_cast<int>(static_cast<long long>(p.red_blocks) * rank / PARTS), kb1 = static_cast<int>(static_cast<long long>(p.red_blocks) * (rank + 1) / PARTS), blocks = kb1 - kb0;
  if (warp == 0) {
    if (elect_one()) {
      uint32_t ph = 0;
      int i = 0;
      for (int s = 0; i < blocks; ++i) {
        if (i >= stages && !mbar_wait_bounded(&ctl->empty[s], ph ^ 1, abort_flag, p.status, 100 + s, p.timeout_ns)) break;
        uint8_t* sa = tiles + s * stage_size;
        const int k = (kb0 + i) * BK;
        mbar_arrive_expect_tx(&ctl->full[s], static_cast<uint32_t>(stage_size));
        if (SWIGLU) {   // tile t: 64 features from half t % 2 of the weight's 256-row tile t / 2
          const int gate = tile / 2 * 256 + tile % 2 * 64;
          tma_load_2d(sa, &map_w, k, gate, &ctl->full[s]);
          tma_load_2d(sa + kFewABytes / 2, &map_w, k, gate + 128, &ctl->full[s]);
        } else if (DGRAD) {
#pragma unroll
          for (int j = 0; j < kRows / 64; ++j) tma_load_2d(sa + j * (BK * 128), &map_w, tile * kRows + j * 64, k, &ctl->full[s]);
        } else {
          tma_load_2d(sa, &map_w, k, tile * kRows, &ctl->full[s]);
        }
        tma_load_2d(sa + kFewABytes, &map_x, k, t0, &ctl->full[s]);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      ctl->issued = i;
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc_bf16(kRows, n, DGRAD, false);
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0, s = 0; i < blocks; ++i) {
        if (!(ok = mbar_wait_bounded(&ctl->full[s], ph, abort_flag, p.status, 300 + s, p.timeout_ns))) break;
        tc_fence_after_sync();
        const uint32_t sa = smem_u32(tiles + s * stage_size), sb = sa + kFewABytes;
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)
          mma_bf16_ss(tmem, DGRAD ? make_smem_desc(sa + k * 2048, BK * 128, 1024) : make_smem_desc(sa + k * 32, 16, 1024), make_smem_desc(sb + k * 32, 16, 1024), idesc, (i | k) != 0 ? 1u : 0u);
        mma_commit(&ctl->empty[s]);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (ok) mma_commit(&ctl->done);
      else { mma_commit(&ctl->products); mbar_drain(&ctl->products, 0); }
    }
  }
  __syncwarp();
  const bool ok = mbar_wait_warp(&ctl->done, 0, abort_flag, p.status, 400, p.timeout_ns);
  tc_fence_after_sync();
  // Four features of a token (SwiGLU: their gates and ups) on their way out.
  const auto finish = [&](int token, int f, float4 v, const float4& up) {
    const int t = t0 + token, col = tile * F + f;
    if (col >= p.columns) return;
    if (p.bias != nullptr) {
      const float4 b = unpack4(p.bias + col);
      v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
    }
    const long long at = static_cast<long long>(t) * p.columns + col;
    if (SWIGLU) {
      if (p.pre != nullptr) {
        __nv_bfloat16* gu = p.pre + static_cast<long long>(t) * p.columns * 4 + tile / 2 * 256 + tile % 2 * 64 + f;
        *reinterpret_cast<uint2*>(gu) = pack4(v);
        *reinterpret_cast<uint2*>(gu + 128) = pack4(up);
        *reinterpret_cast<uint2*>(gu + 2 * p.columns) = rest4(v);
        *reinterpret_cast<uint2*>(gu + 2 * p.columns + 128) = rest4(up);
      }
      v.x = silu(v.x) * up.x; v.y = silu(v.y) * up.y; v.z = silu(v.z) * up.z; v.w = silu(v.w) * up.w;
    } else {
      if (p.pre != nullptr) *reinterpret_cast<uint2*>(p.pre + at) = pack4(v);
      v.x = activated<ACT>(v.x); v.y = activated<ACT>(v.y); v.z = activated<ACT>(v.z); v.w = activated<ACT>(v.w);
    }
    if (p.residual != nullptr) {
      const float4 r = unpack4(p.residual + t * p.residual_stride + col);
      v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
    }
    *reinterpret_cast<uint2*>(p.out + at) = pack4(v);
  };
  const int quarter = warp & 3;                                         // of tensor memory, and of the features
  const auto load = [&](int c, uint32_t (&r)[32]) {
    tmem_ld_32x32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, r);
    tmem_wait_ld();
  };
  // Every CTA sends its sums to the CTA of the cluster that finishes them, [part][token][feature], and reads what has come to it: the way to a peer's
  // shared memory is not waited for value by value, and after one barrier nobody touches another's.
  constexpr int WIDTH = kRows / PARTS;                                // floats of a token
  const int fl = quarter * 32 + lane, owner = fl % F / MINE;
  const uint32_t own = sums + (rank * n * WIDTH + fl / F * MINE + fl % MINE) * 4, to = PARTS > 1 ? map_to_cta(own, owner) : own;
  if (PARTS > 1 && !few_beside(n, PARTS)) cluster_sync_all();          // the peers' products are done too
  else if (PARTS > 1) cluster_wait();                                   // the peers are there
  for (int c = (warp >> 2) * 32; ok && c < T; c += 64) {
    uint32_t r[32];
    load(c, r);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i < T) {
        if (PARTS > 1) st_cluster(to + (c + i) * WIDTH * 4, r[i]);
        else st_own(to + (c + i) * WIDTH * 4, r[i]);
      }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (PARTS > 1) cluster_sync_all();
  constexpr int Q = MINE / 4, U = SWIGLU || PARTS >= 8 ? 2 : 4;       // U in flight
  for (int i0 = threadIdx.x; ok && i0 < T * Q; i0 += U * kThreads) {
    float4 z[U], u[SWIGLU ? U : 1];
    const auto gather = [&](int add, float4* sum) {                   // in the order of the reduction
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = min(i0 + j * kThreads, T * Q - 1);
        const uint32_t at = sums + static_cast<uint32_t>(i / Q * WIDTH + i % Q * 4 + add) * 4u;
        sum[j] = ld_sums(at);
#pragma unroll
        for (int q = 1; q < PARTS; ++q) {
          const float4 w = ld_sums(at + static_cast<uint32_t>(q * n * WIDTH) * 4u);
          sum[j].x += w.x; sum[j].y += w.y; sum[j].z += w.z; sum[j].w += w.w;
        }
      }
    };
    gather(0, z);
    if (SWIGLU) gather(MINE, u);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * kThreads;
      if (i < T * Q) finish(i / Q, rank * MINE + i % Q * 4, z[j], u[SWIGLU ? j : 0]);
    }
  }
  __syncwarp();
  // Given up: not before the products and the loads that are still on their way. (A warp that saw the products done saw the loads done too.)
  if (!ok && warp == 1) {
    if (lane == 0) { mbar_drain(&ctl->done, 0); drain_loads(ctl->full, ctl->issued, stages); }
    __syncwarp();
  }
  if (warp == 1) tmem_dealloc(tmem, columns);
}

}  // namespace

// How many CTAs share a tile's reduction: as many as leave every CTA an SM of its own, whose shared memory it then has for stages (what a CTA has under way
// at a time bounds its stream), and eight blocks of the reduction; eight, two an SM, only where up to 16 tokens make the sums small, for a larger cluster is harder
// to place and its sums travel further. us with 1, 2, 4, 8 CTAs of half an SM's shared memory / of all of it: 32 tiles of 64 blocks (4096 -> 4096), 1 token
// 15.1, 10.7, 9.4, 9.3 / 12.8, 9.6, 9.6, 17.2, 64 tokens 21.2, 14.1, 11.8, 13.0 / 13.7, 10.5, 10.8, 22.5, 128 tokens 26.4, 17.0, 13.1, 16.1 / 17.6, 13.2, 11.9, 27.2;
// 32 tiles of 16, 128 tokens 9.5, 8.2, 7.9, 15.7 / 7.5, 7.4, 7.7, 15.6; 56 of 32 (2048 -> 7168), 48 tokens 12.5, 10.4, 10.3 / 9.0, 9.2, 14.5; 112 of 64 (4096 -> 14336), 64
// tokens 28.0, 24.1, 31.2 / 23.5, 28.0, 38.6; 32 of 224 (14336 -> 4096), 1 token 45.8, 28.0, 23.0, 22.0 / 38.0, 23.6, 22.7, 31.4.
int few_parts(int tiles, int red_blocks, int n, int sms) {
  int parts = 1;
  while (parts < 4 && 2 * tiles * parts <= sms && 8 * 2 * parts <= red_blocks) parts *= 2;
  return n <= 16 && parts == 4 && 4 * tiles <= sms && red_blocks >= 64 ? 8 : parts;
}
FewPlan few_plan(int T, int columns, int red_blocks, bool swiglu, int sms) {
  FewPlan f{};
  const int per_tile = swiglu ? kRows / 2 : kRows;
  f.tiles = (columns + per_tile - 1) / per_tile;
  f.token_tiles = (T + kFewTokens - 1) / kFewTokens;
  f.n = ((T + f.token_tiles - 1) / f.token_tiles + 15) / 16 * 16;
  f.token_tiles = (T + f.n - 1) / f.n;
  f.parts = few_parts(f.tiles * f.token_tiles, red_blocks, f.n, sms);
  f.stages = std::min(few_stages(f.n, f.parts, f.tiles * f.token_tiles * f.parts <= sms ? kFewDeepSmem : kFewSmem), (red_blocks + f.parts - 1) / f.parts);
  f.smem = few_smem(f.n, f.parts, f.stages);
  return f;
}

// Against the kernel with tiles of 256 features by up to 256 tokens (grouped_gemm_tokens.cu), which reads half as much per product but takes 4 us more to
// begin and end. Ahead with up to 64 tokens, and otherwise the longer the fewer rounds of the GPU its tiles take. us, that kernel -> this one: 1 token 4096 -> 57344
// 83.0 -> 72.4, 64 tokens 86.3 -> 79.7, 128 tokens 4096 -> 32000 49.9 -> 50.0; half a round (64 tiles), 256 x 14336 -> 4096 49.6 -> 34.1; a round (96 to 128 tiles): 64 blocks of the
// reduction, 96 x 4096 -> 14336 25.4 -> 23.3, 112 blocks, 500 x 7168 -> 4096 SwiGLU 29.8 -> 29.8, 224 blocks, 384 x 14336 -> 4096 47.2 -> 51.5; two rounds: 16 blocks, 1024 x 1024 -> 4096 12.4 ->
// 11.0, 32 blocks, 384 x 2048 -> 7168 14.6 -> 17.0; four rounds: 4 blocks, 2048 x 256 -> 4096 11.6 -> 11.2, 8 blocks 13.0 -> 14.4. Rows that do not start at sectors of 32 bytes
// come in more slowly, which weighs on what reads more: 1235 x 1000 -> 2760 (two rounds, 16 blocks) 12.9 -> 16.7.
bool few_pays(int T, int columns, int red_blocks, bool swiglu, bool sectors, int sms) {
  const int per_tile = swiglu ? kRows / 2 : kRows;
  const long long tiles = static_cast<long long>((columns + per_tile - 1) / per_tile) * ((T + kFewTokens - 1) / kFewTokens);
  if (T <= 64 || 2 * tiles <= sms) return true;
  return red_blocks <= (tiles <= sms ? 112 : !sectors ? 0 : tiles <= 2 * sms ? 16 : tiles <= 4 * sms ? 4 : 0);
}

cudaError_t launch_linear_few(GemmMode mode, Activation act, bool swiglu, const CUtensorMap& map_w, const CUtensorMap& map_x, const FewArgs& args, int sms, cudaStream_t stream) {
  FewArgs a = args;
  if (a.T < 1 || a.columns < 1 || a.red_blocks < 1 || a.status == nullptr || (mode != GemmMode::kForward && (mode != GemmMode::kDgrad || swiglu || act != Activation::kNone)) || (swiglu && (act != Activation::kNone || a.columns % 128))) return cudaErrorInvalidValue;
  const FewPlan f = few_plan(a.T, a.columns, a.red_blocks, swiglu, sms);
  if (f.token_tiles > 65535) return cudaErrorInvalidValue;
  a.n = f.n;
  a.stages = f.stages;
  const auto go = [&](auto kern) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, f.smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(f.tiles * f.parts, f.token_tiles);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = f.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = f.parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1] = early_start_attribute();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, map_w, map_x, a);
  };
  const auto with = [&](auto act_c, auto swiglu_c, auto dgrad_c) {
    constexpr Activation ACT = decltype(act_c)::value;
    constexpr bool SWIGLU = decltype(swiglu_c)::value, DGRAD = decltype(dgrad_c)::value;
    switch (f.parts) {
      case 1: return go(linear_few_kernel<ACT, SWIGLU, DGRAD, 1>);
      case 2: return go(linear_few_kernel<ACT, SWIGLU, DGRAD, 2>);
      case 4: return go(linear_few_kernel<ACT, SWIGLU, DGRAD, 4>);
      case 8: return go(linear_few_kernel<ACT, SWIGLU, DGRAD, 8>);
      default: return cudaErrorInvalidValue;
    }
  };
  using std::integral_constant;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  using none = integral_constant<Activation, Activation::kNone>;
  cudaError_t e;
  if (mode == GemmMode::kDgrad) e = with(none(), no, yes);
  else if (swiglu) e = with(none(), yes, no);
  else if (act == Activation::kRelu) e = with(integral_constant<Activation, Activation::kRelu>(), no, no);
  else if (act == Activation::kSilu) e = with(integral_constant<Activation, Activation::kSilu>(), no, no);
  else if (act == Activation::kGelu) e = with(integral_constant<Activation, Activation::kGelu>(), no, no);
  else e = with(none(), no, no);
  if (e == cudaSuccess) note_launch();
  return e;
}

}  // namespace fastb
