// RMS norm of rows with the residual's addition in front of it, its e4m3 output and its backward pass.
//
//   forward    h = T(x + residual);  r = 1 / sqrt(mean(h^2) + eps);  y = T(h r w);  q, scales = y in e4m3, one scale per 128 columns
//   backward   g = dy w;  s = mean(g h r);  dx = r (g - h r s) + dh;  dw = sum over rows of dy h r
//
// The sum is rounded to the rows' type before anything else: that is the residual stream which the caller keeps, and the backward pass
// has nothing but it. q is made from the rounded y, so that it is what the dispatch would send for y, bit for bit. Sums are fp32.
// What bounds it: HBM. A row is read once and stays in registers between the sum of squares and the output.
#include <algorithm>

#include "api.h"
#include "e4m3_rows.cuh"
#include "early_start.cuh"

namespace fastb {

namespace {

using bf16 = __nv_bfloat16;

// 16 bytes of a row as floats.
template <class T> struct Pack;
template <> struct Pack<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[N]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 t = __bfloat1622float2(h[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[N]) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
};
template <> struct Pack<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float (&f)[N]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[N]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <class T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <class T> __device__ __forceinline__ T as_type(float v);
template <> __device__ __forceinline__ bf16 as_type(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float as_type(float v) { return v; }
template <class T> __device__ __forceinline__ float rounded(float v) { return as_float<T>(as_type<T>(v)); }

// N consecutive weights from column N c on, whatever their type.
template <class W, int N>
__device__ __forceinline__ void load_weight(const void* weight, int c, float (&w)[N]) {
  const W* at = static_cast<const W*>(weight) + static_cast<size_t>(c) * N;
  if constexpr (sizeof(W) * N == 16) {
    Pack<W>::get(__ldg(reinterpret_cast<const uint4*>(at)), w);
  } else if constexpr (sizeof(W) * N == 32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));   // four bf16
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
    w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the warps of a row; every thread of the block calls it. part: a slot per warp, not written again before the next barrier but one.
__device__ __forceinline__ float row_sum(float v, float* part, int warp, int wpr) {
  v = warp_sum(v);
  if (wpr == 1) return v;
  if ((threadIdx.x & 31) == 0) part[warp] = v;
  __syncthreads();
  const int first = warp / wpr * wpr;
  v = 0.0f;
  for (int i = 0; i < wpr; ++i) v += part[first + i];
  return v;
}

// Most warps of a block whose lanes hold C chunks of 16 bytes.
constexpr int warps_for(int C) { return C <= 2 ? 8 : 16; }

// wpr warps hold a row in registers, C chunks of 16 bytes a lane; a block has several rows where they are short.
template <class T, class W, int C, bool RES, bool QUANT>
__global__ void __launch_bounds__(32 * warps_for(C)) row_norm_kernel(const RowNormArgs a) {
  constexpr int N = Pack<T>::N;
  __shared__ float s_part[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wpr = a.warps_per_row, lanes = 32 * wpr;
  const int row = blockIdx.x * (static_cast<int>(blockDim.x >> 5) / wpr) + warp / wpr, l = warp % wpr * 32 + lane, chunks = a.H / N;
  const bool live = row < a.T;
  const long long t = live ? row : 0;
  grid_dependency_wait();
  launch_dependents();
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + t * a.x_stride);
  const uint4* res = reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + t * a.residual_stride);
  uint4 v[C], u[RES ? C : 1];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = l + i * lanes;
    const bool in = live && c < chunks;
    v[i] = in ? __ldcs(x + c) : make_uint4(0, 0, 0, 0);
    if (RES) u[i] = in ? __ldcs(res + c) : make_uint4(0, 0, 0, 0);
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    float f[N];
    Pack<T>::get(v[i], f);
    if (RES) {
      float g[N];
      Pack<T>::get(u[i], g);
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] += g[k];
      v[i] = Pack<T>::put(f);
      const int c = l + i * lanes;
      if (live && c < chunks) reinterpret_cast<uint4*>(static_cast<T*>(a.h) + t * a.H)[c] = v[i];
      Pack<T>::get(v[i], f);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) ss = fmaf(f[k], f[k], ss);
  }
  const float r = rsqrtf(row_sum(ss, s_part, warp, wpr) / static_cast<float>(a.H) + a.eps);
  if (a.rstd != nullptr && live && l == 0) a.rstd[t] = r;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = l + i * lanes;
    const bool in = live && c < chunks;
    float f[N], w[N];
    Pack<T>::get(v[i], f);
    load_weight<W, N>(a.weight, min(c, chunks - 1), w);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = f[k] * r * w[k];
    const uint4 y = Pack<T>::put(f);
    if (in) reinterpret_cast<uint4*>(static_cast<T*>(a.y) + t * a.H)[c] = y;
    if (QUANT) {
      constexpr int kGroup = 128 / N;   // lanes that share a scale; chunks of a group are neighbours in a warp, all in or all out
      Pack<T>::get(y, f);
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < N; ++k) amax = fmaxf(amax, fabsf(f[k]));
#pragma unroll
      for (int o = kGroup / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float sc = e4m3_scale(amax), inv = 1.0f / sc;
      unsigned short p[N / 2];
#pragma unroll
      for (int k = 0; k < N / 2; ++k) p[k] = e4m3_pair(f[2 * k], f[2 * k + 1], inv);
      if (in) {
        unsigned int* q = reinterpret_cast<unsigned int*>(a.q + t * a.H) + c * (N / 4);
        if (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(p[0] | p[1] << 16, p[N / 2 - 2] | p[N / 2 - 1] << 16);
        else *q = p[0] | p[1] << 16;
        if (lane % kGroup == 0) a.scales[t * (a.H / 128) + c / kGroup] = sc;
      }
    }
  }
}

// Any hidden size, any stride, any alignment: element by element, the row read twice (the second time from the cache). A warp takes 128 columns.
template <class T, class W, bool RES, bool QUANT>
__global__ void __launch_bounds__(256) row_norm_any_kernel(const RowNormArgs a) {
  __shared__ float s_part[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, groups = (a.H + 127) / 128;
  const long long t = blockIdx.x;
  grid_dependency_wait();
  launch_dependents();
  const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
  const T* res = static_cast<const T*>(a.residual) + t * a.residual_stride;
  T* h = static_cast<T*>(a.h) + t * a.H;
  T* y = static_cast<T*>(a.y) + t * a.H;
  const auto sum_at = [&](int c) {
    const float f = as_float<T>(x[c]);
    return RES ? rounded<T>(f + as_float<T>(res[c])) : f;
  };
  float ss = 0.0f;
  for (int g = warp; g < groups; g += warps)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = g * 128 + 32 * k + lane;
      if (c >= a.H) continue;
      const float f = sum_at(c);
      if (RES) h[c] = as_type<T>(f);
      ss = fmaf(f, f, ss);
    }
  const float r = rsqrtf(row_sum(ss, s_part, warp, warps) / static_cast<float>(a.H) + a.eps);
  if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[t] = r;
  for (int g = warp; g < groups; g += warps) {
    float f[4];
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = g * 128 + 32 * k + lane;
      if (c >= a.H) { f[k] = 0.0f; continue; }
      const T out = as_type<T>(sum_at(c) * r * as_float<W>(static_cast<const W*>(a.weight)[c]));
      y[c] = out;
      f[k] = as_float<T>(out);
      amax = fmaxf(amax, fabsf(f[k]));
    }
    if (QUANT) {
#pragma unroll
      for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float sc = e4m3_scale(amax), inv = 1.0f / sc;
#pragma unroll
      for (int k = 0; k < 4; ++k) a.q[t * a.H + g * 128 + 32 * k + lane] = static_cast<unsigned char>(e4m3_pair(f[k], 0.0f, inv));
      if (lane == 0) a.scales[t * (a.H / 128) + g] = sc;
    }
  }
}

// Backward: blocks walk the rows, a thread keeps the same columns for all of them and with them their part of the weight's gradient; the
// next row's loads are under way while this one is worked on. 16 columns a lane and up to 16 warps a row: with 32 columns the registers spill
// (forward + backward of 8192 x 7168 216 us, this 156; 16384 x 4096 171, 96 % of the copy bandwidth; 16384 x 1024 52, 78 %).
constexpr int kBwdWarps = 16;
template <class T, class W, int C, bool DH>
__global__ void __launch_bounds__(32 * kBwdWarps) row_norm_bwd_kernel(const RowNormBwdArgs a) {
  constexpr int N = Pack<T>::N;
  extern __shared__ float s_dw[];            // [H], blocks of several rows
  __shared__ float s_part[2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wpr = a.warps_per_row, lanes = 32 * wpr, rows = static_cast<int>(blockDim.x >> 5) / wpr;
  const int mine = warp / wpr, l = warp % wpr * 32 + lane, chunks = a.H / N;
  grid_dependency_wait();
  launch_dependents();
  float dw[C][N];
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = 0.0f;
  uint4 nh[C], ny[C], nd[DH ? C : 1];
  float nr = 0.0f;
  const auto request = [&](long long t) {
    const bool live = t < a.T;
    const uint4* h = reinterpret_cast<const uint4*>(static_cast<const T*>(a.h) + (live ? t : 0) * a.h_stride);
    const uint4* dy = reinterpret_cast<const uint4*>(static_cast<const T*>(a.dy) + (live ? t : 0) * a.H);
    const uint4* dh = reinterpret_cast<const uint4*>(static_cast<const T*>(a.dh) + (live ? t : 0) * a.H);
    nr = live ? __ldg(a.rstd + t) : 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = l + i * lanes;
      const bool in = live && c < chunks;
      nh[i] = in ? __ldcs(h + c) : make_uint4(0, 0, 0, 0);
      ny[i] = in ? __ldcs(dy + c) : make_uint4(0, 0, 0, 0);
      if (DH) nd[i] = in ? __ldcs(dh + c) : make_uint4(0, 0, 0, 0);
    }
  };
  const long long step = static_cast<long long>(gridDim.x) * rows;
  long long t0 = static_cast<long long>(blockIdx.x) * rows;
  request(t0 + mine);
  for (int buf = 0; t0 < a.T; t0 += step, buf ^= 1) {   // the same number of rounds for all warps of the block
    uint4 h[C], dy[C], dh[DH ? C : 1];
    const float r = nr;
#pragma unroll
    for (int i = 0; i < C; ++i) { h[i] = nh[i]; dy[i] = ny[i]; if (DH) dh[i] = nd[i]; }
    request(t0 + step + mine);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float fh[N], fy[N], w[N];
      Pack<T>::get(h[i], fh);
      Pack<T>::get(dy[i], fy);
      load_weight<W, N>(a.weight, min(l + i * lanes, chunks - 1), w);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float p = fy[k] * (fh[k] * r);
        dw[i][k] += p;
        s = fmaf(p, w[k], s);
      }
    }
    s = row_sum(s, s_part[buf], warp, wpr) / static_cast<float>(a.H);
    const long long t = t0 + mine;
    if (t < a.T) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int c = l + i * lanes;
        float fh[N], fy[N], w[N];
        Pack<T>::get(h[i], fh);
        Pack<T>::get(dy[i], fy);
        load_weight<W, N>(a.weight, min(c, chunks - 1), w);
#pragma unroll
        for (int k = 0; k < N; ++k) fy[k] = r * (fy[k] * w[k] - fh[k] * r * s);
        if (DH) {
          float g[N];
          Pack<T>::get(dh[i], g);
#pragma unroll
          for (int k = 0; k < N; ++k) fy[k] += g[k];
        }
        if (c < chunks) __stcs(reinterpret_cast<uint4*>(static_cast<T*>(a.dx) + t * a.H) + c, Pack<T>::put(fy));
      }
    }
  }
  // The rows of a block in order, then one partial sum a block.
  float* out = a.partials + static_cast<size_t>(blockIdx.x) * a.H;
  for (int m = 0; m < rows; ++m) {
    if (m > 0) __syncthreads();
    if (mine != m) continue;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = l + i * lanes;
      if (c >= chunks) continue;
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        float4 v = make_float4(dw[i][k], dw[i][k + 1], dw[i][k + 2], dw[i][k + 3]);
        float4* slot = reinterpret_cast<float4*>(s_dw + c * N + k);
        if (m > 0) { const float4 p = *slot; v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w; }
        if (m + 1 < rows) *slot = v;
        else *reinterpret_cast<float4*>(out + c * N + k) = v;
      }
    }
  }
}

// ---- rows staged in shared memory -------------------------------------------------------------------------------
// Rows that do not start at 16-byte words or end inside one, and in the backward pass rows too long for the registers of a block (three inputs, the
// next row's and the weight's gradient). A block keeps some rows ahead on their way to shared memory (cp.async: no registers), as the 16-byte words that
// hold them; a thread has the same columns of every row, with their weights and sums in registers. VEC: rows are whole aligned words, a column group is
// one of them; else it is one element, 32 a thread: many small blocks hide a row's way through two barriers better than few large ones (8 elements a
// thread: 16384 x 4097 360 us). us forward + backward in bf16, element by element straight from memory -> this: 16384 x 4097 468 -> 295,
// 32768 x 1001 268 -> 139, 4000 x 16383 882 -> 296; forward alone 190 -> 125, 112 -> 57, 216 -> 122.
constexpr int kStagedSmem = 216 * 1024, kElements = 32;
constexpr int staged_threads(bool vec) { return vec ? 1024 : 512; }   // at most

__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int bytes) {   // 16 bytes, those past the first `bytes` as zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait(int left) {   // until at most `left` groups are under way
  if (left <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
}
// All threads: the words that hold `n` elements from `row` on. What a word holds in front of the row or behind it is never used.
template <class T>
__device__ __forceinline__ void stage_row(unsigned char* to, const T* row, int n) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(15), end = reinterpret_cast<uintptr_t>(row + n);
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  for (int i = threadIdx.x; first + 16ull * i < end; i += blockDim.x) {
    const uintptr_t src = first + 16ull * i;
    copy_async(at + 16u * i, reinterpret_cast<const void*>(src), static_cast<int>(min(static_cast<unsigned long long>(end - src), 16ull)));
  }
}
template <class T>
__device__ __forceinline__ const T* staged(const unsigned char* stage, const T* row) {   // where the row starts in its stage
  return reinterpret_cast<const T*>(stage + (reinterpret_cast<uintptr_t>(row) & 15));
}
__host__ __device__ constexpr int staged_bytes(int H, int size) { return (H * size + 15) / 16 * 16 + 16; }   // a row, wherever in a word it starts

// IPT column groups a thread, `stages` (2 to 4) rows in shared memory.
template <class T, class W, int IPT, bool VEC, bool DH>
__global__ void __launch_bounds__(staged_threads(VEC)) row_norm_bwd_staged_kernel(const RowNormBwdArgs a, const int stages) {
  constexpr int N = VEC ? Pack<T>::N : 1, kInputs = DH ? 3 : 2;
  extern __shared__ __align__(16) unsigned char s_rows[];
  __shared__ float s_part[2][32];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, groups = a.H / N, row_bytes = staged_bytes(a.H, sizeof(T));
  grid_dependency_wait();
  launch_dependents();
  const T *h = static_cast<const T*>(a.h), *dy = static_cast<const T*>(a.dy), *dh = static_cast<const T*>(a.dh);
  const auto request = [&](long long t, int s) {
    if (t < a.T) {
      unsigned char* to = s_rows + static_cast<size_t>(s) * kInputs * row_bytes;
      stage_row(to, h + t * a.h_stride, a.H);
      stage_row(to + row_bytes, dy + t * a.H, a.H);
      if (DH) stage_row(to + 2 * row_bytes, dh + t * a.H, a.H);
    }
    copy_commit();
  };
  for (int s = 0; s + 1 < stages; ++s) request(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  float w[IPT][N], dw[IPT][N];
#pragma unroll
  for (int i = 0; i < IPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if constexpr (VEC) load_weight<W, N>(a.weight, min(c, groups - 1), w[i]);
    else w[i][0] = as_float<W>(static_cast<const W*>(a.weight)[min(c, groups - 1)]);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = 0.0f;
  }
  float next_r = blockIdx.x < a.T ? __ldg(a.rstd + blockIdx.x) : 0.0f;
  int s = 0, buf = 0;
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x, buf ^= 1) {
    copy_wait(stages - 2);
    __syncthreads();   // this row is here, and the row before it has been read by all
    request(t + static_cast<long long>(stages - 1) * gridDim.x, s == 0 ? stages - 1 : s - 1);
    const unsigned char* at = s_rows + static_cast<size_t>(s) * kInputs * row_bytes;
    const T *sh = staged(at, h + t * a.h_stride), *sy = staged(at + row_bytes, dy + t * a.H), *sd = DH ? staged(at + 2 * row_bytes, dh + t * a.H) : nullptr;
    const auto get = [&](const T* row, int c, float (&f)[N]) {
      if constexpr (VEC) Pack<T>::get(reinterpret_cast<const uint4*>(row)[c], f);
      else f[0] = as_float<T>(row[c]);
    };
    const float r = next_r;
    if (t + gridDim.x < a.T) next_r = __ldg(a.rstd + t + gridDim.x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= groups) break;
      float fh[N], fy[N];
      get(sh, c, fh);
      get(sy, c, fy);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float p = fy[k] * (fh[k] * r);
        dw[i][k] += p;
        sum = fmaf(p, w[i][k], sum);
      }
    }
    const float mean = row_sum(sum, s_part[buf], warp, warps) / static_cast<float>(a.H);
    T* dx = static_cast<T*>(a.dx) + t * a.H;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= groups) break;
      float fh[N], fy[N], fd[N];
      get(sh, c, fh);
      get(sy, c, fy);
      if (DH) get(sd, c, fd);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        fy[k] = r * (fy[k] * w[i][k] - fh[k] * r * mean);
        if (DH) fy[k] += fd[k];
      }
      if constexpr (VEC) __stcs(reinterpret_cast<uint4*>(dx) + c, Pack<T>::put(fy));
      else dx[c] = as_type<T>(fy[0]);
    }
    if (++s == stages) s = 0;
  }
  float* out = a.partials + static_cast<size_t>(blockIdx.x) * a.H;
#pragma unroll
  for (int i = 0; i < IPT; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c >= groups) break;
#pragma unroll
    for (int k = 0; k < N; ++k) out[c * N + k] = dw[i][k];
  }
}

// Forward of rows that are not whole aligned words: an element a column group.
template <class T, class W, bool RES>
__global__ void __launch_bounds__(staged_threads(false)) row_norm_staged_kernel(const RowNormArgs a, const int stages) {
  constexpr int kInputs = RES ? 2 : 1, IPT = kElements;
  extern __shared__ __align__(16) unsigned char s_rows[];
  __shared__ float s_part[2][32];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, row_bytes = staged_bytes(a.H, sizeof(T));
  grid_dependency_wait();
  launch_dependents();
  const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
  const auto request = [&](long long t, int s) {
    if (t < a.T) {
      unsigned char* to = s_rows + static_cast<size_t>(s) * kInputs * row_bytes;
      stage_row(to, x + t * a.x_stride, a.H);
      if (RES) stage_row(to + row_bytes, res + t * a.residual_stride, a.H);
    }
    copy_commit();
  };
  for (int s = 0; s + 1 < stages; ++s) request(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  float w[IPT];
#pragma unroll
  for (int i = 0; i < IPT; ++i) w[i] = as_float<W>(static_cast<const W*>(a.weight)[min(static_cast<int>(threadIdx.x + i * blockDim.x), a.H - 1)]);
  int s = 0, buf = 0;
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x, buf ^= 1) {
    copy_wait(stages - 2);
    __syncthreads();
    request(t + static_cast<long long>(stages - 1) * gridDim.x, s == 0 ? stages - 1 : s - 1);
    const unsigned char* at = s_rows + static_cast<size_t>(s) * kInputs * row_bytes;
    const T *sx = staged(at, x + t * a.x_stride), *sr = RES ? staged(at + row_bytes, res + t * a.residual_stride) : nullptr;
    float f[IPT], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      f[i] = 0.0f;
      if (c >= a.H) break;
      f[i] = as_float<T>(sx[c]);
      if (RES) {
        const T v = as_type<T>(f[i] + as_float<T>(sr[c]));
        static_cast<T*>(a.h)[t * a.H + c] = v;
        f[i] = as_float<T>(v);
      }
      ss = fmaf(f[i], f[i], ss);
    }
    const float r = rsqrtf(row_sum(ss, s_part[buf], warp, warps) / static_cast<float>(a.H) + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[t] = r;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c >= a.H) break;
      static_cast<T*>(a.y)[t * a.H + c] = as_type<T>(f[i] * r * w[i]);
    }
    if (++s == stages) s = 0;
  }
}

template <class T, class W, bool DH>
__global__ void __launch_bounds__(256) row_norm_bwd_any_kernel(const RowNormBwdArgs a) {
  extern __shared__ float s_dw[];            // [H], a column always by the same thread
  __shared__ float s_part[2][32];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  grid_dependency_wait();
  launch_dependents();
  for (int c = threadIdx.x; c < a.H; c += blockDim.x) s_dw[c] = 0.0f;
  int buf = 0;
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x, buf ^= 1) {
    const T* h = static_cast<const T*>(a.h) + t * a.h_stride;
    const T* dy = static_cast<const T*>(a.dy) + t * a.H;
    const T* dh = static_cast<const T*>(a.dh) + t * a.H;
    T* dx = static_cast<T*>(a.dx) + t * a.H;
    const W* w = static_cast<const W*>(a.weight);
    const float r = __ldg(a.rstd + t);
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      const float p = as_float<T>(dy[c]) * (as_float<T>(h[c]) * r);
      s_dw[c] += p;
      s = fmaf(p, as_float<W>(w[c]), s);
    }
    s = row_sum(s, s_part[buf], warp, warps) / static_cast<float>(a.H);
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      float v = r * (as_float<T>(dy[c]) * as_float<W>(w[c]) - as_float<T>(h[c]) * r * s);
      if (DH) v += as_float<T>(dh[c]);
      dx[c] = as_type<T>(v);
    }
  }
  for (int c = threadIdx.x; c < a.H; c += blockDim.x) a.partials[static_cast<size_t>(blockIdx.x) * a.H + c] = s_dw[c];
}

// The blocks' partial sums, added in a fixed order: 32 columns a block, a warp every 32nd partial.
template <class W>
__global__ void __launch_bounds__(1024) fold_columns_kernel(const float* __restrict__ partials, int blocks, int H, W* __restrict__ out) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  grid_dependency_wait();
  launch_dependents();
  float v = 0.0f;
  if (c < H)
    for (int b = y; b < blocks; b += 32) v += __ldcs(partials + static_cast<size_t>(b) * H + c);
  s[y][x] = v;
  __syncthreads();
  v = warp_sum(s[x][y]);   // column y of the 32
  if (x == 0 && blockIdx.x * 32 + y < H) out[blockIdx.x * 32 + y] = as_type<W>(v);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How a row is spread: C chunks of 16 bytes a lane, warps a row, rows a block; C = 0: in no such way.
struct Spread { int C, wpr, rows; };
Spread spread(int H, bool rows_bf16, bool vector, int most_c, int most_warps) {
  const int n = rows_bf16 ? 8 : 4, chunks = H / n;
  if (!vector || chunks == 0) return {0, 8, 1};
  for (int c = 1; c <= most_c; c *= 2) {
    const int wpr = (chunks + 32 * c - 1) / (32 * c);
    if (wpr <= 8 || (wpr <= most_warps && 2 * c > most_c)) return {c, wpr, std::max(1, 8 / wpr)};
  }
  return {0, 8, 1};
}
// How rows are staged: column groups a thread, threads, rows in shared memory, blocks an SM; stages = 0: they do not fit.
struct Stages { int ipt, threads, stages, per_sm; size_t smem; };
Stages staging(int H, int size, bool vector, int inputs) {
  const int n = vector ? 16 / size : 1, groups = H / n, most = staged_threads(vector);
  Stages g{vector ? size : kElements, 0, 0, 0, 0};   // vector: 16 columns a thread, or 32
  if (vector && groups > g.ipt * most) g.ipt *= 2;
  if (groups > g.ipt * most) return g;
  g.threads = std::max(32, ((groups + g.ipt - 1) / g.ipt + 31) / 32 * 32);
  const int row = inputs * staged_bytes(H, size);
  // as many blocks as registers allow (at most 64 a thread, or 128), and at least two rows in each
  for (g.per_sm = std::max(1, std::min(16, most / g.threads)); g.per_sm > 0; --g.per_sm) {
    g.stages = std::min(4, kStagedSmem / g.per_sm / row);
    if (g.stages >= 2) { g.smem = static_cast<size_t>(g.stages) * row; return g; }
  }
  g.stages = 0;
  return g;
}

template <class F>
auto with_types(bool rows_bf16, bool weight_bf16, F f) {
  if (rows_bf16) return weight_bf16 ? f(bf16{}, bf16{}) : f(bf16{}, float{});
  return weight_bf16 ? f(float{}, bf16{}) : f(float{}, float{});
}

}  // namespace

cudaError_t launch_row_norm(const RowNormArgs& args, int sms, cudaStream_t stream) {
  RowNormArgs a = args;
  if (a.T < 0 || a.H < 1 || a.H > kRowNormMaxHidden || (a.q != nullptr && (a.H % 128 || a.scales == nullptr))) return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  const int n = a.rows_bf16 ? 8 : 4;
  const bool vector = a.H % n == 0 && aligned16(a.x) && a.x_stride % n == 0 && aligned16(a.residual) && a.residual_stride % n == 0 && aligned16(a.weight);
  const Spread sp = spread(a.H, a.rows_bf16 != 0, vector, 8, 16);
  a.warps_per_row = sp.wpr;
  const int block = 32 * sp.wpr * sp.rows, grid = (a.T + sp.rows - 1) / sp.rows;
  const Stages st = sp.C == 0 && a.q == nullptr ? staging(a.H, a.rows_bf16 ? 2 : 4, false, a.residual ? 2 : 1) : Stages{};
  const cudaError_t e = with_types(a.rows_bf16 != 0, a.weight_bf16 != 0, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const auto go = [&](auto res, auto quant) {
      constexpr bool RES = decltype(res)::value, QUANT = decltype(quant)::value;
      if constexpr (!QUANT) {
        if (st.stages > 0) {
          const auto with = [&](auto kern) {
            const cudaError_t err = allow_smem(kern, st.smem);
            return err != cudaSuccess ? err : launch_early(kern, dim3(std::min(a.T, sms * st.per_sm)), st.threads, st.smem, stream, a, st.stages);
          };
          return with(row_norm_staged_kernel<T, W, RES>);
        }
      }
      switch (sp.C) {
        case 1: return launch_early(row_norm_kernel<T, W, 1, RES, QUANT>, dim3(grid), block, 0, stream, a);
        case 2: return launch_early(row_norm_kernel<T, W, 2, RES, QUANT>, dim3(grid), block, 0, stream, a);
        case 4: return launch_early(row_norm_kernel<T, W, 4, RES, QUANT>, dim3(grid), block, 0, stream, a);
        case 8: return launch_early(row_norm_kernel<T, W, 8, RES, QUANT>, dim3(grid), block, 0, stream, a);
        default: return launch_early(row_norm_any_kernel<T, W, RES, QUANT>, dim3(a.T), 256, 0, stream, a);
      }
    };
    if (a.residual != nullptr) return a.q ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
    return a.q ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
  });
  note_launch();
  return e;
}

namespace {
struct BwdPlan { Spread sp; Stages st; bool vector; };
BwdPlan bwd_plan(const RowNormBwdArgs& a) {
  const int n = a.rows_bf16 ? 8 : 4;
  const bool vector = a.H % n == 0 && aligned16(a.h) && a.h_stride % n == 0 && aligned16(a.dy) && aligned16(a.dh) && aligned16(a.weight);
  const Spread sp = spread(a.H, a.rows_bf16 != 0, vector, a.rows_bf16 ? 2 : 4, kBwdWarps);   // 16 columns a lane
  return {sp, sp.C == 0 ? staging(a.H, a.rows_bf16 ? 2 : 4, vector, a.dh ? 3 : 2) : Stages{}, vector};
}
}  // namespace

int row_norm_bwd_blocks(const RowNormBwdArgs& a, int sms) {
  const BwdPlan p = bwd_plan(a);
  // What an SM holds at once; element by element, what the sums in shared memory leave.
  const int rows = p.sp.C > 0 ? p.sp.rows : 1, per_sm = p.sp.C > 0 ? std::max(1, (p.sp.C * (a.rows_bf16 ? 8 : 4) <= 8 ? 32 : 16) / (p.sp.wpr * rows)) : p.st.stages > 0 ? p.st.per_sm : std::max(1, std::min(8, 200 * 1024 / (4 * a.H)));
  const int least = a.T <= 8 * sms ? 2 : 4;   // rows for every partial sum
  return std::max(1, std::min(sms * per_sm, (a.T + least * rows - 1) / (least * rows)));
}

cudaError_t launch_row_norm_bwd(const RowNormBwdArgs& args, int blocks, cudaStream_t stream) {
  RowNormBwdArgs a = args;
  if (a.T < 1 || a.H < 1 || a.H > kRowNormMaxHidden || blocks < 1 || a.partials == nullptr) return cudaErrorInvalidValue;
  const BwdPlan plan = bwd_plan(a);
  const Spread sp = plan.sp;
  const Stages st = plan.st;
  a.warps_per_row = sp.wpr;
  cudaError_t e = with_types(a.rows_bf16 != 0, a.weight_bf16 != 0, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const auto go = [&](auto dh) {
      constexpr bool DH = decltype(dh)::value;
      const int block = 32 * sp.wpr * sp.rows;
      if (st.stages > 0) {
        const auto with = [&](auto kern) {
          const cudaError_t err = allow_smem(kern, st.smem);
          return err != cudaSuccess ? err : launch_early(kern, dim3(blocks), st.threads, st.smem, stream, a, st.stages);
        };
        if (!plan.vector) return with(row_norm_bwd_staged_kernel<T, W, kElements, false, DH>);
        constexpr int kWords = sizeof(T);   // 16 columns
        return st.ipt == kWords ? with(row_norm_bwd_staged_kernel<T, W, kWords, true, DH>) : with(row_norm_bwd_staged_kernel<T, W, 2 * kWords, true, DH>);
      }
      const size_t smem = sp.C == 0 || sp.rows > 1 ? sizeof(float) * a.H : 0;
      const auto with = [&](auto kern, int threads) {
        const cudaError_t err = allow_smem(kern, smem);
        return err != cudaSuccess ? err : launch_early(kern, dim3(blocks), threads, smem, stream, a);
      };
      switch (sp.C) {
        case 1: return with(row_norm_bwd_kernel<T, W, 1, DH>, block);
        case 2: return with(row_norm_bwd_kernel<T, W, 2, DH>, block);
        case 4:
          if constexpr (sizeof(T) == 4) return with(row_norm_bwd_kernel<T, W, 4, DH>, block);
          else return cudaErrorInvalidValue;
        default: return with(row_norm_bwd_any_kernel<T, W, DH>, 256);
      }
    };
    return a.dh != nullptr ? go(std::true_type()) : go(std::false_type());
  });
  if (e != cudaSuccess) return e;
  note_launch();
  return launch_fold_columns(a.partials, blocks, a.H, a.weight_bf16 != 0, a.dweight, stream);
}

cudaError_t launch_fold_columns(const float* partials, int blocks, int n, bool as_bf16, void* out, cudaStream_t stream) {
  const dim3 grid((n + 31) / 32);
  const cudaError_t e = as_bf16 ? launch_early(fold_columns_kernel<bf16>, grid, 1024, 0, stream, partials, blocks, n, static_cast<bf16*>(out))
                                : launch_early(fold_columns_kernel<float>, grid, 1024, 0, stream, partials, blocks, n, static_cast<float*>(out));
  note_launch();
  return e;
}

}  // namespace fastb
