// Backward of a linear layer's epilogue: out = act(z) + residual, z = x W^T + bias.
//
//   dz = dy act'(z), rounded to bf16 for the two products that take it;  dbias = sum over rows of dz, from the values before that rounding
//
// One pass: 8 columns a thread, rows in turn, column sums in registers and one partial sum a block of rows, added up in a fixed order.
// What bounds it: HBM, 6 bytes an element (2 where there is no activation: then dz is dy, and only the bias wants its sums).
#include <algorithm>

#include "early_start.cuh"
#include "gemm_common.cuh"

namespace fastb {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

// act'(z); that of NaN is NaN
template <Activation ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == Activation::kRelu) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
  if (ACT == Activation::kSilu) {
    const float s = gemm::sigmoid(z);
    return s * (1.0f + z * (1.0f - s));
  }
  if (ACT == Activation::kGelu) return gemm::gelu_slope(z);
  return 1.0f;
}
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = __bfloat1622float2(h[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
}

// blockIdx.x: 256 columns; blockIdx.y: every gridDim.y-th group of eight rows, a row a warp.
template <Activation ACT>
__global__ void __launch_bounds__(kThreads) linear_dz_kernel(const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ z, __nv_bfloat16* __restrict__ dz, float* __restrict__ partials, int T,
                                                             int N) {
  constexpr int U = 4;   // rows in flight
  __shared__ float s_sum[kWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, chunks = N / 8;
  grid_dependency_wait();
  launch_dependents();
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
  const int step = gridDim.y * kWarps;
  for (long long t0 = blockIdx.y * kWarps + warp; t0 < T; t0 += static_cast<long long>(U) * step) {
    uint4 g[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long t = t0 + static_cast<long long>(u) * step;
      const bool in = t < T && c < chunks;
      g[u] = in ? __ldg(reinterpret_cast<const uint4*>(dy) + t * chunks + c) : make_uint4(0, 0, 0, 0);
      if (ACT != Activation::kNone) v[u] = in ? __ldcs(reinterpret_cast<const uint4*>(z) + t * chunks + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long t = t0 + static_cast<long long>(u) * step;
      float d[8];
      unpack8(g[u], d);
      if (ACT != Activation::kNone) {
        float f[8];
        unpack8(v[u], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] *= slope<ACT>(f[k]);
        if (t < T && c < chunks)
          reinterpret_cast<uint4*>(dz)[t * chunks + c] = make_uint4(gemm::pack_bf16(d[0], d[1]), gemm::pack_bf16(d[2], d[3]), gemm::pack_bf16(d[4], d[5]), gemm::pack_bf16(d[6], d[7]));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] += d[k];
    }
  }
  if (partials == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) s_sum[warp][k * 32 + lane] = acc[k];
  __syncthreads();
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) v += s_sum[w][threadIdx.x];
  const int column = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8 + (threadIdx.x >> 5);
  if (column < N) partials[static_cast<size_t>(blockIdx.y) * N + column] = v;
}

// SwiGLU: act = silu(g) u. g and u are read as 16 bits each and what their rounding took off: rounded alone they would add as much to the
// gradients' error as dz's own rounding does. HBM: 14 bytes an element of the output; 8 columns a thread, U of them in flight.
__global__ void __launch_bounds__(kThreads) linear_swiglu_dz_kernel(const __nv_bfloat16* __restrict__ dy, const __nv_bfloat16* __restrict__ pre, __nv_bfloat16* __restrict__ dz, int T, int inter) {
  constexpr int U = 2;
  const uint4 *d_at = reinterpret_cast<const uint4*>(dy), *z_at = reinterpret_cast<const uint4*>(pre);
  uint4* out = reinterpret_cast<uint4*>(dz);
  const int per_row = inter / 8;
  const long long total = static_cast<long long>(T) * per_row, step = static_cast<long long>(gridDim.x) * kThreads * U;
  grid_dependency_wait();
  launch_dependents();
  for (long long i0 = static_cast<long long>(blockIdx.x) * kThreads * U + threadIdx.x; i0 < total; i0 += step) {
    uint4 d[U], g[U], u[U], gl[U], ul[U];
    long long to[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const long long i = min(i0 + q * kThreads, total - 1), t = i / per_row;
      const int c = static_cast<int>(i - t * per_row), at = c / 16 * 32 + c % 16;
      to[q] = t * (2 * per_row) + at;
      const uint4* z = z_at + t * (4 * per_row) + at;
      d[q] = __ldg(d_at + i);
      g[q] = __ldcs(z); u[q] = __ldcs(z + 16);
      gl[q] = __ldcs(z + 2 * per_row); ul[q] = __ldcs(z + 2 * per_row + 16);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (i0 + q * kThreads >= total) break;
      float fd[8], fg[8], fu[8], rest[8];
      unpack8(d[q], fd);
      unpack8(g[q], fg);
      unpack8(gl[q], rest);
#pragma unroll
      for (int k = 0; k < 8; ++k) fg[k] += rest[k];
      unpack8(u[q], fu);
      unpack8(ul[q], rest);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float s = gemm::sigmoid(fg[k]), act = fg[k] * s;
        fg[k] = fd[k] * (fu[k] + rest[k]) * (s + act * (1.0f - s));
        fu[k] = fd[k] * act;
      }
      out[to[q]] = make_uint4(gemm::pack_bf16(fg[0], fg[1]), gemm::pack_bf16(fg[2], fg[3]), gemm::pack_bf16(fg[4], fg[5]), gemm::pack_bf16(fg[6], fg[7]));
      out[to[q] + 16] = make_uint4(gemm::pack_bf16(fu[0], fu[1]), gemm::pack_bf16(fu[2], fu[3]), gemm::pack_bf16(fu[4], fu[5]), gemm::pack_bf16(fu[6], fu[7]));
    }
  }
}

// A weight gradient whose rows were shared out: a warp has 32 rows of a half tile and 16 of its columns, a lane a row.
__global__ void __launch_bounds__(kThreads) fold_slices_kernel(const float* __restrict__ sums, int slices, int m_tiles, int n_tiles, __nv_bfloat16* __restrict__ out, int rows, int cols) {
  const int lane = threadIdx.x & 31, unit = blockIdx.x * kWarps + (threadIdx.x >> 5), tiles = m_tiles * n_tiles;
  const int c16 = unit % 16, part = unit / 16 % 4, half = unit / 64 % 2, tile = unit / 128;
  grid_dependency_wait();
  launch_dependents();
  if (tile >= tiles) return;
  const int row = tile / n_tiles * 256 + half * 128 + part * 32 + lane;
  const long long col = static_cast<long long>(tile % n_tiles) * 256 + c16 * 16;
  if (row >= rows || col >= cols) return;
  const float4* at = reinterpret_cast<const float4*>(sums) + (static_cast<long long>(tile * 2 + half) * 64 + c16 * 4) * 128 + part * 32 + lane;
  float4 v[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = __ldcg(at + q * 128);
#pragma unroll 2
  for (int s = 1; s < slices; ++s) {
    const float4* next = at + static_cast<long long>(s) * tiles * (2 * 64 * 128);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 x = __ldcg(next + q * 128);
      v[q].x += x.x; v[q].y += x.y; v[q].z += x.z; v[q].w += x.w;
    }
  }
  uint4* to = reinterpret_cast<uint4*>(out + static_cast<long long>(row) * cols + col);
  to[0] = make_uint4(gemm::pack_bf16(v[0].x, v[0].y), gemm::pack_bf16(v[0].z, v[0].w), gemm::pack_bf16(v[1].x, v[1].y), gemm::pack_bf16(v[1].z, v[1].w));
  if (col + 8 < cols) to[1] = make_uint4(gemm::pack_bf16(v[2].x, v[2].y), gemm::pack_bf16(v[2].z, v[2].w), gemm::pack_bf16(v[3].x, v[3].y), gemm::pack_bf16(v[3].z, v[3].w));
}

}  // namespace

cudaError_t launch_linear_swiglu_dz(const __nv_bfloat16* dy, const __nv_bfloat16* pre, __nv_bfloat16* dz, int T, int inter, cudaStream_t stream) {
  if (T < 1 || inter < 128 || inter % 128) return cudaErrorInvalidValue;
  const long long blocks = (static_cast<long long>(T) * (inter / 8) + 2 * kThreads - 1) / (2 * kThreads);
  const cudaError_t e = launch_early(linear_swiglu_dz_kernel, dim3(static_cast<unsigned>(std::min(blocks, 8192ll))), kThreads, 0, stream, dy, pre, dz, T, inter);
  note_launch();
  return e;
}

cudaError_t launch_fold_slices(const float* sums, int slices, int m_tiles, int n_tiles, __nv_bfloat16* out, int rows, int cols, cudaStream_t stream) {
  if (slices < 1 || m_tiles < 1 || n_tiles < 1 || rows < 1 || rows > 256 * m_tiles || cols < 8 || cols % 8 || cols > 256 * n_tiles || static_cast<long long>(m_tiles) * n_tiles > 1 << 20) return cudaErrorInvalidValue;
  const cudaError_t e = launch_early(fold_slices_kernel, dim3(m_tiles * n_tiles * 128 / kWarps), kThreads, 0, stream, sums, slices, m_tiles, n_tiles, out, rows, cols);
  note_launch();
  return e;
}

int linear_dz_blocks(int T, int N, int sms) {
  const int columns = (N + 255) / 256;
  return std::max(1, std::min((T + 4 * kWarps - 1) / (4 * kWarps), (8 * sms + columns - 1) / columns));
}

cudaError_t launch_linear_dz(Activation act, const __nv_bfloat16* dy, const __nv_bfloat16* z, __nv_bfloat16* dz, float* partials, int T, int N, int blocks, __nv_bfloat16* dbias, cudaStream_t stream) {
  if (T < 1 || N < 8 || N % 8 || blocks < 1 || (partials == nullptr) != (dbias == nullptr) || (act != Activation::kNone && (z == nullptr || dz == nullptr))) return cudaErrorInvalidValue;
  const dim3 grid((N + 255) / 256, blocks);
  const auto go = [&](auto kern) { return launch_early(kern, grid, kThreads, 0, stream, dy, z, dz, partials, T, N); };
  const cudaError_t e = act == Activation::kRelu ? go(linear_dz_kernel<Activation::kRelu>) : act == Activation::kSilu ? go(linear_dz_kernel<Activation::kSilu>)
                        : act == Activation::kGelu ? go(linear_dz_kernel<Activation::kGelu>) : go(linear_dz_kernel<Activation::kNone>);
  note_launch();
  if (e != cudaSuccess || partials == nullptr) return e;
  return launch_fold_columns(partials, blocks, N, true, dbias, stream);
}

}  // namespace fastb
