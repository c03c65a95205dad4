// Projections over weights held in 4 bits with group scales, y = x W^T (M = 1..32) on 16x16x32 BF16 MFMAs.
//
// W = s (q - z). A pair of codes becomes a pair of BF16 values in one instruction (two with the shift):
// 0x4300 | q is 128 + q exactly. So a group's sum is
//   sum (q - z) x = sum (128 + q) x - (128 + z) sum x,
// both terms on the matrix cores, in one FP32 accumulator: the second is an MFMA whose weight operand is
// the constant -(128 + z) (exact in BF16) in every column. The group's sum is then scaled in FP32.
// The two terms cancel to at most 5 bits of FP32's 24, far below the BF16 rounding of the output.
// Where x holds an infinity (or 128 x overflows) they meet as inf - inf: an output that is not finite is
// summed again, element by element (w4_exact).
#include "ftk_w4.h"

namespace ftk {

namespace {

__device__ __forceinline__ float w4_scale(uint32_t bits, bool half) {
  return half ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : bf16_to_f32(bits);
}

// Columns 32 s + 8 g .. + 7 of chunk c of an x row, zero past the row's end.
__device__ __forceinline__ u32x4_t x_tail(const uint16_t* row, int k, int K) {
  if (k + 8 <= K) return load16_any(row + k);
  uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) o[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
  return u32x4_t{o[0], o[1], o[2], o[3]};
}

// The operand of one step: 128 + q for the 8 codes of a dword.
__device__ __forceinline__ u32x4_t w4_operand(uint32_t v) {
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ((v >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  return o;
}

__device__ __forceinline__ uint32_t w4_code(const W4Args& a, int tile, int li, int k) {
  const int c = k / kW4Chunk, r = k % kW4Chunk, s = r / 32, g = (r % 32) / 8, e = r % 8;
  const uint32_t* d = reinterpret_cast<const uint32_t*>(a.codes + ((size_t)tile * a.chunks + c) * 64 + 16 * g + li);
  return (d[s] >> (4 * (e / 2) + 16 * (e % 2))) & 15u;
}

// One output summed element by element, each product (q - z) s x: what the definition says for an x that holds
// infinities or values whose 128-fold is one.
template <int S>
__device__ __noinline__ float w4_exact(const W4Args& a, int tile, int li, int m) {
  float sum = 0.f;
  for (int k = 0; k < a.K; ++k) {
    const size_t at = (((size_t)tile * a.chunks + k / kW4Chunk) * 16 + li) * S + (k % kW4Chunk) * S / kW4Chunk;
    const float z = a.zeros != nullptr ? (float)a.zeros[at] : 8.f;
    const float w = ((float)w4_code(a, tile, li, k) - z) * w4_scale(a.scales[at], a.half_scales);
    sum += w * bf16_to_f32(a.x[(size_t)m * a.x_stride + k]);
  }
  return sum;
}

__device__ __forceinline__ bool finite_f32(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

}  // namespace

// T tiles of 16 weight rows to a workgroup, its W waves splitting the chunks of K; CB blocks of 16 x rows.
// x is the A operand and the weights the B operand, so a lane's accumulators belong to one weight row and
// one scale serves them all.
template <int T, int W, int CB, int S, bool ZP, bool SWIGLU>
__global__ __launch_bounds__(64 * W) void w4_kernel(W4Args a) {
  __shared__ float red[W][T][16 * CB][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int tile0 = blockIdx.x * T;

  const uint16_t* xrow[CB];
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const int m = 16 * b + li;
    xrow[b] = a.x + (size_t)(m < a.M ? m : a.M - 1) * a.x_stride;
  }
  f32x4_t acc[T][CB] = {};
  for (int c = wave; c < a.chunks; c += W) {
    u32x4_t w[T], x[CB][4];
    uint32_t sc[T][S], zp[T][S];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int tile = tile0 + t < a.tiles ? tile0 + t : a.tiles - 1;
      const size_t at = (size_t)tile * a.chunks + c;
      w[t] = load_stream16(a.codes + at * 64 + lane);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        sc[t][s] = a.scales[(at * 16 + li) * S + s];
        zp[t][s] = ZP ? a.zeros[(at * 16 + li) * S + s] : 8u;
      }
    }
    const int k0 = c * kW4Chunk + 8 * g;
    if ((c + 1) * kW4Chunk <= a.K) {
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) x[b][s] = load16_any(xrow[b] + k0 + 32 * s);
    } else {
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) x[b][s] = x_tail(xrow[b], k0 + 32 * s, a.K);
    }
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const uint32_t zw = (0xC300u | zp[t][s]) * 0x10001u;
          const u32x4_t zo = {zw, zw, zw, zw};
          f32x4_t part = {};
#pragma unroll
          for (int i = 4 / S * s; i < 4 / S * (s + 1); ++i) {
            part = mfma16x16x32(x[b][i], zo, part);
            const uint32_t wv = w[t][i];
            part = mfma16x16x32(x[b][i], w4_operand(wv), part);
          }
          acc[t][b] += part * w4_scale(sc[t][s], a.half_scales);
        }
  }
  // Element r of acc[t][b]: x row 16 b + 4 g + r, weight row li of tile t.
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int b = 0; b < CB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][t][16 * b + 4 * g + r][li] = acc[t][b][r];
  __syncthreads();
  constexpr int COLS = SWIGLU ? 8 : 16;  // outputs of a tile
  for (int i = threadIdx.x; i < T * a.M * COLS; i += 64 * W) {
    const int col = i % COLS, m = i / COLS % a.M, t = i / COLS / a.M;
    const int tile = tile0 + t;
    const int n = tile * COLS + col;
    if (n >= a.N) continue;
    float v = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      v += red[w][t][m][col];
      if constexpr (SWIGLU) u += red[w][t][m][col + 8];
    }
    if (!finite_f32(v)) v = w4_exact<S>(a, tile, col, m);
    if constexpr (SWIGLU) {
      if (!finite_f32(u)) u = w4_exact<S>(a, tile, col + 8, m);
      v = silu_f32(v) * u;
    }
    if (a.add != nullptr) v += bf16_to_f32(a.add[(size_t)m * a.N + n]);
    a.y[(size_t)m * a.N + n] = (uint16_t)f32_to_bf16(v);
  }
}

// W itself, BF16 row-major (the native GEMM's operand past the rows these kernels take): one rounding of
// s (q - z). A thread takes the 32 columns of one lane of a chunk.
template <int S>
__global__ __launch_bounds__(256) void w4_dequantize_kernel(W4Args a, int swiglu, uint16_t* w) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.tiles * a.chunks * 64) return;
  const int lane = (int)(i & 63), li = lane & 15, g = lane >> 4;
  const int64_t block = i >> 6;
  const int c = (int)(block % a.chunks), tile = (int)(block / a.chunks);
  // A SwiGLU tile's rows: 8 gate rows, then the up rows beside them (a.N outputs: the up half begins at row a.N).
  const int n = swiglu ? tile * 8 + (li & 7) : tile * 16 + li;
  if (n >= a.N) return;
  const int64_t row = swiglu && li >= 8 ? (int64_t)a.N + n : n;
  const u32x4_t v = a.codes[i];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const size_t at = ((size_t)block * 16 + li) * S + s * S / 4;
    const float scale = w4_scale(a.scales[at], a.half_scales), z = a.zeros != nullptr ? (float)a.zeros[at] : 8.f;
    const int k = c * kW4Chunk + 32 * s + 8 * g;
    const uint32_t d = v[s];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < a.K)
        w[row * a.K + k + e] = (uint16_t)f32_to_bf16(((float)((d >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - z) * scale);
  }
}

namespace {

template <int S, bool ZP, bool SWIGLU>
void launch_rows(const W4Args& a, hipStream_t stream) {
  constexpr int T = 1, W = 8;
  const dim3 grid((unsigned)((a.tiles + T - 1) / T));
  if (a.M <= 16)
    hipLaunchKernelGGL((w4_kernel<T, W, 1, S, ZP, SWIGLU>), grid, dim3(64 * W), 0, stream, a);
  else
    hipLaunchKernelGGL((w4_kernel<T, W, 2, S, ZP, SWIGLU>), grid, dim3(64 * W), 0, stream, a);
}

template <int S>
void launch_groups(const W4Args& a, bool swiglu, hipStream_t stream) {
  if (a.zeros != nullptr)
    swiglu ? launch_rows<S, true, true>(a, stream) : launch_rows<S, true, false>(a, stream);
  else
    swiglu ? launch_rows<S, false, true>(a, stream) : launch_rows<S, false, false>(a, stream);
}

}  // namespace

hipError_t launch_w4(const W4Args& a, int subs, bool swiglu, hipStream_t stream) {
  if (subs == 1)
    launch_groups<1>(a, swiglu, stream);
  else if (subs == 2)
    launch_groups<2>(a, swiglu, stream);
  else
    launch_groups<4>(a, swiglu, stream);
  return hipGetLastError();
}

hipError_t launch_w4_dequantize(const W4Args& a, int subs, bool swiglu, uint16_t* w, hipStream_t stream) {
  const int64_t threads = (int64_t)a.tiles * a.chunks * 64;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (subs == 1)
    hipLaunchKernelGGL(w4_dequantize_kernel<1>, grid, dim3(256), 0, stream, a, (int)swiglu, w);
  else if (subs == 2)
    hipLaunchKernelGGL(w4_dequantize_kernel<2>, grid, dim3(256), 0, stream, a, (int)swiglu, w);
  else
    hipLaunchKernelGGL(w4_dequantize_kernel<4>, grid, dim3(256), 0, stream, a, (int)swiglu, w);
  return hipGetLastError();
}

}  // namespace ftk
