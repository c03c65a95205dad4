// Projections over weights held in 4 bits with group scales, y = x W^T (M = 1..32) on 16x16x32 BF16 MFMAs: the launch
// rule and the weights' way back to BF16 (the kernel is ftk_w4_walk.h).
//
// W = s (q - z). A pair of codes becomes a pair of BF16 values in one instruction (two with the shift):
// 0x4300 | q is 128 + q exactly. So a group's sum is
//   sum (q - z) x = sum (128 + q) x - (128 + z) sum x,
// with sum x (per group and row of x) found once per workgroup; the second term is where the group's accumulators
// start, the matrix instructions add the first, and the group's sum is scaled in FP32.
// The two terms cancel to at most 5 bits of FP32's 24, far below the BF16 rounding of the output.
// Where x holds an infinity (or 128 x overflows) they meet as inf - inf: an output that is not finite is
// summed again, element by element (exact_sum).
//
// What bounds it (us per graph node, cold weights; in brackets a pure read of the same bytes in one launch): one row of
// the large matrices the weight read -- 24576 x 4096 + norm + SwiGLU 12.1 (9.5) or 4.3 TB/s, 4096 x 12288 7.6 (5.5); one
// row of the small ones the launch and the chain x, operand, first product, outputs -- 4096 x 1024 + norm 3.7 (2.2). From
// about 8 rows on it is the vector unit: x becomes the operand in every workgroup (some 65 instructions for 8 elements
// of a normalised row), and a tile's codes are unpacked once per row block (7 for 8 codes): 6144 x 4096 + norm at 16 rows
// 10.0 (3.5), 24576 x 4096 + norm + SwiGLU at 8 / 16 / 24 rows 14.4 / 19.0 / 26.5 (9.6). An operand formed by a launch of
// its own took that launch's 4 to 5 us again (16 rows of 6144 x 4096 13.3, 24 rows of 24576 x 4096 29.3).
#include "ftk_w4_walk.h"

namespace ftk {

// W itself, BF16 row-major (the native GEMM's operand past the rows these kernels take): one rounding of
// s (q - z). A thread takes the 32 columns of one lane of a chunk.
template <int S>
__global__ __launch_bounds__(256) void w4_dequantize_kernel(W4Args a, uint16_t* w) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.tiles * a.chunks * 64) return;
  const int lane = (int)(i & 63), li = lane & 15, g = lane >> 4;
  const int64_t block = i >> 6;
  const int c = (int)(block % a.chunks), tile = (int)(block / a.chunks);
  // A SwiGLU tile's rows: 8 gate rows, then the up rows beside them (a.N outputs: the up half begins at row a.N).
  const int n = a.swiglu ? tile * 8 + (li & 7) : tile * 16 + li;
  if (n >= a.N) return;
  const int64_t row = a.swiglu && li >= 8 ? (int64_t)a.N + n : n;
  const u32x4_t v = a.codes[i];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const size_t at = ((size_t)block * 16 + li) * S + s * S / 4;
    const float scale = w4::scale_f32(a.scales[at], a.half_scales), z = a.zeros != nullptr ? (float)a.zeros[at] : 8.f;
    const int k = c * kW4Chunk + 32 * s + 8 * g;
    const uint32_t d = v[s];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < a.K)
        w[row * a.K + k + e] = (uint16_t)f32_to_bf16(((float)((d >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - z) * scale);
  }
}

// Rows of x to a workgroup, chunks per wave and the grid.
W4Shape w4_shape(W4Args& a, int subs, int cus) {
  // The builds: what the registers of two waves on a SIMD hold (several groups to a chunk take more of them).
  static const int held[] = {1, 2, 3, 4, 6, 8};
  const int most_held = subs == 1 ? 8 : subs == 2 ? 6 : 4;
  const int need = (a.chunks + kW4Waves - 1) / kW4Waves, per = a.gain != nullptr ? 2 : 1;
  // The launch whose workgroups take `blocks` blocks of operand rows (with a gain a row has two), and the tiles that its
  // longest walk takes.
  auto shape = [&](int blocks, int& rounds) {
    W4Shape s;
    const int most = 16 * blocks / per;
    a.row_blocks = (a.M + most - 1) / most;
    a.rows = (a.M + a.row_blocks - 1) / a.row_blocks;
    a.row_blocks = (a.M + a.rows - 1) / a.rows;
    s.blocks = blocks;
    s.one = a.M == 1;
    s.passes = need > most_held ? kW4Passes : kW4Held;
    s.held = blocks == 2 ? 4 : s.one && subs < 4 ? 6 : 4;
    if (blocks == 1 && s.passes == kW4Held)
      for (const int* h = held; (s.held = *h) < need; ++h) {}
    // One workgroup to a CU (two where its waves hold few chunks), as many for each row block, by eights; all walks as
    // even as they come.
    const int all = cus * (w4_pairs(s.held, s.blocks, subs, s.passes, s.one) ? 2 : 1) / a.row_blocks / 8 * 8;
    const int slots = all > 0 ? all : 8;
    rounds = (a.tiles + slots - 1) / slots;
    // Four chunks to a wave and at most four tiles: 16 waves of two chunks each form x sooner and hide more. Longer walks
    // pay for the 16 partial sums of each output (8 waves, 16: 6144 x 4096 + norm at 8 rows 8.4 us, 7.8, at 16 rows 9.5,
    // 9.0; 4096 x 4096 at 8 rows 5.7, 5.0; 24576 x 4096 + norm at 8 rows 14.6, 15.3), and idle waves cost more than they
    // hide (9497 x 2570 at 5 rows, 21 chunks, 6.9, 7.5).
    s.waves = kW4Waves;
    if (blocks == 1 && !s.one && need == 4 && rounds <= 4) s.waves = 16, s.held = 2;
    // Passes of several rows and more than one tile: the tiles of a batch take each pass in turn, so that a pass's x
    // becomes the operand once a batch, not once a tile (a tile's passes in turn, batches: 16384 x 12288 at 32 rows 80 us,
    // 41; 4096 x 12288 + norm at 16 rows 25.3, 19.0; a single tile, 4096 x 12288 at 16 rows, 13.6, 14.7).
    if (s.passes == kW4Passes && !s.one && rounds > 1) s.passes = kW4Batches;
    const int walkers = (a.tiles + rounds - 1) / rounds;
    s.grid = (walkers + 7) / 8 * 8 * a.row_blocks;
    return s;
  };
  int rounds = 0, rounds2 = 0;
  const W4Shape s = shape(1, rounds);
  // More rows than a block holds go to several workgroups, which read the weights again from their XCD's L2. Two blocks
  // to a workgroup halve the walks, but form twice the operand ahead of them and take most of the registers; that pays
  // from about four tiles fewer on (norm, 16 rows, K = 4096: 24576 outputs 20.7 us by one block, 19.0 by two; 16384:
  // 15.0, 15.4; 6144: 9.5, 11.6), and only where two blocks leave a wave its 3 or 4 chunks.
  if (per * a.M > 16 && subs < 4 && (need == 3 || need == 4)) {
    const W4Shape s2 = shape(2, rounds2);
    if (rounds - rounds2 > 4) return s2;
    return shape(1, rounds);
  }
  return s;
}

hipError_t launch_w4(const W4Args& args, int subs, int cus, hipStream_t stream) {
  W4Args a = args;
  const W4Shape s = w4_shape(a, subs, cus);
  return subs == 1 ? launch_w4_s1(a, s, stream) : subs == 2 ? launch_w4_s2(a, s, stream) : launch_w4_s4(a, s, stream);
}

hipError_t launch_w4_dequantize(const W4Args& a, int subs, uint16_t* w, hipStream_t stream) {
  const int64_t threads = (int64_t)a.tiles * a.chunks * 64;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (subs == 1)
    hipLaunchKernelGGL(w4_dequantize_kernel<1>, grid, dim3(256), 0, stream, a, w);
  else if (subs == 2)
    hipLaunchKernelGGL(w4_dequantize_kernel<2>, grid, dim3(256), 0, stream, a, w);
  else
    hipLaunchKernelGGL(w4_dequantize_kernel<4>, grid, dim3(256), 0, stream, a, w);
  return hipGetLastError();
}

}  // namespace ftk
