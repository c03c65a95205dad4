// Arguments of the projections whose weights are held in 4 bits with group scales (ftk_w4.hip).
#pragma once

#include "ftk_internal.h"

namespace ftk {

// W[n, k] = s[n, k / g] (q[n, k] - z[n, k / g]), laid out in tiles of 16 weight rows and chunks of 128
// columns. A chunk of a tile is 1 KiB: lane (li, g) = (lane % 16, lane / 16) of a wave has row li's columns
// 32 s + 8 g + e (e = 0..7) in dword s, column e at bit 4 (e / 2) + 16 (e % 2).
struct W4Args {
  const uint16_t* x;       // [M, K] BF16, rows x_stride elements apart, any 2-byte alignment
  int64_t x_stride;
  const uint16_t* gain;    // [K]: x is RMS-normalised first; or null
  float eps;
  const u32x4_t* codes;    // [tiles][chunks][64]
  const uint16_t* scales;  // [tiles][chunks][16][S], S = groups per chunk (1, 2, 4)
  const uint8_t* zeros;    // the same layout, or null: 8 everywhere
  const uint16_t* add;     // [M, outputs] joining the outputs, or null
  uint16_t* y;             // [M, outputs] BF16
  int M, N, K;             // N: outputs of the epilogue (columns of y)
  int tiles, chunks;
  int half_scales;         // scales are FP16 (else BF16)
  int swiglu;              // tiles of 8 gate and 8 up rows; y = silu(gate) up
  int rows;                // rows of x to a workgroup (the launch's row blocks: ceil(M / rows))
  int row_blocks;
};

constexpr int kW4Chunk = 128;   // columns of a chunk
constexpr int kW4Tile = 16;     // weight rows of a tile (SwiGLU: 8 gate rows and the 8 up rows beside them)
constexpr int kW4MaxRows = 32;  // rows of x

// A workgroup's waves, which split a row's chunks (16 for a few short walks, see w4_shape).
constexpr int kW4Waves = 8;
// Where x is: its chunks held in registers; or more than they hold, taken in passes, a tile's passes in turn or a batch's
// tiles in turn for each pass.
constexpr int kW4Held = 0, kW4Passes = 1, kW4Batches = 2;
constexpr int kW4Turns = 8;  // tiles of a batch

// Builds of 128 registers, two workgroups to a CU: where x takes few of them, and one row with one scale to a chunk. (Three
// chunks held for several rows fit too, with one tile in flight instead of two: 9497 x 2570 at 5 rows 7.9 -> 8.3 us.)
constexpr bool w4_pairs(int held, int blocks, int subs, int passes, bool one) {
  return blocks == 1 && passes == kW4Held && (held <= 2 || (held <= 4 && subs == 1 && one));
}

// The launch: `held` chunks per wave in registers (of a pass: at a time), `blocks` blocks of 16 operand rows.
struct W4Shape {
  int held, blocks, grid, waves, passes;  // passes: kW4Held, ...
  bool one;                               // a single row of x
};
W4Shape w4_shape(W4Args& a, int subs, int cus);
hipError_t launch_w4_s1(const W4Args& a, const W4Shape& s, hipStream_t stream);  // by groups per chunk
hipError_t launch_w4_s2(const W4Args& a, const W4Shape& s, hipStream_t stream);
hipError_t launch_w4_s4(const W4Args& a, const W4Shape& s, hipStream_t stream);
hipError_t launch_w4(const W4Args& a, int subs, int cus, hipStream_t stream);
hipError_t launch_w4_dequantize(const W4Args& a, int subs, uint16_t* w, hipStream_t stream);

}  // namespace ftk
