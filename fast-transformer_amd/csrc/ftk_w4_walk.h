// The walk over 4-bit weight tiles (ftk_w4.hip has the mathematics and the launch rule).
#pragma once

#include "ftk_dma.h"
#include "ftk_w4.h"

namespace ftk {

namespace w4 {

__device__ __forceinline__ float scale_f32(uint32_t bits, bool half) {
  return half ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : bf16_to_f32(bits);
}

__device__ __forceinline__ bool finite_f32(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// Elements k .. k + 7 of a row of K >= 8, zero past its end: the last 8 of the row (row_part), moved down.
__device__ __forceinline__ u32x4_t row_part(const uint16_t* row, int k, int K) {
  return load16_any(row + (k <= K - 8 ? k : K - 8));
}
__device__ __forceinline__ u32x4_t row_moved(u32x4_t v, int k, int K) {
  const int down = k <= K - 8 ? 0 : k - (K - 8);
  uint64_t lo = v[0] | (uint64_t)v[1] << 32, hi = v[2] | (uint64_t)v[3] << 32;
  lo = down & 4 ? hi : lo;
  hi = down & 4 ? 0 : hi;
  lo = down & 3 ? lo >> 16 * (down & 3) | hi << (64 - 16 * (down & 3)) : lo;
  hi >>= 16 * (down & 3);
  lo = down >= 8 ? 0 : lo;
  hi = down >= 8 ? 0 : hi;
  return u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// The operand of one step: 128 + q for the 8 codes of a dword. The constants sit in registers (an instruction takes
// one literal): (v >> 4 i) & mask | ones is a shift and one v_and_or_b32.
struct Unpack {
  uint32_t mask = 0x000F000Fu, ones = 0x43004300u;
  __device__ __forceinline__ Unpack() { asm volatile("" : "+s"(mask), "+v"(ones)); }
  __device__ __forceinline__ u32x4_t operator()(uint32_t v) const {
    u32x4_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = ((v >> (4 * i)) & mask) | ones;
    return o;
  }
};

__device__ __forceinline__ uint32_t code(const W4Args& a, int tile, int li, int k) {
  const int c = k / kW4Chunk, r = k % kW4Chunk, s = r / 32, g = (r % 32) / 8, e = r % 8;
  const uint32_t* d = reinterpret_cast<const uint32_t*>(a.codes + ((size_t)tile * a.chunks + c) * 64 + 16 * g + li);
  return (d[s] >> (4 * (e / 2) + 16 * (e % 2))) & 15u;
}

// One output's sum element by element, each product s (q - z) x: what the definition says for an x that holds
// infinities or values whose 128-fold is one. (A short loop, not a fast one: with eight elements to a step its registers
// cost every other call 2 to 6 %; a row that holds NaN takes 2 to 9 ms.)
template <int S>
__device__ __forceinline__ float exact_sum(const W4Args& a, int tile, int li, int m) {
  float sum = 0.f;
#pragma unroll 1
  for (int k = 0; k < a.K; ++k) {
    const size_t at = (((size_t)tile * a.chunks + k / kW4Chunk) * 16 + li) * S + (k % kW4Chunk) * S / kW4Chunk;
    const float z = a.zeros != nullptr ? (float)a.zeros[at] : 8.f;
    const float w = ((float)code(a, tile, li, k) - z) * scale_f32(a.scales[at], a.half_scales);
    float x = bf16_to_f32(a.x[(size_t)m * a.x_stride + k]);
    if (a.gain != nullptr) x *= bf16_to_f32(a.gain[k]);
    sum += w * x;
  }
  return sum;
}

// S scales (16 bits each) or zero points (8 bits each) of one row and chunk. Past the tile's range: zeros. Kept as
// narrow as they are loaded: widened at the load, they would be waited for there, and every load before them.
template <int BITS>
struct Narrow;
template <>
struct Narrow<8> {
  uint8_t v;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at) {
    v = __builtin_amdgcn_raw_buffer_load_b8(rsrc, at, 0, 2);
  }
  __device__ __forceinline__ uint32_t word(int) const { return v; }
};
template <>
struct Narrow<16> {
  uint16_t v;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at) {
    v = __builtin_amdgcn_raw_buffer_load_b16(rsrc, 2 * at, 0, 2);
  }
  __device__ __forceinline__ uint32_t word(int) const { return v; }
};
template <>
struct Narrow<32> {
  uint32_t v;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at) {
    v = __builtin_amdgcn_raw_buffer_load_b32(rsrc, 4 * at, 0, 2);
  }
  __device__ __forceinline__ uint32_t word(int) const { return v; }
};
template <>
struct Narrow<64> {
  u32x2_t v;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at) {
    v = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rsrc, 8 * at, 0, 2));
  }
  __device__ __forceinline__ uint32_t word(int i) const { return v[i]; }
};
template <int S>
struct Scales : Narrow<16 * S> {
  __device__ __forceinline__ float get(int s, bool half) const {
    const uint32_t w = this->word(s >> 1);
    const float as_half = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> (16 * (s & 1))));
    return half ? as_half : s & 1 ? hi_f32(w) : lo_f32(w);
  }
};
template <int S>
struct Zeros : Narrow<8 * S> {
  __device__ __forceinline__ uint32_t get(int s) const { return (this->word(0) >> (8 * s)) & 0xFFu; }
};

// Eight x values times their gains as two BF16 addends: the product has 16 significant bits, so the rounded one and
// what is left of it hold it exactly.
struct Gained {
  u32x4_t hi, low;
};
__device__ __forceinline__ Gained gained(u32x4_t x, const float (&gain)[8]) {
  float xf[8];
  widen8(x, xf);
  Gained o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p0 = xf[2 * i] * gain[2 * i], p1 = xf[2 * i + 1] * gain[2 * i + 1];
    const uint32_t hi = rne_pair(p0, p1);
    o.hi[i] = hi;
    o.low[i] = rne_pair(p0 - lo_f32(hi), p1 - hi_f32(hi));
  }
  return o;
}

// Sum of a lane's value over the 4, 8 or 16 lanes that hold a group's pieces (S groups to 16 pieces).
template <int S>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp<0xB1, 0xF>(v);
  v += dpp<0x4E, 0xF>(v);
  if constexpr (S < 4) v += dpp<0x141, 0xF>(v);
  if constexpr (S < 2) v += dpp<0x140, 0xF>(v);
  return v;
}

}  // namespace w4

// A workgroup walks tiles walker, walker + walkers, ... Its W waves split a tile's chunks (chunk = wave + W j), so
// every wave needs its own chunks of x only. KC: chunks per wave in registers; CB: blocks of 16 operand rows. x is
// the A operand and the weights the B operand: a lane's accumulators belong to one weight row, one scale serves them.
// XS: more chunks than registers hold. kW4Passes: a tile takes several passes, and x is read again for each. kW4Batches:
// the tiles of a batch take a pass in turn, their sums so far in LDS, and x is read again for each batch and pass.
// With a gain the operand rows are the rows' x gain as two BF16 addends (rows, then their low parts), and 1 / rms
// joins in the epilogue: no product waits for the norm's sum, and x gain loses nothing.
// Rows reach the operand through the wave's own part of LDS: read in the operand's layout, a load touches 16 rows x 64
// bytes in 64 separate pieces (16 rows of 6144 x 4096: 21 us, most of it those loads); read along the rows, 256 bytes
// of four at a time, they cost a quarter. ONE (a single row of x, CB = 1): a load takes the row's four chunks instead.
// Either way a piece of 8 elements is multiplied by its gain and summed in one lane, once.
// One row with one scale to a chunk and at most 4 chunks takes 128 registers with PF = 1: two workgroups to a CU hide
// more than two tiles in flight do (24576 x 4096 + norm 12.6 -> 12.1 us, 6144 x 4096 + norm 6.2 -> 6.0).
// The weights of the next PF tiles are in flight; x goes out ahead of the first ones, since loads return in order.
template <int KC, int CB, int S, bool ZP, int XS, bool ONE, int W>
__global__ __launch_bounds__(64 * W, (W == 16 || w4_pairs(KC, CB, S, XS, ONE) ? 4 : 2)) void w4_walk_kernel(W4Args a) {
  using namespace w4;
  static_assert(!ONE || CB == 1, "one row fills no block");
  constexpr int PF = w4_pairs(KC, CB, S, XS, ONE) && KC > 2 ? 1 : (S == 4 ? KC * CB <= 4 : KC * CB <= 6) && !XS ? 2 : 1;
  constexpr int Q = ONE ? (KC + 3) / 4 : 1;  // pieces of the row per lane
  constexpr bool TURNS = XS == kW4Batches, PASSES = XS == kW4Passes && !ONE;
  constexpr int T = TURNS ? kW4Turns : 2;
  __shared__ float red[T][W][16 * CB][17];
  __shared__ float ssq[W][16 * CB];
  __shared__ f32x4_t xsum[W][KC * S][4 * CB];  // per group: sums of the operand rows
  // ONE: pieces [W][KC 16][R]; else a chunk's [W][16 CB rows][16], piece p of row r at place p ^ (r % 16).
  extern __shared__ u32x4_t dyn[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4;
  const Unpack unpack;
  // The row blocks of one walk are 8 workgroups apart: on one XCD, whose L2 then serves their weights twice.
  const int unit = blockIdx.x >> 3, row_block = unit % a.row_blocks;
  const int walker = (unit / a.row_blocks) * 8 + (blockIdx.x & 7), walkers = gridDim.x / a.row_blocks;
  const int m0 = row_block * a.rows, rows = a.M - m0 < a.rows ? a.M - m0 : a.rows;
  const bool norm = a.gain != nullptr;
  const int operands = norm ? 2 * rows : rows;
  const u32x4_t one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  const uint32_t chunk_bytes = (uint32_t)a.chunks * 1024u;
  struct Tile {
    __amdgpu_buffer_rsrc_t codes, scales, zeros;
  };
  auto tile_of = [&](int tile) {  // past the last tile: empty ranges, whose loads read nothing
    const bool there = tile < a.tiles;
    const size_t block = (size_t)(there ? tile : 0) * a.chunks;
    Tile t;
    t.codes = __builtin_amdgcn_make_buffer_rsrc((void*)(a.codes + block * 64), 0, there ? chunk_bytes : 0u, kBufferFlags);
    t.scales = __builtin_amdgcn_make_buffer_rsrc((void*)(a.scales + block * 16 * S), 0,
                                                 there ? (uint32_t)a.chunks * 32u * S : 0u, kBufferFlags);
    if constexpr (ZP)
      t.zeros = __builtin_amdgcn_make_buffer_rsrc((void*)(a.zeros + block * 16 * S), 0,
                                                  there ? (uint32_t)a.chunks * 16u * S : 0u, kBufferFlags);
    return t;
  };
  u32x4_t w[PF][KC];
  Scales<S> sc[PF][KC];
  Zeros<S> zp[PF][KC];
  auto load_weights = [&](const Tile& t, int f, int j, int chunk) {
    w[f][j] = buffer_load16(t.codes, (uint32_t)chunk * 1024u + 16u * lane);
    sc[f][j].load(t.scales, (uint32_t)chunk * 16u + li);
    if constexpr (ZP) zp[f][j].load(t.zeros, (uint32_t)chunk * 16u + li);
  };

  u32x4_t x[CB][PASSES ? 1 : KC][4];
  if constexpr (ONE) {
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int s = 0; s < 4; ++s) x[0][j][s] = u32x4_t{};
  }

  // With a gain the low parts follow `lower` operand rows after the rows.
  const int lower = ONE ? rows : 8 * CB;

  // A group's sum of an operand row, times what the accumulators start at (with zero points that is their matter). The
  // low parts' share is in their row's; theirs is zero.
  auto keep_sum = [&](int group, int r, float sum) {
    float* const at = reinterpret_cast<float*>(&xsum[wave][group][0]);
    at[r] = ZP ? sum : -136.f * sum;
    if (norm) at[lower + r] = 0.f;
  };

  // ONE: raw pieces of a pass (chunk wave + 8 (4 q + g) of it, piece li), and their way into the operand.
  u32x4_t raw[Q], raw_gain[Q];
  u32x4_t* const pieces = dyn + (ONE ? (size_t)wave * KC * 16 * operands : 0);
  float row_squares = 0.f;
  auto piece_chunk = [&](int pass, int q, int g4) { return pass * KC * W + wave + W * (4 * q + g4); };
  auto load_pieces = [&](int pass) {
    if constexpr (ONE) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int k = piece_chunk(pass, q, g) * kW4Chunk + 8 * li;
        raw[q] = row_part(a.x, k, a.K);
        raw_gain[q] = row_part(norm ? a.gain : a.x, k, a.K);
      }
    }
  };
  auto form_pieces = [&](int pass, bool count) {
    if constexpr (ONE) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int j = 4 * q + g;
        u32x4_t v = raw[q], gn = raw_gain[q];
        if ((piece_chunk(pass, q, 3) + 1) * kW4Chunk > a.K) {  // wave-uniform: the row's end is among these chunks
          const int k = piece_chunk(pass, q, g) * kW4Chunk + 8 * li;
          v = row_moved(v, k, a.K);
          gn = row_moved(gn, k, a.K);
        }
        float sum;
        const int at = (16 * j + li) * operands;
        const bool mine = KC % 4 == 0 || j < KC;
        if (norm) {
          float gf[8];
          widen8(gn, gf);
          if (count && mine) row_squares = sum_squares8(v, row_squares);  // (past KC: the next pass's)
          const Gained o = gained(v, gf);
          if (mine) {
            pieces[at] = o.hi;
            pieces[at + 1] = o.low;
          }
          sum = dot8(o.low, one, dot8(o.hi, one, 0.f));
        } else {
          if (mine) pieces[at] = v;
          sum = dot8(v, one, 0.f);
        }
        sum = group_sum<S>(sum);
        if (mine && li % (16 / S) == 0) keep_sum(j * S + li / (16 / S), 0, sum);
      }
      if (li < operands) {  // (the other lanes' operands stay zero)
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int s = 0; s < 4; ++s) x[0][j][s] = pieces[(16 * j + 4 * s + g) * operands + li];
      }
    }
  };

  // Many rows: piece li of rows 4 i + g of a chunk.
  constexpr int I = 4 * CB;  // row quads (with a gain half of them, where CB = 2: the other block holds low parts)
  u32x4_t many[ONE ? 1 : KC][ONE ? 1 : I], many_gain[KC];
  float ss[I] = {};
  u32x4_t* const chunk_lds = dyn + (ONE ? 0 : (size_t)wave * 16 * 16 * CB);
  auto load_chunk = [&](int j, int chunk) {
    if constexpr (!ONE) {
      const int k = chunk * kW4Chunk + 8 * li;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if (4 * i >= rows) continue;
        const int m = 4 * i + g < rows ? 4 * i + g : rows - 1;
        many[j][i] = row_part(a.x + (size_t)(m0 + m) * a.x_stride, k, a.K);
      }
      if (norm) many_gain[j] = row_part(a.gain, k, a.K);
    }
  };
  auto form_chunk = [&](int j, int chunk, bool count) {
    if constexpr (!ONE) {
      const int k = chunk * kW4Chunk + 8 * li;
      u32x4_t gn = many_gain[j];
      if ((chunk + 1) * kW4Chunk > a.K) {  // wave-uniform: a row's last chunk and beyond, zeros past its end
#pragma unroll
        for (int i = 0; i < I; ++i)
          if (4 * i < rows) many[j][i] = row_moved(many[j][i], k, a.K);
        if (norm) gn = row_moved(gn, k, a.K);
      }
      float gf[8];
      widen8(gn, gf);
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if (4 * i >= rows) continue;
        const u32x4_t v = many[j][i];
        const int r = 4 * i + g;
        float sum;
        if (norm) {  // (at most 8 CB rows: the quads past them are never reached)
          if (count) ss[i] = sum_squares8(v, ss[i]);
          const Gained o = gained(v, gf);
          chunk_lds[r * 16 + (li ^ (r & 15))] = o.hi;
          chunk_lds[(lower + r) * 16 + (li ^ ((lower + r) & 15))] = o.low;
          sum = group_sum<S>(dot8(o.low, one, dot8(o.hi, one, 0.f)));
        } else {
          chunk_lds[r * 16 + (li ^ (r & 15))] = v;
          sum = group_sum<S>(dot8(v, one, 0.f));
        }
        if (li % (16 / S) == 0) keep_sum(j * S + li / (16 / S), r, sum);
      }
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          x[b][PASSES ? 0 : j][s] = chunk_lds[(16 * b + li) * 16 + ((4 * s + g) ^ li)];
    }
  };
  auto keep_squares = [&]() {
    if constexpr (ONE) {
      const float sum = wave_sum(row_squares);
      if (lane == 0) ssq[wave][0] = sum;
      return;
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const float sum = group_sum<1>(ss[i]);
      if (li == 0) ssq[wave][4 * i + g] = sum;
    }
  };

  const int passes = XS ? (a.chunks + KC * W - 1) / (KC * W) : 1;
  if constexpr (ONE) {
    load_pieces(0);
  } else {
#pragma unroll
    for (int j = 0; j < KC; ++j) load_chunk(j, wave + W * j);
  }
  asm volatile("" ::: "memory");
  // Steps: a tile's passes in turn, then the next tile's. TURNS: a batch's tiles in turn, then their next pass, then the
  // next batch. The loads are PF steps ahead of the one computed.
  struct Step {
    int tile, pass, first, at;  // at: the tile's place in the batch that begins with tile `first`
  };
  auto last_of_pass = [&](const Step& st) { return st.at + 1 == T || st.tile + walkers >= a.tiles; };
  auto advance = [&](Step& st) {
    if constexpr (TURNS) {
      if (!last_of_pass(st)) {
        st.tile += walkers;
        ++st.at;
        return;
      }
      if (++st.pass == passes) {
        st.pass = 0;
        st.first = st.tile + walkers;
      }
      st.tile = st.first;
      st.at = 0;
    } else if (!XS || ++st.pass == passes) {
      st.pass = 0;
      st.tile += walkers;
      st.first = st.tile;
    }
  };
  Step ahead = {walker, 0, walker, 0};
  Tile from = tile_of(walker);
  auto next_load = [&]() {
    const int was = ahead.tile;
    advance(ahead);
    if (!XS || ahead.tile != was) from = tile_of(ahead.tile);
  };
#pragma unroll
  for (int f = 0; f < PF; ++f) {
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      load_weights(from, f, j, ahead.pass * KC * W + wave + W * j);
      // (In the loop's order: a wait counts the loads behind the one it waits for, on this way into the loop as well.)
      __builtin_amdgcn_sched_barrier(0);
    }
    next_load();
  }
  if constexpr (!XS) {
    if constexpr (ONE) {
      form_pieces(0, true);
    } else {
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        form_chunk(j, wave + W * j, true);
        __builtin_amdgcn_sched_barrier(0);  // one chunk's temporaries at a time
      }
    }
    if (norm) keep_squares();
  }

  __shared__ float inverse[16 * CB];  // 1 / rms of the rows, from the first tile on
  int buf = 0, turn = 0;
  Step now = {walker, 0, walker, 0};
  f32x4_t acc[CB] = {};
  while (now.tile < a.tiles) {
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      // Past the walk's end a step computes nothing, but its loads (of nothing) go out: with an exit here the waits at
      // the loop's head would allow for the loads of this step only.
      const int tile = now.tile, p = now.pass;
      const bool active = f == 0 || tile < a.tiles;
      // Many groups' sums stay in LDS: read for every tile (an index the compiler cannot see through), not kept in
      // registers over the walk.
      int part_of = 0;
      if constexpr (KC * S * CB > 4) asm volatile("" : "+s"(part_of));
      if constexpr (ONE && XS) {
        if (active) form_pieces(p, tile == walker);
        load_pieces(p + 1 == passes ? 0 : p + 1);
      }
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        if constexpr (TURNS || PASSES) {
          if (PASSES || now.at == 0) {  // (the first of a batch's tiles brings the pass's x into the operand)
            form_chunk(j, p * KC * W + wave + W * j, now.first == walker);
            load_chunk(j, (p + 1 == passes ? 0 : p + 1) * KC * W + wave + W * j);
          }
        }
        if (active) {
          float scale[S];
#pragma unroll
          for (int s = 0; s < S; ++s) scale[s] = sc[f][j].get(s, a.half_scales);
#pragma unroll
          for (int s = 0; s < S; ++s) {
            f32x4_t part[CB];
#pragma unroll
            for (int b = 0; b < CB; ++b) {
              part[b] = xsum[wave][j * S + s + part_of][4 * b + g];
              if constexpr (ZP) part[b] *= -(128.f + (float)zp[f][j].get(s));
            }
#pragma unroll
            for (int i = 4 / S * s; i < 4 / S * (s + 1); ++i) {
              const uint32_t wv = w[f][j][i];
              const u32x4_t o = unpack(wv);
#pragma unroll
              for (int b = 0; b < CB; ++b) part[b] = mfma16x16x32(x[b][PASSES ? 0 : j][i], o, part[b]);
            }
#pragma unroll
            for (int b = 0; b < CB; ++b) acc[b] += part[b] * scale[s];
          }
          // The scales are formed before the loads that replace their words: a word still to be read would be loaded
          // into another register, and the copy back at the end of the loop waits for every load in flight.
#pragma unroll
          for (int s = 0; s < S; ++s) asm volatile("" ::"v"(scale[s]) : "memory");
        }
        load_weights(from, f, j, ahead.pass * KC * W + wave + W * j);
        __builtin_amdgcn_sched_barrier(0);
      }
      next_load();
      if constexpr (XS) {
        const Step done = now;
        if (active) advance(now);
        if constexpr (TURNS) {
          // A tile's sums over the passes so far stay in its wave's place. (A batch's last tile may still be read for the
          // outputs of the batch before; the others' readers have passed that tile's barrier.)
          if (done.at + 1 == T && p == 0 && done.first != walker) lds_barrier();
#pragma unroll
          for (int b = 0; b < CB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float* const at = &red[done.at][wave][16 * b + 4 * g + r][li];
              *at = p == 0 ? acc[b][r] : acc[b][r] + *at;
              if (r == 3) acc[b] = f32x4_t{};
            }
          buf = done.at;
        }
        if (active && p + 1 < passes) continue;
      } else {
        if (active) advance(now);
      }
      if (!active) continue;
      // Element r of acc[b]: operand row 16 b + 4 g + r, weight row li of the tile.
      if constexpr (!TURNS) {
#pragma unroll
        for (int b = 0; b < CB; ++b) {
#pragma unroll
          for (int r = 0; r < 4; ++r) red[buf][wave][16 * b + 4 * g + r][li] = acc[b][r];
          acc[b] = f32x4_t{};
        }
      }
      if (XS && norm && tile == walker) keep_squares();
      lds_barrier();
      // (The other buffer is written next; its readers all pass this barrier's successor first. The waves take turns
      // with a tile's outputs, so that few rows do not always hold up the same one.)
      const int cols = a.swiglu ? 8 : 16;  // outputs of a tile
      for (int i = (threadIdx.x + 64 * turn) & (64 * W - 1); i < rows * cols; i += 64 * W) {
        const int col = a.swiglu ? i & 7 : i & 15, r = a.swiglu ? i >> 3 : i >> 4, m = m0 + r;
        const int n = tile * cols + col;
        if (n >= a.N) continue;
        float v = 0.f, u = 0.f, inv = 1.f;
#pragma unroll
        for (int wv = 0; wv < W; ++wv) v += red[buf][wv][r][col];
        if (a.swiglu) {
#pragma unroll
          for (int wv = 0; wv < W; ++wv) u += red[buf][wv][r][col + 8];
        }
        if (norm) {
#pragma unroll
          for (int wv = 0; wv < W; ++wv) v += red[buf][wv][lower + r][col];
          if (a.swiglu) {
#pragma unroll
            for (int wv = 0; wv < W; ++wv) u += red[buf][wv][lower + r][col + 8];
          }
          if (tile == walker) {
            float sum = 0.f;
#pragma unroll
            for (int wv = 0; wv < W; ++wv) sum += ssq[wv][r];
            inv = 1.0f / sqrtf(sum / (float)a.K + a.eps);
            if (col == 0) inverse[r] = inv;
          } else {
            inv = inverse[r];
          }
        }
        if (__builtin_expect(!finite_f32(v), 0)) v = exact_sum<S>(a, tile, col, m);
        v *= inv;
        if (a.swiglu) {
          if (__builtin_expect(!finite_f32(u), 0)) u = exact_sum<S>(a, tile, col + 8, m);
          v = silu_f32(v) * (u * inv);
        }
        if (a.add != nullptr) v += bf16_to_f32(a.add[(size_t)m * a.N + n]);
        a.y[(size_t)m * a.N + n] = (uint16_t)f32_to_bf16(v);
      }
      buf ^= 1;
      turn = (turn + 1) & (W - 1);
    }
  }
}

namespace w4 {

template <int KC, int CB, int S, int XS, bool ONE, int W = kW4Waves>
void launch(const W4Args& a, const W4Shape& s, hipStream_t stream) {
  const int operands = (a.gain != nullptr ? 2 : 1) * a.rows;
  const size_t lds = W * 256 * (ONE ? (size_t)KC * operands : (size_t)16 * CB);
  if (a.zeros != nullptr)
    hipLaunchKernelGGL((w4_walk_kernel<KC, CB, S, true, XS, ONE, W>), dim3(s.grid), dim3(64 * W), lds, stream, a);
  else
    hipLaunchKernelGGL((w4_walk_kernel<KC, CB, S, false, XS, ONE, W>), dim3(s.grid), dim3(64 * W), lds, stream, a);
}

// Every launch that w4_shape makes.
template <int S>
hipError_t launch_shape(const W4Args& a, const W4Shape& s, hipStream_t stream) {
  const int key = (s.waves == 16 ? 8000 : 0) + (s.one ? 4000 : 0) + 1000 * s.passes + s.blocks * 100 + s.held;
  if constexpr (S < 4) {
    if (key == 204) {
      launch<4, 2, S, kW4Held, false>(a, s, stream);
      return hipGetLastError();
    }
  }
  switch (key) {
    case 101: launch<1, 1, S, kW4Held, false>(a, s, stream); break;
    case 102: launch<2, 1, S, kW4Held, false>(a, s, stream); break;
    case 103: launch<3, 1, S, kW4Held, false>(a, s, stream); break;
    case 104: launch<4, 1, S, kW4Held, false>(a, s, stream); break;
    case 106: launch<(S < 4 ? 6 : 4), 1, S, kW4Held, false>(a, s, stream); break;
    case 108: launch<(S < 2 ? 8 : 4), 1, S, kW4Held, false>(a, s, stream); break;
    case 8102: launch<2, 1, S, kW4Held, false, 16>(a, s, stream); break;
    case 1104: launch<4, 1, S, kW4Passes, false>(a, s, stream); break;
    // (Four groups to a chunk: three chunks of a pass, four would spill.)
    case 2104: launch<(S < 4 ? 4 : 3), 1, S, kW4Batches, false>(a, s, stream); break;
    case 4101: launch<1, 1, S, kW4Held, true>(a, s, stream); break;
    case 4102: launch<2, 1, S, kW4Held, true>(a, s, stream); break;
    case 4103: launch<3, 1, S, kW4Held, true>(a, s, stream); break;
    case 4104: launch<4, 1, S, kW4Held, true>(a, s, stream); break;
    case 4106: launch<(S < 4 ? 6 : 4), 1, S, kW4Held, true>(a, s, stream); break;
    case 4108: launch<(S < 2 ? 8 : 4), 1, S, kW4Held, true>(a, s, stream); break;
    case 5104:
    case 5106: launch<(S < 4 ? 6 : 4), 1, S, kW4Passes, true>(a, s, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace w4

}  // namespace ftk
