// The cache held in 8 bits: codes [B, Hkv, C, D] (e4m3 or int8) and one FP32 scale per block of slots of a row and
// head; slot t's value is code * scale[t / block]. Arguments of its writer and of the attention that reads it.
#pragma once

#include "ftk_attn.h"

namespace ftk {

constexpr int kQ8E4m3 = 0, kQ8Int8 = 1;
constexpr int kQ8MaxGroup = 16;  // query heads per KV head (the columns of one matrix instruction)

// Eight codes (two dwords) as the BF16 operand of a matrix instruction. Both types fit BF16 exactly.
template <int KIND>
__device__ __forceinline__ u32x4_t q8_operand(uint32_t lo, uint32_t hi) {
  u32x4_t o;
  if constexpr (KIND == kQ8E4m3) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    const uint32_t d[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = d[i >> 1];
      const float a = (float)(int8_t)(v >> (16 * (i & 1))), b = (float)(int8_t)(v >> (16 * (i & 1) + 8));
      o[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
  }
  return o;
}

struct AttnQ8Args {
  AttnArgs base;          // q, position, out, partials; k and v unused
  const uint8_t* k;       // [groups, capacity, D]
  const uint8_t* v;
  const float* k_scales;  // [groups, blocks]
  const float* v_scales;
  int blocks;             // ceil(capacity / block)
  int block_log;          // log2(block), 4..7
};
hipError_t launch_attn_q8(const AttnQ8Args& a, const AttnShape& s, int kind, hipStream_t stream);

struct RopeQ8Args {
  const uint16_t* packed;    // [B, T, (Hq + 2 Hkv) D] BF16
  const uint16_t* q_gain;    // [D]
  const uint16_t* k_gain;
  float q_eps, k_eps;
  const uint16_t* cos;       // [table_rows, D] BF16
  const uint16_t* sin;
  int64_t table_rows;
  const int64_t* position;
  const int64_t* phases;
  uint16_t* query;           // [B, T, Hq, D] BF16
  uint8_t* keys;             // [B, Hkv, C, D]
  uint8_t* values;
  float* k_scales;           // [B, Hkv, blocks]
  float* v_scales;
  int batch, tokens, q_heads, kv_heads, capacity, dim, mode, blocks, block_log;
};
hipError_t launch_rope_q8(const RopeQ8Args& a, int kind, hipStream_t stream);

}  // namespace ftk
