// Q/K head RMSNorm, RoPE and the write of a step's (or a prompt's) keys and values into the 8-bit cache.
//
// FP32 from the BF16 inputs to the one rounding of each result: n = x / sqrt(mean(x^2) + eps) gain,
// out = n cos + rotate_half(n) sin; query heads rounded to BF16, key and value heads to codes.
// A block's scale is the smallest power of two that keeps its largest finite magnitude within the codes' range
// (448 for e4m3, 127 for int8), at least 2^-126. A power of two loses e4m3 nothing (a floating format), int8 at most
// one bit, and makes a later change of scale cheap to bear: when new slots raise the scale of a block that already
// holds slots, those are re-scaled in place, for e4m3 an exponent shift (exact above its subnormals), for int8 a
// rounding shift (half a step of the final scale, and less than half a step more from all earlier ones).
// A block's slots before the first new one are the valid ones; writing a block's first slot starts its scale anew.
// One workgroup owns a (row, KV head, block) of K or of V, all of its new slots in registers: no atomics, the result
// does not depend on any order.
//
// A step's write is one launch's start and drain (3.4 us for one row of 48 heads of 128, 3.6 for 32 rows); a prompt's
// moves its bytes at a copy's rate: 4001 tokens x 48 heads of 128, 92 MB, 18.5 us or 5.0 TB/s.
#include "../../include/ftk.h"
#include "ftk_q8.h"
#include "ftk_rope.h"

namespace ftk {

namespace {

template <int KIND>
struct Q8 {
  static constexpr float top = KIND == kQ8E4m3 ? 448.f : 127.f;
  static constexpr int top_exp = KIND == kQ8E4m3 ? 8 : 6;                       // top = m 2^top_exp
  static constexpr uint32_t top_frac = KIND == kQ8E4m3 ? 0x600000u : 0x7E0000u;  // m's fraction bits
};

// The smallest power of two s >= 2^-126 with amax <= top s (amax finite, not negative).
template <int KIND>
__device__ __forceinline__ float q8_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - Q8<KIND>::top_exp + ((u & 0x7FFFFFu) > Q8<KIND>::top_frac ? 1 : 0);
  return __uint_as_float((uint32_t)(e > 1 ? e : 1) << 23);
}

// A code's value brought into range: infinities and what lies past the largest code saturate; NaN stays.
template <int KIND>
__device__ __forceinline__ float q8_clamp(float v) {
  return v != v ? v : fminf(fmaxf(v, -Q8<KIND>::top), Q8<KIND>::top);
}

// Four values as four codes, round to nearest even; NaN is e4m3's NaN, and 0 in int8, which has none.
template <int KIND>
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {
  a = q8_clamp<KIND>(a), b = q8_clamp<KIND>(b), c = q8_clamp<KIND>(c), d = q8_clamp<KIND>(d);
  if constexpr (KIND == kQ8E4m3) {
    int o = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, o, true);
  } else {
    const float f[4] = {a, b, c, d};
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o |= ((uint32_t)(int)(f[i] != f[i] ? 0.f : rintf(f[i])) & 0xFFu) << (8 * i);
    return o;
  }
}

template <int KIND>
__device__ __forceinline__ void q8_decode4(uint32_t v, float (&f)[4]) {
  if constexpr (KIND == kQ8E4m3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(v >> (8 * i));
  }
}

// One head's 8 elements of this lane, normalised and rotated; the head is spread over LANES lanes.
template <int LANES>
__device__ __forceinline__ void head_rope(u32x4_t x, u32x4_t gain, u32x4_t cw, u32x4_t sw, float eps, int lane,
                                          float (&out)[8]) {
  float xf[8], gf[8], cf[8], sf[8];
  widen8(x, xf);
  widen8(gain, gf);
  widen8(cw, cf);
  widen8(sw, sf);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += xf[e] * xf[e];
  ss = head_sum<LANES>(ss);
  const float inv_std = 1.0f / sqrtf(ss / (float)(8 * LANES) + eps);
  const bool first = lane < LANES / 2;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = xf[e] * inv_std * gf[e];
    const float partner = __uint_as_float(half_partner<LANES>(__float_as_uint(n)));
    out[e] = n * cf[e] + (first ? -partner : partner) * sf[e];
  }
}

// The table row of token t of batch row b; false: outside the tables (the token is skipped).
__device__ __forceinline__ bool table_row(const RopeQ8Args& a, int b, int t, int64_t& at) {
  at = (a.mode & FTK_ROPE_ROWS) ? (int64_t)b * a.tokens + t : t;
  if (a.mode & FTK_ROPE_TABLE) at = a.position[b] + a.phases[at];
  return at >= 0 && at < a.table_rows;
}

}  // namespace

// Workgroups [0, kv_items): one block of K or V each, its new slots U to a group of D / 8 lanes. The others: query
// heads, QU of one token to a group.
template <int D, int KIND, int U, int QU>
__global__ __launch_bounds__(kThreads) void rope_q8_kernel(RopeQ8Args a, int kv_items, int touched) {
  constexpr int LANES = D / 8, GROUPS = kThreads / LANES;
  const int lane = threadIdx.x & (LANES - 1), group = (int)threadIdx.x / LANES, col = lane * 8;
  const int heads = a.q_heads + 2 * a.kv_heads;
  if ((int)blockIdx.x >= kv_items) {
    const int sets = (a.q_heads + QU - 1) / QU;
    const int64_t item = (int64_t)(blockIdx.x - kv_items) * GROUPS + group;
    const int64_t r = item / sets;
    if (r >= (int64_t)a.batch * a.tokens) return;
    const int first = (int)(item - r * sets) * QU, b = (int)(r / a.tokens), t = (int)(r - (int64_t)b * a.tokens);
    const uint16_t* src = a.packed + r * heads * D + col;
    u32x4_t x[QU];
#pragma unroll
    for (int u = 0; u < QU; ++u) x[u] = load16_any(src + (size_t)(first + u < a.q_heads ? first + u : first) * D);
    const u32x4_t gain = load16_any(a.q_gain + col);
    int64_t at;
    if (!table_row(a, b, t, at)) return;
    const u32x4_t cw = load16_any(a.cos + at * D + col), sw = load16_any(a.sin + at * D + col);
#pragma unroll
    for (int u = 0; u < QU; ++u) {
      if (first + u >= a.q_heads) return;
      float o[8];
      head_rope<LANES>(x[u], gain, cw, sw, a.q_eps, lane, o);
      store16(a.query + (r * a.q_heads + first + u) * D + col,
              u32x4_t{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7])});
    }
    return;
  }
  const int is_v = blockIdx.x & 1, rest = (int)(blockIdx.x >> 1);
  const int j = rest % touched, bh = rest / touched, b = bh / a.kv_heads, kv = bh - b * a.kv_heads;
  const int64_t p0 = (a.mode & FTK_ROPE_PREFILL) ? 0 : a.position[(a.mode & FTK_ROPE_ROWS) ? b : 0];
  if (p0 >= a.capacity || p0 <= -(int64_t)a.tokens) return;
  const int begin = p0 > 0 ? (int)p0 : 0;  // slots [begin, end) are written
  const int end = p0 + a.tokens < a.capacity ? (int)(p0 + a.tokens) : a.capacity;
  const int block = (begin >> a.block_log) + j, start = block << a.block_log;
  if (start >= end) return;
  const int lo = begin > start ? begin : start;
  const int hi = end < start + (1 << a.block_log) ? end : start + (1 << a.block_log);
  uint8_t* const cells = (is_v ? a.values : a.keys) + ((size_t)bh * a.capacity) * D;
  float* const scale_at = (is_v ? a.v_scales : a.k_scales) + (size_t)bh * a.blocks + block;

  float v[U][8];
  uint32_t most = 0;  // the largest finite magnitude's bits + 1 (magnitudes order as their bits); 0: no slot
  bool have[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int slot = lo + group + GROUPS * u;
    const int t = (int)((slot < hi ? slot : hi - 1) - p0);
    int64_t at;
    have[u] = table_row(a, b, t, at) && slot < hi;
    const uint16_t* src = a.packed + ((int64_t)b * a.tokens + t) * heads * D + col;
    if (is_v) {
      widen8(load16_any(src + (size_t)(a.q_heads + a.kv_heads + kv) * D), v[u]);
    } else {
      const int64_t row = have[u] ? at : 0;
      head_rope<LANES>(load16_any(src + (size_t)(a.q_heads + kv) * D), load16_any(a.k_gain + col), load16_any(a.cos + row * D + col),
                       load16_any(a.sin + row * D + col), a.k_eps, lane, v[u]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(v[u][e]);
      if (have[u]) most = max(most, 1u + (m < INFINITY ? __float_as_uint(m) : 0u));
    }
  }
  __shared__ uint32_t red[kThreads / 64];
  most = wave_max_u32(most);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  const uint32_t all = max(max(red[0], red[1]), max(red[2], red[3]));
  if (all == 0) return;  // every token's phase lies outside the tables
  float scale = q8_scale<KIND>(__uint_as_float(all - 1));
  if (lo > start) {
    const float old = *scale_at;
    if (scale > old) {
      const float ratio = old / scale;
      u32x4_t* const p = reinterpret_cast<u32x4_t*>(cells + (size_t)start * D);
      for (int i = threadIdx.x; i < (lo - start) * (D / 16); i += kThreads) {
        const u32x4_t c = p[i];
        u32x4_t o;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float f[4];
          q8_decode4<KIND>(c[w], f);
          o[w] = q8_encode4<KIND>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        }
        p[i] = o;
      }
    } else {
      scale = old;
    }
  }
  const float inv = 1.0f / scale;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int slot = lo + group + GROUPS * u;
    if (!have[u]) continue;
    *reinterpret_cast<u32x2_t*>(cells + (size_t)slot * D + col) =
        u32x2_t{q8_encode4<KIND>(v[u][0] * inv, v[u][1] * inv, v[u][2] * inv, v[u][3] * inv),
                q8_encode4<KIND>(v[u][4] * inv, v[u][5] * inv, v[u][6] * inv, v[u][7] * inv)};
  }
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale_at = scale;
}

namespace {

template <int D, int KIND, int U>
void launch_u(const RopeQ8Args& a, int kv_items, int touched, hipStream_t stream) {
  constexpr int GROUPS = kThreads * 8 / D;
  const int64_t rows = (int64_t)a.batch * a.tokens;
  // A few heads of a token share its table rows where the tokens alone fill the CUs.
  const bool wide = rows >= 1024;
  const int64_t items = rows * (wide ? (a.q_heads + 3) / 4 : a.q_heads);
  const dim3 grid((unsigned)(kv_items + (items + GROUPS - 1) / GROUPS));
  if (wide)
    hipLaunchKernelGGL((rope_q8_kernel<D, KIND, U, 4>), grid, dim3(kThreads), 0, stream, a, kv_items, touched);
  else
    hipLaunchKernelGGL((rope_q8_kernel<D, KIND, U, 1>), grid, dim3(kThreads), 0, stream, a, kv_items, touched);
}

template <int D, int KIND>
void launch_dim(const RopeQ8Args& a, hipStream_t stream) {
  constexpr int GROUPS = kThreads * 8 / D;
  const int block = 1 << a.block_log;
  // Blocks that `tokens` slots can touch: from slot 0 in a prompt, from anywhere in a block else.
  const int touched = (a.mode & FTK_ROPE_PREFILL) ? (a.tokens + block - 1) / block : (a.tokens + block - 2) / block + 1;
  const int kv_items = 2 * a.batch * a.kv_heads * touched;
  const int slots = a.tokens < block ? a.tokens : block;
  if (slots <= GROUPS)
    launch_u<D, KIND, 1>(a, kv_items, touched, stream);
  else if (slots <= 2 * GROUPS)
    launch_u<D, KIND, 2>(a, kv_items, touched, stream);
  else if (slots <= 4 * GROUPS)
    launch_u<D, KIND, 4>(a, kv_items, touched, stream);
  else
    launch_u<D, KIND, 8>(a, kv_items, touched, stream);  // D = 128 and blocks of 128
}

}  // namespace

hipError_t launch_rope_q8(const RopeQ8Args& a, int kind, hipStream_t stream) {
  if (a.dim == 128)
    kind == kQ8E4m3 ? launch_dim<128, kQ8E4m3>(a, stream) : launch_dim<128, kQ8Int8>(a, stream);
  else
    kind == kQ8E4m3 ? launch_dim<64, kQ8E4m3>(a, stream) : launch_dim<64, kQ8Int8>(a, stream);
  return hipGetLastError();
}

}  // namespace ftk
