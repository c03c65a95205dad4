// One-token GQA attention over the 8-bit cache: softmax(q (k s_k)^T scale) (v s_v), split over the slots.
//
// The tile kernel's scheme (ftk_attn_tile.hip) on codes: a wave takes units of 64 slots, whose K and V reach LDS by
// direct loads; codes become BF16 (exactly: e4m3 has 4 significant bits, int8 8) on the way to the 16x16x32 MFMAs, one
// conversion for two values. Scales never touch the codes: a block's K scale joins the softmax scale of its scores
// and its V scale the weights p, one multiplication per score. p goes into the second product as two BF16 addends
// (16 bits of it). V's operand is the transposed 8-bit LDS read: 16 lanes give 8 slots of 16 dimensions and each
// receives one dimension's 8 slots.
//
// The cache read bounds long caches: 32 rows x 8 KV heads x 16K ragged slots (591 MB, read at 1.004 times that) 103 us,
// 5.7 TB/s, against 86 for a pure read in one launch; 1 x 8 x 32K (67 MB) 17.1 against 11.4, the difference the chain
// position -> K -> scores -> V and the merge's launch. Short ones are that chain alone: 4 x 2 x 777 slots 7.0 us, of
// which 5.0 and 2.0 are the two launches.
#include "ftk_dma.h"
#include "ftk_q8.h"

namespace ftk {

namespace {

constexpr int kUnit = 64;  // slots of a unit

// K's codes: tile t (16 slots) at at[j] + t * TILE bytes, j < D / 64 (16 codes each).
template <int J, int TILE>
__device__ __forceinline__ void read_k(const uint32_t (&at)[2], u32x4_t (&k)[4][2]) {
  if constexpr (J == 2) {
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\t"
        "ds_read_b128 %2, %8 offset:%10\n\tds_read_b128 %3, %9 offset:%10\n\t"
        "ds_read_b128 %4, %8 offset:%11\n\tds_read_b128 %5, %9 offset:%11\n\t"
        "ds_read_b128 %6, %8 offset:%12\n\tds_read_b128 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(k[2][0]), "=&v"(k[2][1]),
          "=&v"(k[3][0]), "=&v"(k[3][1])
        : "v"(at[0]), "v"(at[1]), "n"(TILE), "n"(2 * TILE), "n"(3 * TILE)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%5\n\tds_read_b128 %2, %4 offset:%6\n\t"
        "ds_read_b128 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[1][0]), "=&v"(k[2][0]), "=&v"(k[3][0])
        : "v"(at[0]), "n"(TILE), "n"(2 * TILE), "n"(3 * TILE)
        : "memory");
  }
}

// V's codes, transposed: four dimension tiles at at[0..3], slots of both 32-slot halves (HALF bytes apart). Of each
// 16 lanes lane i gives 8 codes of its row i / 2 and receives column i of the eight rows.
template <int HALF>
__device__ __forceinline__ void read_v4(const uint32_t* at, u32x2_t (&v)[4][2]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b8 %2, %9\n\tds_read_b64_tr_b8 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b8 %4, %10\n\tds_read_b64_tr_b8 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b8 %6, %11\n\tds_read_b64_tr_b8 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]),
        "=&v"(v[3][0]), "=&v"(v[3][1])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(HALF)
      : "memory");
}

struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair halves(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return {__uint_as_float(p[0]), __uint_as_float(p[1])};
}
__device__ __forceinline__ Pair row_pairs(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return {__uint_as_float(p[0]), __uint_as_float(p[1])};
}
// Sum, or maximum, over the four lanes li, li + 16, li + 32, li + 48, the same bits in every one of them.
__device__ __forceinline__ float quarter_sum(float v) {
  const Pair r = row_pairs(v);
  const Pair h = halves(r.a + r.b);
  return h.a + h.b;
}
__device__ __forceinline__ float quarter_max(float v) {
  const Pair r = row_pairs(v);
  const Pair h = halves(fmaxf(r.a, r.b));
  return fmaxf(h.a, h.b);
}

// A scale at a wave-uniform index, through the scalar cache.
__device__ __forceinline__ float uniform_f32(const float* p, int i) {
  return ((const __attribute__((address_space(4))) float*)p)[__builtin_amdgcn_readfirstlane(i)];
}

}  // namespace

template <int D, int W, int KIND>
__global__ __launch_bounds__(64 * W, 2) void attn_q8_kernel(AttnQ8Args args) {
  const AttnArgs& a = args.base;
  constexpr int CH = D / 16;                        // 16-byte chunks per cache row
  constexpr int J = D / 64, S = D / 32, DT = D / 16;  // chunks per lane, MFMA steps of a score, dimension tiles
  constexpr int RPL = 64 / CH, L = kUnit / RPL;     // rows per wave load, loads per unit of K (or V)
  constexpr int US = kUnit * CH;                    // 16-byte LDS places of a unit's K (or V)
  constexpr int T = kUnit / 16;                     // slot tiles of a unit
  __shared__ u32x4_t ring[W][2 * US];               // per wave: K, V; at the end the waves' numerators
  __shared__ float m_lds[W][16], l_lds[W][16];
  static_assert(sizeof(ring) >= W * kQ8MaxGroup * D * 4, "the numerators reuse the ring");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, g = lane >> 4, G = a.group_size;
  const int group = blockIdx.x / a.splits, split = blockIdx.x - group * a.splits;
  const int row = group / a.kv_heads;
  const int64_t newest = a.position[a.pos_stride * row];
  const int64_t last = newest < (int64_t)a.capacity - 1 ? newest : (int64_t)a.capacity - 1;
  const int64_t visible = last >= 0 ? last + 1 : 0;
  const int64_t share = interval_slots(a, visible, kUnit);
  const int64_t begin64 = split * share;
  const int begin = (int)(begin64 < visible ? begin64 : visible);  // an interval past the row is empty
  const int end = (int)(begin64 + share < visible ? begin64 + share : visible);
  const int units = (end - begin + kUnit - 1) / kUnit;

  // Query operands: step s = 2 j + h of a score has dimensions 64 j + 16 g + 8 h .. + 7, as K's chunks give them.
  u32x4_t qv[S];
  const u32x4_t zero = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int s = 0; s < S; ++s) {
    qv[s] = load16(a.q + ((size_t)group * G + (li < G ? li : 0)) * D + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
    if (li >= G) qv[s] = zero;
  }

  // Load q brings rows RPL q + lane / CH of a unit; chunk c of a row goes to place c ^ swz(row). Rows at or past
  // `end` re-read row end - 1 (their scores are -inf and their values zeroed below).
  auto swz = [](int r) { return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3; };
  const size_t cache = (size_t)group * a.capacity * D;
  u32x4_t* const mine = ring[wave];
  auto issue = [&](const uint8_t* base, int unit, u32x4_t* dst) {
    const int first = begin + unit * kUnit;
#pragma unroll
    for (int q = 0; q < L; ++q) {
      const int r = RPL * q + lane / CH;
      const int t = first + r < end ? first + r : end - 1;
      dma16<2>(base + cache + (size_t)t * D + 16 * ((lane % CH) ^ swz(r)), dst + 64 * q);
    }
  };
  asm volatile("" ::: "memory");
  if (wave < units) {
    issue(args.k, wave, mine);
    issue(args.v, wave, mine + US);
  }

  float m = -INFINITY, l = 0.f;  // head li's maximum, and this lane's share of its denominator
  f32x4_t acc[DT] = {};          // head li's numerators of dimensions 16 i + 4 g .. + 3
  uint32_t k_at[2], v_at[DT];
  {
    const uint32_t base = lds_address(mine);
#pragma unroll
    for (int j = 0; j < J; ++j) k_at[j] = base + 16 * (li * CH + ((4 * j + g) ^ swz(li)));
    if constexpr (J == 1) k_at[1] = 0;
    const int i8 = li >> 1, r = (i8 < 4 ? 0 : 16) + 4 * g + (i8 & 3);  // the row whose codes this lane gives to its 16
#pragma unroll
    for (int i = 0; i < DT; ++i) v_at[i] = base + 16 * US + 16 * (r * CH + (i ^ swz(r))) + 8 * (li & 1);
  }
  const float* const ks = args.k_scales + (size_t)group * args.blocks;
  const float* const vs = args.v_scales + (size_t)group * args.blocks;

  for (int unit = wave; unit < units; unit += W) {
    const int next = unit + W, first = begin + unit * kUnit;
    const bool more = next < units, ragged = first + kUnit > end;
    float k_scale[T], v_scale[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int at = (first + 16 * t < end ? first + 16 * t : end - 1) >> args.block_log;
      k_scale[t] = uniform_f32(ks, at) * a.scale_log2;
      v_scale[t] = uniform_f32(vs, at);
    }
    wait_vm<L>();  // K; V may still be in flight
    u32x4_t kr[4][2];
    read_k<J, 16 * D>(k_at, kr);
    if (more) issue(args.k, next, mine);
    f32x4_t sc[T] = {};
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const u32x4_t c = kr[t][s >> 1];
        const uint32_t c0 = s & 1 ? c[2] : c[0], c1 = s & 1 ? c[3] : c[1];
        sc[t] = mfma16x16x32(q8_operand<KIND>(c0, c1), qv[s], sc[t]);
      }

    // Element r of sc[t]: slot 16 t + 4 g + r, head li.
    float top = m;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = sc[t][r] * k_scale[t];
        if (ragged && first + 16 * t + 4 * g + r >= end) v = -INFINITY;
        sc[t][r] = v;
        top = fmaxf(top, v);
      }
    top = quarter_max(top);
    const float pivot = top == -INFINITY ? 0.f : top;
    const float corr = exp2_f32(m - pivot);
    float sum = 0.f;
    u32x4_t ph[T / 2], pl[T / 2];  // p s_v as two BF16 addends, the operands of the second product's two steps
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float p[4], low[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = exp2_f32(sc[t][r] - pivot);
        sum += p[r];
        p[r] *= v_scale[t];
        low[r] = p[r] - __uint_as_float(__float_as_uint(p[r]) & 0xFFFF0000u);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ph[t >> 1][2 * (t & 1) + h] =
            __builtin_amdgcn_perm(__float_as_uint(p[2 * h + 1]), __float_as_uint(p[2 * h]), 0x07060302u);
        pl[t >> 1][2 * (t & 1) + h] = rne_pair(low[2 * h], low[2 * h + 1]);
      }
    }
    l = l * corr + sum;
    m = top;
    if (__any(corr != 1.f)) {
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= corr;
    }

    if (more) wait_vm<L>(); else wait_vm<0>();  // V; the next K may still be in flight
    u32x2_t vr[DT / 4][4][2];
#pragma unroll
    for (int i = 0; i < DT / 4; ++i) read_v4<32 * D>(v_at + 4 * i, vr[i]);
    if (more) issue(args.v, next, mine + US);
    if (ragged) {  // codes of slots past the end: zero, whatever the re-read row holds
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int left = end - (first + 32 * h + 16 * w + 4 * g);  // slots of this dword inside the row
          const uint32_t keep = left >= 4 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
          for (int i = 0; i < DT; ++i) vr[i / 4][i % 4][h][w] &= keep;
        }
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x2_t c = vr[i / 4][i % 4][h];
        const u32x4_t va = q8_operand<KIND>(c[0], c[1]);
        acc[i] = mfma16x16x32(va, pl[h], acc[i]);
        acc[i] = mfma16x16x32(va, ph[h], acc[i]);
      }
  }

  // The waves' states, merged in wave order (their numerators through the ring's LDS).
  l = quarter_sum(l);
  __syncthreads();  // every wave is past its last read of the ring
  float* const num = reinterpret_cast<float*>(&ring[0][0]);  // [W][G][D]
  if (li < G) {
#pragma unroll
    for (int i = 0; i < DT; ++i)
      *reinterpret_cast<f32x4_t*>(num + ((size_t)wave * G + li) * D + 16 * i + 4 * g) = acc[i];
    if (g == 0) {
      m_lds[wave][li] = m;
      l_lds[wave][li] = l;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < G * (D / 8); t += 64 * W) {
    const int h = t / (D / 8), cc = t - h * (D / 8);
    float mm = m_lds[0][h], ll = l_lds[0][h], aa[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) aa[e] = num[(size_t)h * D + cc * 8 + e];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      float a2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a2[e] = num[((size_t)w * G + h) * D + cc * 8 + e];
      merge_state(mm, ll, aa, m_lds[w][h], l_lds[w][h], a2);
    }
    // A row that sees no slot gives zeros (with several intervals the merge sees to it).
    store_state(a, group, split, h, cc, G, D, mm, a.splits == 1 && ll == 0.f ? 1.f : ll, aa);
  }
}

hipError_t launch_attn_q8(const AttnQ8Args& a, const AttnShape& s, int kind, hipStream_t stream) {
  AttnQ8Args args = a;
  args.base.group_size = s.group_size;
  args.base.splits = s.splits;
  int log = 0;  // ceil(log2 splits)
  while ((1 << log) < s.splits) ++log;
  args.base.split_magic = (uint32_t)(((uint64_t)1 << (31 + log)) / s.splits + 1);
  args.base.split_shift = 31 + log;
  // Four waves: with eight (all of a CU's LDS) no shape was faster, since a CU's own rate bounds few intervals
  // (1 x 1K slots in one interval 10.4 us either way) and the device's many (1 x 32K in 32: 17.2 against 17.9).
  const dim3 grid((unsigned)(s.groups * s.splits)), block(256);
  typedef void (*Kernel)(AttnQ8Args);
  const Kernel kernel = s.dim == 128 ? (kind == kQ8E4m3 ? attn_q8_kernel<128, 4, kQ8E4m3> : attn_q8_kernel<128, 4, kQ8Int8>)
                                     : (kind == kQ8E4m3 ? attn_q8_kernel<64, 4, kQ8E4m3> : attn_q8_kernel<64, 4, kQ8Int8>);
  hipLaunchKernelGGL(kernel, grid, block, 0, stream, args);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || s.splits == 1) return e;
  return launch_attn_merge(args.base, s, true, stream);
}

}  // namespace ftk
