// extern "C" entry points of the operators over weights and caches held in few bits: argument checks and dispatch.
#include "../../include/ftk.h"
#include "ftk_q8.h"
#include "ftk_w4.h"

using namespace ftk;

namespace {

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Checks a weight handle and fills what both entry points take from it.
int w4_args(const ftk_w4* w, W4Args& a, int& subs) {
  if (!w || !w->codes || !w->scales || w->N < 1 || w->K < 8) return FTK_ERR_INVALID;
  if (w->group != 32 && w->group != 64 && w->group != 128) return FTK_ERR_INVALID;
  if (w->scale_type != FTK_W4_SCALE_BF16 && w->scale_type != FTK_W4_SCALE_FP16) return FTK_ERR_INVALID;
  if (w->layout != FTK_W4_ROWS && w->layout != FTK_W4_GATE_UP) return FTK_ERR_INVALID;
  const bool gate_up = w->layout == FTK_W4_GATE_UP;
  if (gate_up && w->N % 2) return FTK_ERR_INVALID;
  if (!aligned(w->codes, 16) || !aligned(w->scales, 8) || !aligned(w->zeros, 4)) return FTK_ERR_UNSUPPORTED;
  const int64_t outputs = gate_up ? w->N / 2 : w->N, per = gate_up ? kW4Tile / 2 : kW4Tile;
  const int64_t tiles = (outputs + per - 1) / per, chunks = (w->K + kW4Chunk - 1) / kW4Chunk;
  if (w->N > INT32_MAX / 2 || w->K > (int64_t)1 << 28 || tiles * chunks > INT64_MAX / 4096) return FTK_ERR_INVALID;
  a.codes = (const u32x4_t*)w->codes;
  a.scales = (const uint16_t*)w->scales;
  a.zeros = (const uint8_t*)w->zeros;
  a.N = (int)outputs;
  a.K = (int)w->K;
  a.tiles = (int)tiles;
  a.chunks = (int)chunks;
  a.half_scales = w->scale_type == FTK_W4_SCALE_FP16;
  a.swiglu = gate_up;
  subs = kW4Chunk / w->group;
  return FTK_OK;
}

// The head layouts and sizes both cache entry points take. Blocks: 16, 32, 64 or 128 slots.
int q8_shape(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t capacity, int64_t dim) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || capacity < 1) return FTK_ERR_INVALID;
  if (batch > INT32_MAX / 2 || q_heads > 65536 || kv_heads > 65536 || capacity > INT32_MAX / 2) return FTK_ERR_INVALID;
  if (batch * kv_heads > INT32_MAX / 2) return FTK_ERR_INVALID;
  return dim == 64 || dim == 128 ? FTK_OK : FTK_ERR_UNSUPPORTED;
}

int block_log2(int64_t block) {
  for (int log = 4; log <= 7; ++log)
    if (block == (int64_t)1 << log) return log;
  return -1;
}

// Intervals per (row, KV head): one workgroup a CU, in intervals of at least 256 slots (a unit for each wave); rows of
// long caches stand at different places, and take intervals of 2048 so that the CUs end together. us: 1 x 8 KV heads
// x 32K slots 17.2 in 32 intervals, 19.9 / 18.9 in 16 / 64; 1 x 4K 8.9 in 16, 10.1 / 9.1 in 8 / 32; 16 x 4K 27.2 in 2,
// 30.1 in 1; 32 x 4K (64 heads) 40.1 in 1, 43.9 in 2; 32 x 16K ragged 103 in 8, 113 / 109 in 1 / 16.
// Up to 512 slots one interval needs no merge (8 KV heads 7.1 against 7.6).
constexpr int64_t kQ8OneInterval = 512, kQ8Interval = 256, kQ8LongInterval = 2048, kQ8LongSlots = 8192, kQ8MostIntervals = 64;

int q8_splits(int64_t batch, int64_t kv_heads, int64_t capacity, int cus) {
  if (capacity <= kQ8OneInterval) return 1;
  const int64_t fill = cus / (batch * kv_heads), most = (capacity + kQ8Interval - 1) / kQ8Interval;
  int64_t splits = fill < most ? fill : most;
  const int64_t many = batch > 1 && capacity >= kQ8LongSlots ? capacity / kQ8LongInterval : 1;
  splits = splits > many ? splits : many;
  return (int)(splits < 1 ? 1 : splits > kQ8MostIntervals ? kQ8MostIntervals : splits);
}

int64_t q8_partials(int64_t batch, int64_t q_heads, int64_t dim, int64_t splits) {
  return splits > 1 ? batch * q_heads * splits * (dim + 2) * 4 : 0;
}

}  // namespace

extern "C" {

int ftk_w4_project_bf16(const void* x, int64_t x_stride, const void* gamma, float eps, const ftk_w4* w,
                        const void* residual, void* y, int64_t M, void* stream) {
  W4Args a{};
  int subs = 1;
  const int st = w4_args(w, a, subs);
  if (st != FTK_OK) return st;
  if (!x || !y || M < 1 || M > kW4MaxRows || (M > 1 && x_stride < w->K)) return FTK_ERR_INVALID;
  if (a.swiglu && residual) return FTK_ERR_INVALID;
  if (!aligned(x, 2) || !aligned(y, 2) || !aligned(residual, 2)) return FTK_ERR_UNSUPPORTED;
  if (!aligned(gamma, 2)) return FTK_ERR_UNSUPPORTED;
  const DeviceInfo d = device_info();
  if (!d.ok) return FTK_ERR_INVALID;
  a.gain = (const uint16_t*)gamma;
  a.eps = eps;
  a.x = (const uint16_t*)x;
  a.x_stride = x_stride;
  a.add = (const uint16_t*)residual;
  a.y = (uint16_t*)y;
  a.M = (int)M;
  return hip_status(launch_w4(a, subs, d.cus, reinterpret_cast<hipStream_t>(stream)));
}

int ftk_w4_dequantize_bf16(const ftk_w4* w, void* out, void* stream) {
  W4Args a{};
  int subs = 1;
  const int st = w4_args(w, a, subs);
  if (st != FTK_OK) return st;
  if (!out) return FTK_ERR_INVALID;
  if (!aligned(out, 2)) return FTK_ERR_UNSUPPORTED;
  if ((int64_t)a.tiles * a.chunks * 64 > (int64_t)INT32_MAX * 256) return FTK_ERR_INVALID;
  return hip_status(launch_w4_dequantize(a, subs, (uint16_t*)out, reinterpret_cast<hipStream_t>(stream)));
}

int ftk_qk_rope_cache_q8(const void* packed, const void* q_gain, const void* k_gain, float q_eps, float k_eps,
                         const void* cos, const void* sin, int64_t table_rows, const int64_t* position,
                         const int64_t* phases, void* query, void* keys, void* values, float* k_scales,
                         float* v_scales, int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                         int64_t capacity, int64_t dim, int64_t block, int type, int mode, void* stream) {
  if (!packed || !q_gain || !k_gain || !cos || !sin || !query || !keys || !values || !k_scales || !v_scales)
    return FTK_ERR_INVALID;
  const int st = q8_shape(batch, q_heads, kv_heads, capacity, dim);
  if (st != FTK_OK) return st;
  const int log = block_log2(block);
  if (log < 0 || (type != FTK_Q8_E4M3 && type != FTK_Q8_INT8)) return FTK_ERR_INVALID;
  if (mode & ~(FTK_ROPE_PREFILL | FTK_ROPE_ROWS | FTK_ROPE_TABLE)) return FTK_ERR_INVALID;
  if ((mode & FTK_ROPE_PREFILL) && (mode & FTK_ROPE_ROWS)) return FTK_ERR_INVALID;
  if ((mode & FTK_ROPE_TABLE) && (!(mode & FTK_ROPE_ROWS) || !phases)) return FTK_ERR_INVALID;
  if (!(mode & FTK_ROPE_PREFILL) && !position) return FTK_ERR_INVALID;
  if (tokens < 1 || tokens > capacity || table_rows < 1) return FTK_ERR_INVALID;
  if (!(mode & FTK_ROPE_TABLE) && table_rows < ((mode & FTK_ROPE_ROWS) ? batch * tokens : tokens))
    return FTK_ERR_INVALID;  // shared [1, T, D] or per-row [B, T, D] rows must cover every phase
  // Workgroups: two per block touched, and a query head to 8 or 16 lanes.
  if (batch * tokens > INT32_MAX / 2 || batch * tokens * q_heads > (int64_t)INT32_MAX * 4 ||
      2 * batch * kv_heads * (tokens / block + 2) > INT32_MAX / 2)
    return FTK_ERR_INVALID;
  const void* twos[] = {packed, q_gain, k_gain, cos, sin};
  for (const void* p : twos)
    if (!aligned(p, 2)) return FTK_ERR_UNSUPPORTED;
  if (!aligned(query, 16) || !aligned(keys, 16) || !aligned(values, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4))
    return FTK_ERR_UNSUPPORTED;
  RopeQ8Args a;
  a.packed = (const uint16_t*)packed;
  a.q_gain = (const uint16_t*)q_gain;
  a.k_gain = (const uint16_t*)k_gain;
  a.q_eps = q_eps;
  a.k_eps = k_eps;
  a.cos = (const uint16_t*)cos;
  a.sin = (const uint16_t*)sin;
  a.table_rows = table_rows;
  a.position = position;
  a.phases = phases;
  a.query = (uint16_t*)query;
  a.keys = (uint8_t*)keys;
  a.values = (uint8_t*)values;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.batch = (int)batch;
  a.tokens = (int)tokens;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.capacity = (int)capacity;
  a.dim = (int)dim;
  a.mode = mode;
  a.blocks = (int)((capacity + block - 1) / block);
  a.block_log = log;
  return hip_status(launch_rope_q8(a, type, reinterpret_cast<hipStream_t>(stream)));
}

int ftk_decode_attention_q8_splits(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t capacity, int64_t dim,
                                   int compute_units) {
  if (q8_shape(batch, q_heads, kv_heads, capacity, dim) != FTK_OK || q_heads % kv_heads) return -1;
  if (q_heads / kv_heads > kQ8MaxGroup || compute_units < 0) return -1;
  if (compute_units == 0) {
    const DeviceInfo d = device_info();
    if (!d.ok) return -1;
    compute_units = d.cus;
  }
  return q8_splits(batch, kv_heads, capacity, compute_units);
}

int64_t ftk_decode_attention_q8_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                int splits) {
  if (q8_shape(batch, q_heads, kv_heads, 1, dim) != FTK_OK || splits < 1 || splits > kAttnMaxSplits) return -1;
  return q8_partials(batch, q_heads, dim, splits);
}

int ftk_decode_attention_q8(const void* q, const void* keys, const void* values, const float* k_scales,
                            const float* v_scales, const int64_t* position, int positions, void* out, int64_t batch,
                            int64_t q_heads, int64_t kv_heads, int64_t capacity, int64_t dim, int64_t block,
                            int type, double scale, int splits, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  if (!q || !keys || !values || !k_scales || !v_scales || !position || !out) return FTK_ERR_INVALID;
  const int st = q8_shape(batch, q_heads, kv_heads, capacity, dim);
  if (st != FTK_OK) return st;
  const int log = block_log2(block);
  if (log < 0 || (type != FTK_Q8_E4M3 && type != FTK_Q8_INT8)) return FTK_ERR_INVALID;
  if ((positions != 1 && positions != batch) || q_heads % kv_heads) return FTK_ERR_INVALID;
  if (splits < 0 || splits > kAttnMaxSplits) return FTK_ERR_INVALID;
  if (q_heads / kv_heads > kQ8MaxGroup) return FTK_ERR_UNSUPPORTED;
  if (!aligned(q, 16) || !aligned(keys, 16) || !aligned(values, 16) || !aligned(out, 16) || !aligned(k_scales, 4) ||
      !aligned(v_scales, 4))
    return FTK_ERR_UNSUPPORTED;
  if (splits == 0) {
    const DeviceInfo d = device_info();
    if (!d.ok) return FTK_ERR_INVALID;
    splits = q8_splits(batch, kv_heads, capacity, d.cus);
  }
  if (batch * kv_heads * splits > INT32_MAX / 2) return FTK_ERR_INVALID;
  if (splits > 1 && (!workspace || !aligned(workspace, 16) || workspace_bytes < q8_partials(batch, q_heads, dim, splits)))
    return FTK_ERR_WORKSPACE;
  AttnQ8Args a{};
  AttnShape s{};
  s.dim = (int)dim;
  s.group_size = (int)(q_heads / kv_heads);
  s.groups = (int)(batch * kv_heads);
  s.splits = splits;
  a.base.q = (const uint16_t*)q;
  a.base.position = position;
  a.base.pos_stride = (positions == 1 && batch > 1) ? 0 : 1;
  a.base.out = (uint16_t*)out;
  a.base.partial = (float*)workspace;
  a.base.stats = (float*)workspace + (size_t)batch * q_heads * splits * dim;
  a.base.kv_heads = (int)kv_heads;
  a.base.q_heads = (int)q_heads;
  a.base.capacity = (int)capacity;
  a.base.scale_log2 = (float)(scale * 1.4426950408889634);
  a.k = (const uint8_t*)keys;
  a.v = (const uint8_t*)values;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.blocks = (int)((capacity + block - 1) / block);
  a.block_log = log;
  return hip_status(launch_attn_q8(a, s, type, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
