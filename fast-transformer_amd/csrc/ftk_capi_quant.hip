// extern "C" entry points of the operators over weights and caches held in few bits: argument checks and dispatch.
#include "../../include/ftk.h"
#include "ftk_w4.h"

using namespace ftk;

namespace {

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Checks a weight handle and fills what both entry points take from it.
int w4_args(const ftk_w4* w, W4Args& a, int& subs, bool& gate_up) {
  if (!w || !w->codes || !w->scales || w->N < 1 || w->K < 1) return FTK_ERR_INVALID;
  if (w->group != 32 && w->group != 64 && w->group != 128) return FTK_ERR_INVALID;
  if (w->scale_type != FTK_W4_SCALE_BF16 && w->scale_type != FTK_W4_SCALE_FP16) return FTK_ERR_INVALID;
  if (w->layout != FTK_W4_ROWS && w->layout != FTK_W4_GATE_UP) return FTK_ERR_INVALID;
  gate_up = w->layout == FTK_W4_GATE_UP;
  if (gate_up && w->N % 2) return FTK_ERR_INVALID;
  if (!aligned(w->codes, 16) || !aligned(w->scales, 8) || !aligned(w->zeros, 4)) return FTK_ERR_UNSUPPORTED;
  const int64_t outputs = gate_up ? w->N / 2 : w->N, per = gate_up ? kW4Tile / 2 : kW4Tile;
  const int64_t tiles = (outputs + per - 1) / per, chunks = (w->K + kW4Chunk - 1) / kW4Chunk;
  if (w->N > INT32_MAX / 2 || w->K > INT32_MAX / 2 || tiles * chunks > INT64_MAX / 4096) return FTK_ERR_INVALID;
  a.codes = (const u32x4_t*)w->codes;
  a.scales = (const uint16_t*)w->scales;
  a.zeros = (const uint8_t*)w->zeros;
  a.N = (int)outputs;
  a.K = (int)w->K;
  a.tiles = (int)tiles;
  a.chunks = (int)chunks;
  a.half_scales = w->scale_type == FTK_W4_SCALE_FP16;
  subs = kW4Chunk / w->group;
  return FTK_OK;
}

}  // namespace

extern "C" {

int ftk_w4_project_bf16(const void* x, int64_t x_stride, const void* gamma, float eps, const ftk_w4* w,
                        const void* residual, void* y, int64_t M, void* stream) {
  W4Args a{};
  int subs = 1;
  bool gate_up = false;
  const int st = w4_args(w, a, subs, gate_up);
  if (st != FTK_OK) return st;
  if (!x || !y || M < 1 || M > kW4MaxRows || (M > 1 && x_stride < w->K)) return FTK_ERR_INVALID;
  if (gate_up && residual) return FTK_ERR_INVALID;
  if (!aligned(x, 2) || !aligned(y, 2) || !aligned(residual, 2)) return FTK_ERR_UNSUPPORTED;
  if (gamma) return FTK_ERR_UNSUPPORTED;
  a.x = (const uint16_t*)x;
  a.x_stride = x_stride;
  a.add = (const uint16_t*)residual;
  a.y = (uint16_t*)y;
  a.M = (int)M;
  return hip_status(launch_w4(a, subs, gate_up, reinterpret_cast<hipStream_t>(stream)));
}

int ftk_w4_dequantize_bf16(const ftk_w4* w, void* out, void* stream) {
  W4Args a{};
  int subs = 1;
  bool gate_up = false;
  const int st = w4_args(w, a, subs, gate_up);
  if (st != FTK_OK) return st;
  if (!out) return FTK_ERR_INVALID;
  if (!aligned(out, 2)) return FTK_ERR_UNSUPPORTED;
  if ((int64_t)a.tiles * a.chunks * 64 > (int64_t)INT32_MAX * 256) return FTK_ERR_INVALID;
  return hip_status(launch_w4_dequantize(a, subs, gate_up, (uint16_t*)out, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
