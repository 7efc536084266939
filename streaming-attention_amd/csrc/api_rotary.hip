// Entry points of the head norm with rotation (see include/streamattn.h) and their launches.
#include <cmath>

#include "api_common.hpp"
#include "head_rotary.hip"

using namespace sta_api;

namespace {

constexpr int kRotaryBlocks = 1024;  // workgroups over the positions, at most

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

sta::Rows rows_of(const void* p, const int64_t* strides, int es) {
  sta::Rows r{p, strides[0], strides[1], strides[2], 0};
  r.aligned = aligned16(p) && r.sb * es % 16 == 0 && r.sh * es % 16 == 0 && r.sn * es % 16 == 0;
  return r;
}

// The shape part of the arguments and the launch shape that goes with it.
struct Plan {
  int status, blocks;
  bool units;  // rows in 16-byte units (the row alignment still to be looked at)
};

Plan rotary_plan(sta::RotArgs& a, int dtype, int64_t batch, int heads, int kv_heads, int64_t n, int d, int rotary,
                 int interleaved) {
  a = sta::RotArgs{};
  if (!dtype_ok(dtype)) return {STA_ERR_DTYPE, 0, false};
  if (batch < 1 || heads < 0 || kv_heads < 0 || heads + kv_heads < 1 || n < 1 || d < 1 || rotary < 0 || rotary > d ||
      rotary % 2)
    return {STA_ERR_SHAPE, 0, false};
  if (d > kMaxD || batch > (int64_t(1) << 30) / n || heads > 16384 || kv_heads > 16384)
    return {STA_ERR_UNSUPPORTED, 0, false};
  a.heads[0] = heads;
  a.heads[1] = kv_heads;
  a.n = static_cast<int>(n);
  a.items = static_cast<int>(batch * n);
  a.d = d;
  a.r = rotary;
  a.inv_d = 1.f / d;
  a.interleaved = interleaved;
  const int e = dtype == STA_F32 ? 4 : 8;
  Plan p{STA_OK, 0, d % e == 0 && (interleaved || rotary / 2 % e == 0)};
  const int units = interleaved ? (d + 2 * e - 1) / (2 * e) : rotary / 2 / e + (d - rotary + 2 * e - 1) / (2 * e);
  a.lanes = 1;
  while (a.lanes < units) a.lanes *= 2;
  return p;
}

// Workgroups over the positions, and heads a workgroup walks over: as many as keep about four workgroups a compute
// unit, at most 16 (8 x 16 x 4096 x 64 bf16, forward / backward: 4 heads 78 / 117 us, 8 71 / 96, 16 62 / 98).
void rotary_grid(sta::RotArgs& a, Plan& p) {
  const int per = p.units ? 256 / a.lanes : 4;
  const int64_t blocks = (static_cast<int64_t>(a.items) + per - 1) / per;
  p.blocks = static_cast<int>(blocks < kRotaryBlocks ? blocks : kRotaryBlocks);
  const int64_t seg = static_cast<int64_t>(p.blocks) * (a.heads[0] + a.heads[1]) / 1024;
  a.per_seg = static_cast<int>(seg < 1 ? 1 : (seg > 16 ? 16 : seg));
  for (int i = 0; i < 2; ++i) a.segs[i] = (a.heads[i] + a.per_seg - 1) / a.per_seg;
}

template <int IN, bool BACK>
void launch(const sta::RotArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid(p.blocks, a.segs[0] + a.segs[1]);
  if (!p.units)
    hipLaunchKernelGGL((sta::head_rotary_any_kernel<IN, BACK>), grid, dim3(256), 0, s, a);
  else if (a.interleaved)
    hipLaunchKernelGGL((sta::head_rotary_kernel<IN, true, BACK>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((sta::head_rotary_kernel<IN, false, BACK>), grid, dim3(256), 0, s, a);
}

template <bool BACK>
void launch_typed(const sta::RotArgs& a, const Plan& p, int dtype, hipStream_t s) {
  if (dtype == STA_F32)
    launch<sta::F32, BACK>(a, p, s);
  else if (dtype == STA_BF16)
    launch<sta::BF16, BACK>(a, p, s);
  else
    launch<sta::F16, BACK>(a, p, s);
}

}  // namespace

extern "C" {

int sta_head_rotary(const void* q, const void* k, int dtype, int64_t batch, int heads, int kv_heads, int64_t n, int d,
                    const int64_t* strides, const void* q_weight, const void* k_weight, int weight_dtype,
                    const float* table, int64_t limit, int rotary, int interleaved, const void* positions,
                    int positions_64, int64_t position_stride_b, int64_t position_stride_n, float eps, void* q_out,
                    void* k_out, void* stream) {
  sta::RotArgs a;
  Plan p = rotary_plan(a, dtype, batch, heads, kv_heads, n, d, rotary, interleaved);
  if (p.status) return p.status;
  if ((heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)) || !strides || (!table && rotary) || limit < 1 ||
      limit > 0x7fffffff || !(eps >= 0.f) || !std::isfinite(eps) || !aligned16(q_out) || !aligned16(k_out))
    return STA_ERR_ARG;
  if (!dtype_ok(weight_dtype)) return STA_ERR_DTYPE;
  const int es = dtype == STA_F32 ? 4 : 2;
  a.x[0] = rows_of(q, strides, es);
  a.x[1] = rows_of(k, strides + 3, es);
  p.units = p.units && (!heads || a.x[0].aligned) && (!kv_heads || a.x[1].aligned);
  rotary_grid(a, p);
  a.y[0] = q_out;
  a.y[1] = k_out;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.wtype[0] = a.wtype[1] = weight_dtype;
  a.table = table;
  a.limit = static_cast<int>(limit);
  a.positions = positions;
  a.pos64 = positions_64;
  a.pos_sb = position_stride_b;
  a.pos_sn = position_stride_n;
  a.eps = eps;
  launch_typed<false>(a, p, dtype, static_cast<hipStream_t>(stream));
  return check_launch();
}

int64_t sta_head_rotary_backward_bytes(int64_t batch, int heads, int kv_heads, int64_t n, int d) {
  if (batch < 1 || heads < 0 || kv_heads < 0 || n < 1 || d < 1 || heads > 16384 || kv_heads > 16384) return -1;
  const int64_t rows = batch > kRotaryBlocks || n > kRotaryBlocks || batch * n > kRotaryBlocks ? kRotaryBlocks : batch * n;
  return 4 * rows * (heads + kv_heads) * d;
}

int sta_head_rotary_backward(const void* q_grad, const void* k_grad, const void* q, const void* k, int dtype,
                             int64_t batch, int heads, int kv_heads, int64_t n, int d, const int64_t* strides,
                             const void* q_weight, const void* k_weight, int weight_dtype, const float* table,
                             int64_t limit, int rotary, int interleaved, const void* positions, int positions_64,
                             int64_t position_stride_b, int64_t position_stride_n, float eps, void* dq, void* dk,
                             void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  sta::RotArgs a;
  Plan p = rotary_plan(a, dtype, batch, heads, kv_heads, n, d, rotary, interleaved);
  if (p.status) return p.status;
  if ((heads && (!q || !q_grad || !dq)) || (kv_heads && (!k || !k_grad || !dk)) || !strides || (!table && rotary) || limit < 1 ||
      limit > 0x7fffffff || !(eps >= 0.f) || !std::isfinite(eps) || !aligned16(dq) || !aligned16(dk) || !workspace ||
      !aligned16(workspace))
    return STA_ERR_ARG;
  if (!dtype_ok(weight_dtype)) return STA_ERR_DTYPE;
  if (workspace_bytes < sta_head_rotary_backward_bytes(batch, heads, kv_heads, n, d)) return STA_ERR_SCRATCH;
  const int es = dtype == STA_F32 ? 4 : 2;
  a.x[0] = rows_of(q, strides, es);
  a.x[1] = rows_of(k, strides + 3, es);
  a.g[0] = rows_of(q_grad, strides + 6, es);
  a.g[1] = rows_of(k_grad, strides + 9, es);
  for (int i = 0; i < 2; ++i)
    p.units = p.units && (!a.heads[i] || (a.x[i].aligned && a.g[i].aligned));
  rotary_grid(a, p);
  a.y[0] = dq;
  a.y[1] = dk;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.wtype[0] = a.wtype[1] = weight_dtype;
  a.table = table;
  a.limit = static_cast<int>(limit);
  a.positions = positions;
  a.pos64 = positions_64;
  a.pos_sb = position_stride_b;
  a.pos_sn = position_stride_n;
  a.eps = eps;
  float* part = static_cast<float*>(workspace);
  const int rows[2] = {a.segs[0] * p.blocks, a.segs[1] * p.blocks};
  a.part[0] = dq_weight && heads ? part : nullptr;
  a.part[1] = dk_weight && kv_heads ? part + static_cast<int64_t>(rows[0]) * d : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  launch_typed<true>(a, p, dtype, s);
  if (a.part[0] || a.part[1])
    hipLaunchKernelGGL(sta::head_rotary_weight_kernel, dim3((d + 3) / 4, 2), dim3(256), 0, s, a.part[0], a.part[1],
                       rows[0], rows[1], d, dq_weight, dk_weight, weight_dtype);
  return check_launch();
}

}  // extern "C"
