// Gradients of the masked attention: checks, cutting into tasks and C entries (kernels:
// masked_attention_bwd.h).
#include "masked_attention_bwd.h"

namespace vgo {
namespace masked {

GradPlan grad_plan(const vgo_masked_attn* p, int dtype) {
  GradPlan r{};
  r.query_tiles = static_cast<int>(tiles_of(p->n_query)), r.key_tiles = static_cast<int>(tiles_of(p->n_key));
  const int64_t keys = dtype != VGO_F32 && p->head_dim == 128 ? KeyLds<bf16_t, 128>::kBlock : KeyLds<bf16_t, 64>::kBlock;
  r.key_blocks = static_cast<int>((p->n_key + keys - 1) / keys);
  r.row_blocks = static_cast<int>((p->n_query + kRowBlock - 1) / kRowBlock);
  // Times of a tile and work-groups a CU holds, as splits_of() counts them, from 16 heads of 8,232 x 8,232: dK and
  // dV 790 us (64 channels), 1,539 (128), dQ 494 and 909; and 2,058 x 2,058 in fp32.
  const bool wide = p->head_dim == 128, f32 = dtype == VGO_F32;
  const double key_us = f32 ? (wide ? 17.4 : 8.7) : wide ? 4.0 : 1.1, row_us = f32 ? (wide ? 12.8 : 6.4) : wide ? 1.26 : 0.68;
  const int64_t tasks = p->batch * p->kv_heads * r.key_blocks, rows = p->batch * p->heads * r.row_blocks;
  const int units = static_cast<int>(std::min<int64_t>(p->heads / p->kv_heads * std::max(1, r.query_tiles), 1 << 20));
  const double key_bytes = 16.0 * p->batch * p->kv_heads * p->n_key * p->head_dim;
  const double row_bytes = 8.0 * p->batch * p->heads * p->n_query * p->head_dim;
  r.splits = tasks == 0 ? 1 : std::min(32, splits_of(p, tasks, units, f32 || wide ? 1 : 3, key_us, key_bytes / 7e6));
  r.row_splits = rows == 0 || r.key_tiles == 0 ? 1 : std::min(32, splits_of(p, rows, r.key_tiles, f32 ? 1 : wide ? 2 : 3, row_us, row_bytes / 7e6));
  r.key_tasks = tasks * r.splits, r.row_tasks = rows * r.row_splits;
  return r;
}

GradPieces grad_pieces(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, const GradPlan& plan) {
  GradPieces r{};
  size_t at = info_bytes(p);
  const auto take = [&](size_t bytes) {
    const size_t was = at;
    at += (bytes + 15) & ~static_cast<size_t>(15);
    return was;
  };
  const size_t rows = static_cast<size_t>(p->batch) * p->heads;
  r.delta = take(rows * p->n_query * 4);
  r.marks = take(rows * plan.query_tiles);
  const size_t keys = static_cast<size_t>(plan.splits) * p->batch * p->kv_heads * p->n_key;
  r.kv = take(plan.splits > 1 && g->dk ? keys * 2 * p->head_dim * 4 : 0);
  r.q = take(plan.row_splits > 1 && g->dq ? plan.row_splits * rows * p->n_query * p->head_dim * 4 : 0);
  r.mass = take(g->d_log_mass ? keys * 4 : 0);
  const size_t parts = static_cast<size_t>(plan.row_splits) * p->batch * plan.row_blocks * p->heads;
  r.slopes = take(g->d_slopes ? parts * 4 : 0);
  r.table = take(g->d_table ? parts * p->n_buckets * 4 : 0);
  r.bytes = at;
  return r;
}

namespace {

int check_grads(const vgo_masked_attn* p, const vgo_masked_attn_grads* g, int dtype) {
  const int status = check_problem(p, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(g, "masked_attn_grad: null gradients");
  VGO_REQUIRE(!g->dk == !g->dv || p->n_key == 0, "masked_attn_grad: dk and dv go together");
  VGO_REQUIRE(!g->d_log_mass || p->log_mass, "masked_attn_grad: no log_mass to take the gradient of");
  VGO_REQUIRE(!g->d_slopes || p->slopes, "masked_attn_grad: no slopes to take the gradient of");
  VGO_REQUIRE(!g->d_table || p->bucket_table, "masked_attn_grad: no table to take the gradient of");
  const GradPlan plan = grad_plan(p, dtype);
  VGO_REQUIRE(fits_grid(p->batch * p->heads * plan.query_tiles, 256) && fits_grid(plan.key_tasks, 512) &&
                  fits_grid(plan.row_tasks, 256),
              "masked_attn_grad: too many rows");
  return VGO_OK;
}

}  // namespace
}  // namespace masked
}  // namespace vgo

extern "C" int vgo_masked_attn_grad_workspace(const vgo_masked_attn* problem, const vgo_masked_attn_grads* grads,
                                              int dtype, size_t* bytes) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_grads(problem, grads, dtype);
  if (status != VGO_OK) return status;
  VGO_REQUIRE(bytes, "masked_attn_grad: null pointer");
  *bytes = grad_pieces(problem, grads, grad_plan(problem, dtype)).bytes;
  return VGO_OK;
}

extern "C" int vgo_masked_attn_grad(const vgo_masked_attn* problem, const vgo_masked_attn_grads* grads, int dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace vgo;
  using namespace vgo::masked;
  const int status = check_grads(problem, grads, dtype);
  if (status != VGO_OK) return status;
  const vgo_masked_attn* p = problem;
  const vgo_masked_attn_grads* g = grads;
  if (p->batch > 0 && p->n_query > 0)
    VGO_REQUIRE(g->out && g->grad_out && g->lse && aligned(g->out, 16) && aligned(g->grad_out, 16) &&
                    strides_fit(g->out_stride, p->head_dim, dtype) &&
                    strides_fit(g->grad_out_stride, p->head_dim, dtype),
                "masked_attn_grad: out and grad_out must be 16-byte aligned, with strides of whole 16 bytes");
  VGO_REQUIRE(aligned(g->out_rest, 16) && (!g->out_rest || dtype != VGO_F32),
              "masked_attn_grad: out_rest must be 16-byte aligned, and of a 16-bit type");
  VGO_REQUIRE((!g->dq || (aligned(g->dq, 16) && strides_fit(g->dq_stride, p->head_dim, dtype))) &&
                  (!g->dk || (aligned(g->dk, 16) && aligned(g->dv, 16) &&
                              strides_fit(g->dk_stride, p->head_dim, dtype) &&
                              strides_fit(g->dv_stride, p->head_dim, dtype))),
              "masked_attn_grad: dq, dk and dv must be 16-byte aligned, with strides of whole 16 bytes");
  const GradPlan plan = grad_plan(p, dtype);
  const size_t need = grad_pieces(p, g, plan).bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(VGO_EWORKSPACE, "masked_attn_grad: workspace of " + std::to_string(need) + " bytes needed");
  char* ws = static_cast<char*>(workspace);
  const hipStream_t s = as_stream(stream);
  if (dtype == VGO_BF16) return run_grad<bf16_t>(p, g, plan, ws, s);
  if (dtype == VGO_F16) return run_grad<f16_t>(p, g, plan, ws, s);
  return run_grad<float>(p, g, plan, ws, s);
}
