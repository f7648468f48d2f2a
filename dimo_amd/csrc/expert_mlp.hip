// The expert block as one call per direction: routing, grouping, both products, the weighted sum, and their gradients --
// the launches of experts.hip and grouped.hip in order on one stream, intermediates in a workspace of the caller's.  (One
// by one from Python the same launches cost more host time than a step of 4096 rows costs the GPU.)
//   forward   w, e = route(logits);  h = act(W1 x[rows] + b1);  y = W2 h + b2;  out = x + sum_j w_j y[position_j]
//   backward  gy = w g, gw = <g, y>;  gz = (gy W2) act';  gx = g + sum_j (gz W1)[position_j];  g_logits from gw
// h, z, y, gy, gz and gx of the places have the tensors' type: each is an operand of the next product in that type (y and gx:
// read once, by a sum), and 32 bits would double their traffic and take the products off the 16-bit instructions.  Against
// one rounding at the end the weight gradients' error is 1.7 times as large (bf16, rms: 0.0029 of the value, 0.0017).
#include <hip/hip_runtime.h>

#include "numeric.hpp"

using namespace dimo;

namespace {

struct BlockLayout {
  size_t weights, experts, offsets, position, rows, h, z, y, bytes;
  int64_t S;
  __host__ BlockLayout(const dimo_expert_mlp_desc &d, bool keep) {
    S = (int64_t)d.T * d.k;
    const size_t b = dtype_bytes(d.dtype), s = (size_t)S;
    size_t o = 0;
    weights = o, o = align_up(o + s * sizeof(float));
    experts = o, o = align_up(o + s * sizeof(int32_t));
    offsets = o, o = align_up(o + ((size_t)d.E + 1) * sizeof(int32_t));
    position = o, o = align_up(o + s * sizeof(int32_t));
    rows = o, o = align_up(o + s * sizeof(int32_t));
    // h also holds the grouping's counts before it is written
    const size_t counts = dimo_group_rows_workspace_bytes(S, d.E), hidden = s * d.F * b;
    h = o, o = align_up(o + (hidden > counts ? hidden : counts));
    z = o, o = align_up(o + (keep && d.act == DIMO_ACT_SILU ? hidden : 0));
    y = o, o = align_up(o + s * d.K * b);
    bytes = o;
  }
};
struct ScratchLayout {
  size_t gw, gy, gz, gxs, partial, partial_bytes, bytes;
  __host__ explicit ScratchLayout(const dimo_expert_mlp_desc &d) {
    const size_t b = dtype_bytes(d.dtype), s = (size_t)d.T * d.k;
    size_t o = 0;
    gw = o, o = align_up(o + s * sizeof(float));
    gy = o, o = align_up(o + s * d.K * b);
    gz = o, o = align_up(o + s * d.F * b);
    gxs = o, o = align_up(o + s * d.K * b);
    const size_t p1 = dimo_grouped_linear_wgrad_workspace_bytes(d.dtype, (int)s, d.E, d.K, d.F);
    const size_t p2 = dimo_grouped_linear_wgrad_workspace_bytes(d.dtype, (int)s, d.E, d.F, d.K);
    partial_bytes = p1 > p2 ? p1 : p2;
    partial = o, o = align_up(o + partial_bytes);
    bytes = o;
  }
};

bool bad(const dimo_expert_mlp_desc *d) {
  return !d || !known_dtype(d->dtype) || d->T < 0 || d->K < 1 || d->F < 1 || d->E < 1 || d->E > DIMO_MAX_EXPERTS || d->k < 1 ||
         d->k > d->E || (int64_t)d->T * d->k > DIMO_MAX_SIZE || d->K > DIMO_MAX_SIZE || d->F > DIMO_MAX_SIZE || d->act < DIMO_ACT_NONE || d->act > DIMO_ACT_SILU ||
         d->ld_x < d->K || d->ld_logits < d->E;
}

}  // namespace

extern "C" size_t dimo_expert_mlp_workspace_bytes(const dimo_expert_mlp_desc *d, int keep) {
  return bad(d) ? 0 : BlockLayout(*d, keep != 0).bytes;
}
extern "C" size_t dimo_expert_mlp_scratch_bytes(const dimo_expert_mlp_desc *d) { return bad(d) ? 0 : ScratchLayout(*d).bytes; }

extern "C" int dimo_expert_mlp_forward(const dimo_expert_mlp_desc *d, int keep, void *out, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  if (bad(d) || (d->T > 0 && (!d->x || !d->logits || !d->w1 || !d->w2 || !out))) return DIMO_E_ARG;
  const BlockLayout L(*d, keep != 0);
  if (!workspace || !aligned16(workspace) || workspace_bytes < L.bytes) return DIMO_E_WORKSPACE;
  float *weights = at<float>(workspace, L.weights);
  int32_t *experts = at<int32_t>(workspace, L.experts), *offsets = at<int32_t>(workspace, L.offsets);
  int32_t *position = at<int32_t>(workspace, L.position), *rows = at<int32_t>(workspace, L.rows);
  void *h = at<char>(workspace, L.h), *y = at<char>(workspace, L.y);
  void *z = keep && d->act == DIMO_ACT_SILU ? at<char>(workspace, L.z) : nullptr;
  const int R = (int)L.S;
  int rc = dimo_route_topk_forward(d->T, d->E, d->k, d->dtype, d->logits, d->ld_logits, d->row_mask, d->normalize, weights,
                                   experts, nullptr, nullptr, 0, stream);
  if (!rc)
    rc = dimo_group_rows(L.S, d->E, d->k, experts, offsets, nullptr, position, rows, h,
                         dimo_group_rows_workspace_bytes(L.S, d->E), stream);
  if (!rc)
    rc = dimo_grouped_linear_forward(d->dtype, R, d->E, d->K, d->F, d->x, d->ld_x, rows, offsets, d->w1, d->b1, d->act, h, z,
                                     stream);
  if (!rc) rc = dimo_grouped_linear_forward(d->dtype, R, d->E, d->F, d->K, h, d->F, nullptr, offsets, d->w2, d->b2,
                                            DIMO_ACT_NONE, y, nullptr, stream);
  if (!rc) rc = dimo_combine_rows_forward(d->T, d->k, d->K, L.S, d->dtype, y, d->K, weights, position, d->x, d->ld_x, out, stream);
  return rc;
}

extern "C" int dimo_expert_mlp_backward(const dimo_expert_mlp_desc *d, const void *g_out, int64_t ld_g,
                                        const void *workspace, void *scratch, size_t scratch_bytes, void *g_x,
                                        void *g_logits, void *g_w1, void *g_b1, void *g_w2, void *g_b2, void *stream) {
  if (bad(d) || ld_g < d->K || (g_b1 && !g_w1) || (g_b2 && !g_w2)) return DIMO_E_ARG;
  if (!workspace || (d->T > 0 && (!g_out || !d->x || !d->logits || !d->w1 || !d->w2))) return DIMO_E_ARG;
  const BlockLayout L(*d, true);
  const ScratchLayout P(*d);
  if (d->T > 0 && (!scratch || !aligned16(scratch) || scratch_bytes < P.bytes)) return DIMO_E_WORKSPACE;
  const int R = (int)L.S;
  const float *weights = at<float>(workspace, L.weights);
  const int32_t *experts = at<int32_t>(workspace, L.experts), *offsets = at<int32_t>(workspace, L.offsets);
  const int32_t *position = at<int32_t>(workspace, L.position), *rows = at<int32_t>(workspace, L.rows);
  const void *h = at<char>(workspace, L.h), *y = at<char>(workspace, L.y);
  const void *saved = d->act == DIMO_ACT_SILU ? at<char>(workspace, L.z) : at<char>(workspace, L.h);
  float *gw = at<float>(scratch, P.gw);
  void *gy = at<char>(scratch, P.gy), *gz = at<char>(scratch, P.gz), *gxs = at<char>(scratch, P.gxs);
  void *partial = at<char>(scratch, P.partial);
  int rc = dimo_combine_rows_backward(d->T, d->k, d->K, L.S, d->E, d->dtype, g_out, ld_g, y, d->K, weights, position, offsets,
                                      gy, g_logits ? gw : nullptr, stream);
  if (!rc && g_logits)
    rc = dimo_route_topk_backward(d->T, d->E, d->k, d->dtype, d->logits, d->ld_logits, d->row_mask, d->normalize, weights,
                                  experts, gw, nullptr, g_logits, stream);
  if (!rc && g_w2)
    rc = dimo_grouped_linear_wgrad(d->dtype, R, d->E, d->F, d->K, gy, h, d->F, nullptr, offsets, g_w2, g_b2, partial,
                                   P.partial_bytes, stream);
  if (!rc && (g_w1 || g_x))
    rc = dimo_grouped_linear_dgrad(d->dtype, R, d->E, d->F, d->K, gy, offsets, d->w2, d->act, saved, gz, stream);
  if (!rc && g_w1)
    rc = dimo_grouped_linear_wgrad(d->dtype, R, d->E, d->K, d->F, gz, d->x, d->ld_x, rows, offsets, g_w1, g_b1, partial,
                                   P.partial_bytes, stream);
  if (!rc && g_x) rc = dimo_grouped_linear_dgrad(d->dtype, R, d->E, d->K, d->F, gz, offsets, d->w1, DIMO_ACT_NONE, nullptr, gxs, stream);
  if (!rc && g_x) rc = dimo_combine_rows_forward(d->T, d->k, d->K, L.S, d->dtype, gxs, d->K, nullptr, position, g_out, ld_g, g_x, stream);
  return rc;
}
