// policy_abi.cuh — the C ABI of drawing, the policy loss and gradient clipping
// (kc_draw*, kc_policy_loss, kc_set_policy, kc_clip_*): argument checks, host
// staging, and the launchers of policy.cu.
#pragma once

namespace {

static_assert(kc::pol::kMaxRow == KC_MAX_ROW, "the header's longest row is the kernels'");
static_assert(kc::kF32 == KC_DTYPE_F32 && kc::kF16 == KC_DTYPE_F16 && kc::kBF16 == KC_DTYPE_BF16 &&
              kc::kF64 == KC_DTYPE_F64, "element types");

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// The limits of a policy; row arrays are the caller's to fill.
kc_status check_sampling(kc_handle* h, const kc_sampling* s, bool learns) {
  if (!s) return fail(h, KC_ERR_INVALID_ARG, "sampling is null");
  if (!s->row_temperature && (!(s->temperature >= 0.0f) || !std::isfinite(s->temperature)))
    return fail(h, KC_ERR_INVALID_ARG, "temperature must be a finite number, 0 or above");
  if (learns && !s->row_temperature && s->temperature == 0.0f)
    return fail(h, KC_ERR_INVALID_ARG, "a policy at temperature 0 has no gradient");
  if (!s->row_top_p && !(s->top_p >= 0.0f)) return fail(h, KC_ERR_INVALID_ARG, "top_p must be a number, 0 or above");
  if (!s->row_min_p && !(s->min_p >= 0.0f && s->min_p <= 1.0f))
    return fail(h, KC_ERR_INVALID_ARG, "min_p must lie in [0, 1]");
  if (!aligned(s->row_temperature, 4) || !aligned(s->row_top_k, 4) || !aligned(s->row_top_p, 4) ||
      !aligned(s->row_min_p, 4))
    return fail(h, KC_ERR_INVALID_ARG, "the row limits must be 4-byte aligned");
  return KC_OK;
}

kc::pol::CutArg cut_arg(const kc_sampling* s) {
  return kc::pol::CutArg{s->temperature > 0.0f ? 1.0 / double(s->temperature) : 0.0, s->temperature, s->top_k, s->top_p, s->min_p,
                         s->row_temperature, s->row_top_k, s->row_top_p, s->row_min_p};
}

// Checks a rows view and fills in its defaults; *out_pitch likewise.
kc_status check_rows(kc_handle* h, const kc_rows_view* v, kc::pol::RowsArg* r, uint64_t* out_pitch) {
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the rows view is null");
  if (v->dtype != KC_DTYPE_F32 && v->dtype != KC_DTYPE_F16 && v->dtype != KC_DTYPE_BF16)
    return fail(h, KC_ERR_INVALID_ARG, "rows hold f32, f16 or bf16 values");
  if (v->kind != KC_ROWS_SCORES && v->kind != KC_ROWS_P)
    return fail(h, KC_ERR_INVALID_ARG, "unknown kind of rows");
  if (v->kind == KC_ROWS_P && v->dtype != KC_DTYPE_F32)
    return fail(h, KC_ERR_INVALID_ARG, "probabilities are f32");
  r->values = v->values;
  r->q_off = v->q_off;
  r->p_off = v->p_off;
  r->rows = v->rows;
  r->frames = v->frames;
  r->row_len = v->frames && v->row_len == 0 ? KC_MAX_BANK : v->row_len;
  r->pitch = v->row_pitch ? v->row_pitch : v->row_len;
  r->kind = v->kind;
  if (v->rows > 0x7fffffffu) return fail(h, KC_ERR_CAPACITY, "a call takes at most 2147483647 rows");
  if (r->row_len > KC_MAX_ROW) return fail(h, KC_ERR_CAPACITY, "a row is longer than KC_MAX_ROW");
  if (v->frames) {
    if (!v->p_off || !aligned(v->p_off, 8) || !aligned(v->q_off, 8))
      return fail(h, KC_ERR_INVALID_ARG, "a batch of rows needs p_off, and its offsets 8-byte aligned");
  } else {
    if (r->pitch < r->row_len) return fail(h, KC_ERR_INVALID_ARG, "row_pitch is smaller than row_len");
    if (*out_pitch == 0) *out_pitch = r->row_len;
    if (*out_pitch < r->row_len) return fail(h, KC_ERR_INVALID_ARG, "an output's pitch is smaller than row_len");
  }
  if (v->rows && (v->frames || v->row_len) && !v->values) return fail(h, KC_ERR_INVALID_ARG, "the rows have no values");
  if (!aligned(v->values, v->dtype == KC_DTYPE_F32 ? 4 : 2))
    return fail(h, KC_ERR_INVALID_ARG, "the rows' values must be aligned to their type");
  return KC_OK;
}

kc_status draw_rows(kc_handle* h, const kc_rows_view* v, const kc_sampling* s, const double* uniforms,
                    const kc_draw_out* out) {
  kc::pol::DrawArg a{};
  if (!out || (!out->index && !out->kept && !out->logp && !out->p))
    return fail(h, KC_ERR_INVALID_ARG, "a draw needs at least one output");
  a.out_pitch = out->p_pitch;
  KC_CHECK(check_rows(h, v, &a.r, &a.out_pitch));
  KC_CHECK(check_sampling(h, s, false));
  if (!aligned(uniforms, 8)) return fail(h, KC_ERR_INVALID_ARG, "uniforms must be 8-byte aligned");
  if (!aligned(out->index, 4) || !aligned(out->kept, 4) || !aligned(out->logp, 4) || !aligned(out->p, 4))
    return fail(h, KC_ERR_INVALID_ARG, "a draw's outputs must be 4-byte aligned");
  a.c = cut_arg(s);
  a.uniforms = uniforms;
  a.index = out->index;
  a.kept = out->kept;
  a.logp = out->logp;
  a.p = out->p;
  if (a.p && a.p == v->values && (v->dtype != KC_DTYPE_F32 || (!v->frames && a.out_pitch != a.r.pitch)))
    return fail(h, KC_ERR_INVALID_ARG, "p over the values needs f32 rows and one pitch");
  KC_TRY(kc::pol::launch_draw(a, v->dtype, h->sms, h->stream, &h->launches), "draw launch");
  return KC_OK;
}

// A host draw: the limits and uniforms staged, the draw of `rows` device rows,
// the results read back.
kc_status draw_host(kc_handle* h, const kc_rows_view& v, uint64_t entries, const kc_sampling* sampling,
                    const double* uniforms, const kc_draw_out* out) {
  KC_CHECK(check_sampling(h, sampling, false));
  DrawWs& dw = h->dw;
  kc_sampling s = *sampling;
  const uint64_t n = v.rows;
  KC_CHECK(stage(h, dw.temperature, s.row_temperature, s.row_temperature ? n : 0));
  KC_CHECK(stage(h, dw.top_k, s.row_top_k, s.row_top_k ? n : 0));
  KC_CHECK(stage(h, dw.top_p, s.row_top_p, s.row_top_p ? n : 0));
  KC_CHECK(stage(h, dw.min_p, s.row_min_p, s.row_min_p ? n : 0));
  if (s.row_temperature) s.row_temperature = P<float>(dw.temperature);
  if (s.row_top_k) s.row_top_k = P<uint32_t>(dw.top_k);
  if (s.row_top_p) s.row_top_p = P<float>(dw.top_p);
  if (s.row_min_p) s.row_min_p = P<float>(dw.min_p);
  if (uniforms) KC_CHECK(stage(h, dw.uniforms, uniforms, n));
  kc_draw_out d{};
  auto want = [&](DevBuf& b, uint64_t bytes, bool asked) -> cudaError_t {
    return asked ? ensure(h, b, bytes) : cudaSuccess;
  };
  KC_TRY(want(dw.index, n * 4, out->index), "workspace");
  KC_TRY(want(dw.kept, n * 4, out->kept), "workspace");
  KC_TRY(want(dw.logp, n * 4, out->logp), "workspace");
  KC_TRY(want(dw.p, entries * 4, out->p), "workspace");
  if (out->index) d.index = P<uint32_t>(dw.index);
  if (out->kept) d.kept = P<uint32_t>(dw.kept);
  if (out->logp) d.logp = P<float>(dw.logp);
  if (out->p) d.p = P<float>(dw.p);
  KC_CHECK(draw_rows(h, &v, &s, uniforms ? P<double>(dw.uniforms) : nullptr, &d));
  auto get = [&](void* dst, const DevBuf& src, uint64_t bytes) -> cudaError_t {
    return dst && bytes ? cudaMemcpyAsync(dst, src.p, bytes, cudaMemcpyDeviceToHost, h->stream) : cudaSuccess;
  };
  KC_TRY(get(out->index, dw.index, n * 4), "readback");
  KC_TRY(get(out->kept, dw.kept, n * 4), "readback");
  KC_TRY(get(out->logp, dw.logp, n * 4), "readback");
  KC_TRY(get(out->p, dw.p, entries * 4), "readback");
  KC_TRY(wait_stream(h), "draw");
  return KC_OK;
}

// The backward's policy of the batch in ws: pi of every p row into `pi`.
kc_status policy_rows(kc_handle* h, Workspace& ws, uint32_t frames, const kc::FrameTotals& tot, float* pi) {
  kc_rows_view v{ws.p.p, P<uint64_t>(ws.q_off), P<uint64_t>(ws.p_off), uint32_t(tot.q), frames,
                 tot.max_r ? tot.max_r : 1u, 0, KC_DTYPE_F32, KC_ROWS_P};
  kc_draw_out out{};
  out.p = pi;
  return draw_rows(h, &v, &h->policy, nullptr, &out);
}

}  // namespace

extern "C" {

kc_status kc_draw_device(kc_handle* h, const kc_rows_view* rows, const kc_sampling* sampling, const double* uniforms,
                         const kc_draw_out* out) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  return draw_rows(h, rows, sampling, uniforms, out);
}

kc_status kc_draw(kc_handle* h, uint32_t q, uint32_t r, const float* p, const kc_sampling* sampling,
                  const double* uniforms, const kc_draw_out* out) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  if (!out || (uint64_t(q) * r && !p)) return fail(h, KC_ERR_INVALID_ARG, "draw arguments are incomplete");
  if (r > KC_MAX_BANK) return fail(h, KC_ERR_CAPACITY, "bank records exceed capacity");
  if (out->p_pitch && out->p_pitch != r)
    return fail(h, KC_ERR_INVALID_ARG, "a host draw's p is laid out like its input");
  const uint64_t n = uint64_t(q) * r;
  KC_CHECK(stage(h, h->dw.values, p, n));
  const kc_rows_view v{h->dw.values.p, nullptr, nullptr, q, 0, r, 0, KC_DTYPE_F32, KC_ROWS_P};
  return draw_host(h, v, n, sampling, uniforms, out);
}

kc_status kc_draw_batch(kc_handle* h, const kc_sampling* sampling, const double* uniforms, const kc_draw_out* out) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  if (!out) return fail(h, KC_ERR_INVALID_ARG, "draw arguments are incomplete");
  if (h->resident_epoch == 0 || h->resident_epoch != h->ws_epoch)
    return fail(h, KC_ERR_INVALID_ARG,
                "no batch is resident: run kc_forward_batch first (another call on this handle, or a weight "
                "change, since then releases it)");
  const kc::FrameTotals tot = h->resident_tot;
  if ((out->p && out->p_capacity < tot.p) || ((out->index || out->kept || out->logp) && out->q_capacity < tot.q))
    return fail(h, KC_ERR_CAPACITY, "output buffers are smaller than the batch's p / index");
  Workspace& ws = h->ws;
  const kc_rows_view v{ws.p.p, P<uint64_t>(ws.q_off), P<uint64_t>(ws.p_off), uint32_t(tot.q), h->resident_frames,
                       tot.max_r ? tot.max_r : 1u, 0, KC_DTYPE_F32, KC_ROWS_P};
  return draw_host(h, v, tot.p, sampling, uniforms, out);
}

kc_status kc_policy_loss(kc_handle* h, const kc_rows_view* rows, const kc_sampling* sampling,
                         const kc_policy_loss_view* loss) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  kc::pol::LossArg a{};
  if (!loss || (!loss->loss && !loss->logp && !loss->entropy && !loss->grad))
    return fail(h, KC_ERR_INVALID_ARG, "a policy loss needs at least one output");
  a.out_pitch = loss->grad_pitch;
  KC_CHECK(check_rows(h, rows, &a.r, &a.out_pitch));
  KC_CHECK(check_sampling(h, sampling, true));
  if (rows->kind != KC_ROWS_SCORES) return fail(h, KC_ERR_INVALID_ARG, "a policy loss is taken from scores");
  if (rows->rows && (!loss->actions || !loss->advantage))
    return fail(h, KC_ERR_INVALID_ARG, "a policy loss needs actions and advantages");
  if (!std::isfinite(loss->entropy_coef)) return fail(h, KC_ERR_INVALID_ARG, "entropy_coef must be finite");
  if (!aligned(loss->actions, 4) || !aligned(loss->advantage, 4) || !aligned(loss->row_weight, 4) ||
      !aligned(loss->loss, 4) || !aligned(loss->logp, 4) || !aligned(loss->entropy, 4) ||
      !aligned(loss->grad, rows->dtype == KC_DTYPE_F32 ? 4 : 2))
    return fail(h, KC_ERR_INVALID_ARG, "a policy loss's arrays must be aligned to their type");
  a.c = cut_arg(sampling);
  a.actions = loss->actions;
  a.advantage = loss->advantage;
  a.row_weight = loss->row_weight;
  a.beta = loss->entropy_coef;
  a.loss = loss->loss;
  a.logp = loss->logp;
  a.entropy = loss->entropy;
  a.grad = loss->grad;
  if (a.grad && a.grad == rows->values && !rows->frames && a.out_pitch != a.r.pitch)
    return fail(h, KC_ERR_INVALID_ARG, "a gradient over the scores needs one pitch");
  KC_TRY(kc::pol::launch_policy_loss(a, rows->dtype, h->sms, h->stream, &h->launches), "policy loss launch");
  return KC_OK;
}

kc_status kc_set_policy(kc_handle* h, const kc_sampling* sampling) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  if (!sampling) {
    h->policy_on = false;
    return KC_OK;
  }
  if (sampling->row_temperature || sampling->row_top_k || sampling->row_top_p || sampling->row_min_p)
    return fail(h, KC_ERR_INVALID_ARG, "the backward's policy takes scalar limits only");
  KC_CHECK(check_sampling(h, sampling, true));
  h->policy = *sampling;
  h->policy_on = true;
  return KC_OK;
}

uint64_t kc_clip_workspace(uint64_t count) { return kc::clip::workspace_doubles(count ? count : 1) * 8; }

kc_status kc_clip_grads(kc_handle* h, const kc_grad_view* grads, uint64_t count, double max_norm, void* workspace,
                        uint64_t workspace_bytes, double* result) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  if ((count && !grads) || !workspace || !result)
    return fail(h, KC_ERR_INVALID_ARG, "clip arguments are incomplete");
  if (!(max_norm >= 0.0)) return fail(h, KC_ERR_INVALID_ARG, "max_norm must be a number, 0 or above");
  if (!aligned(workspace, 8) || !aligned(result, 8))
    return fail(h, KC_ERR_INVALID_ARG, "the workspace and the result must be 8-byte aligned");
  if (count > (1u << 20)) return fail(h, KC_ERR_CAPACITY, "a gradient list holds at most 1048576 tensors");
  if (workspace_bytes < kc_clip_workspace(count))
    return fail(h, KC_ERR_CAPACITY, "the workspace is smaller than kc_clip_workspace(count)");
  try {
    h->clip_list.clear();
    h->clip_list.reserve(count);
    for (uint64_t i = 0; i < count; i++) {
      const kc_grad_view& g = grads[i];
      if (g.dtype < KC_DTYPE_F32 || g.dtype > KC_DTYPE_F64)
        return fail(h, KC_ERR_INVALID_ARG, "gradients are f32, f16, bf16 or f64");
      const uintptr_t size = g.dtype == KC_DTYPE_F32 ? 4 : g.dtype == KC_DTYPE_F64 ? 8 : 2;
      if (g.n && !g.in) return fail(h, KC_ERR_INVALID_ARG, "a gradient is null");
      if (g.n >> 40) return fail(h, KC_ERR_CAPACITY, "a gradient holds more than 2^40 elements");
      if (!aligned(g.in, size) || !aligned(g.out, size))
        return fail(h, KC_ERR_INVALID_ARG, "a gradient must be aligned to its type");
      if (!std::isfinite(g.weight)) return fail(h, KC_ERR_INVALID_ARG, "a gradient's weight must be finite");
      h->clip_list.push_back(kc::clip::Tensor{g.in, g.out, g.n, g.weight, g.dtype, 0u});
    }
  } catch (const std::bad_alloc&) {
    return fail(h, KC_ERR_CAPACITY, "out of host memory for the gradient list");
  }
  KC_TRY(kc::clip::launch_clip(h->clip_list.data(), count, max_norm, static_cast<double*>(workspace), result, h->sms,
                               h->stream, &h->launches), "clip launch");
  return KC_OK;
}

}  // extern "C"
