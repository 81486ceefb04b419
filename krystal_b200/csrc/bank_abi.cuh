// bank_abi.cuh — kc_bank_turn: a turn of many sessions whose banks lie in caches
// (cache_abi.cuh). The turn's records are encoded as a batch's are; what the mixer
// blocks and the selector read of the bank records among them is appended to the
// sessions' caches; the questions among them are answered over all that these hold.
#pragma once

namespace {

// Score offsets of dense rows: frame f's questions begin at question q_off[f].
__global__ void k_turn_offsets(const uint64_t* q_off, uint32_t frames, uint64_t row, uint64_t* off) {
  const uint32_t f = blockIdx.x * blockDim.x + threadIdx.x;
  if (f <= frames) off[f] = q_off[f] * row;
}

// qstate += the attention's output.
__global__ void k_turn_add(float4* x, const float4* y, uint64_t n) {
  const uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float4 a = x[i];
  const float4 b = y[i];
  a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  x[i] = a;
}

struct Bank {
  std::vector<kc::cache::Store> mixer;
  kc::cache::Store selector;
  kc::cache::Table table;
};

kc_status check_bank(kc_handle* h, const kc_bank_view* v, uint32_t frames, Bank* b) {
  if (!v || (h->d.mix && !v->mixer)) return fail(h, KC_ERR_INVALID_ARG, "the bank view is incomplete");
  KC_CHECK(check_table(h, &v->table, &b->table));
  if (v->table.sequences != frames) return fail(h, KC_ERR_INVALID_ARG, "a turn's table has a sequence a frame");
  for (uint32_t i = 0; i < h->d.mix; i++) {
    b->mixer.emplace_back();
    KC_CHECK(check_cache(h, v->mixer + i, &b->mixer.back()));
    if (b->mixer.back().heads != h->d.heads || b->mixer.back().dim != h->d.hd)
      return fail(h, KC_ERR_INVALID_ARG, "a mixer block's cache has the brain's heads (4 of 32)");
  }
  KC_CHECK(check_cache(h, &v->selector, &b->selector));
  if (b->selector.heads != 1 || b->selector.dim != h->d.h)
    return fail(h, KC_ERR_INVALID_ARG, "the selector's cache has one head of the hidden size (128)");
  if (b->table.max_len > KC_MAX_ROW) return fail(h, KC_ERR_CAPACITY, "a turn's banks hold at most KC_MAX_ROW rows");
  return KC_OK;
}

// Everything a turn queues after its records are packed.
kc_status turn_pass(kc_handle* h, const DevBatch& b, const kc::FrameTotals& tot, const Bank& bank,
                    const kc_sampling* sampling, const kc_bank_out* out) {
  const Dims& d = h->d;
  Workspace& ws = h->ws;
  const uint64_t Q = tot.q, R = tot.r, H = d.h;
  const int mix_m = 3 * int(d.enc), sel_m = mix_m + 5 * int(d.mix);
  const uint64_t row = bank.table.max_len;
  kc::cache::Ask ask{P<float>(ws.mq), P<uint64_t>(ws.q_off), uint32_t(Q), d.heads, tot.max_q, H, kc::kF32};
  kc::cache::AttendArg a{};  // of a mixer block: they differ in their caches
  a.t = bank.table;
  a.a = ask;
  a.scale = kc::cache::scale_by(float(1.0 / std::sqrt(double(d.hd))));
  a.out_pitch = H;
  // what can be refused is refused before anything is appended
  if (Q > 0) {
    if (d.mix) {
      a.c = bank.mixer[0];
      KC_TRY(ensure(h, ws.turn_attend, Q * H * 4), "workspace");
      KC_TRY(ensure(h, ws.turn_work, kc::cache::plan_attend(a, h->sms) * 4 + 16), "workspace");
      a.out = ws.turn_attend.p;
      a.work = P<float>(ws.turn_work);
    }
    KC_TRY(ensure(h, ws.turn_off, (b.frames + 1) * 8ull), "workspace");
  }
  const bool planes = !h->kplanes.empty();
  if (planes && R > 0) {
    KC_TRY(ensure(h, ws.sk, h->kplanes.size() * R * H * 4), "workspace");
    KC_TRY(ensure(h, ws.mv, h->vplanes.size() * R * H * 4), "workspace");
  }
  KC_CHECK(encode_fast(h, ws, b, tot));
  if (R > 0) {
    if (planes) {  // bk through the selector's Wk and every block's Wk, bv through every block's Wv
      KC_CHECK(tc_gemm_planes(h, P<float>(ws.bk), R, h->kplanes, P<float>(ws.sk)));
      KC_CHECK(tc_gemm_planes(h, P<float>(ws.bv), R, h->vplanes, P<float>(ws.mv)));
    } else {
      KC_CHECK(tc_gemm<kc::tc::kEpiStore>(h, P<float>(ws.bk), R, sel_m + 1, P<float>(ws.sk)));
    }
    auto append = [&](const kc::cache::Store& c, float* keys, float* values) -> kc_status {
      const kc::cache::Rows r{keys, values, P<uint64_t>(ws.r_off), nullptr, R, H, kc::kF32};
      KC_TRY(kc::cache::launch_write(c, bank.table, r, h->sms, h->stream, &h->launches), "cache write launch");
      return KC_OK;
    };
    for (uint32_t blk = 0; blk < d.mix; blk++) {
      float* mk = planes ? P<float>(ws.sk) + (1 + blk) * R * H : P<float>(ws.mk);
      float* mv = planes ? P<float>(ws.mv) + blk * R * H : P<float>(ws.mv);
      if (!planes) {
        KC_CHECK(tc_gemm<kc::tc::kEpiStore>(h, P<float>(ws.bk), R, mix_m + 5 * int(blk) + 1, mk));
        KC_CHECK(tc_gemm<kc::tc::kEpiStore>(h, P<float>(ws.bv), R, mix_m + 5 * int(blk) + 2, mv));
      }
      KC_CHECK(append(bank.mixer[blk], mk, mv));
    }
    KC_CHECK(append(bank.selector, P<float>(ws.sk), P<float>(ws.bv)));
  }
  if (Q == 0) return KC_OK;
  for (uint32_t blk = 0; blk < d.mix; blk++) {
    const int m0 = mix_m + 5 * int(blk);
    KC_CHECK(tc_gemm<kc::tc::kEpiStore>(h, P<float>(ws.qstate), Q, m0, P<float>(ws.mq)));
    a.c = bank.mixer[blk];
    kc::cache::plan_attend(a, h->sms);
    KC_TRY(kc::cache::launch_attend(a, h->sms, h->stream, &h->launches), "attention launch");
    k_turn_add<<<unsigned((Q * H / 4 + 255) / 256), 256, 0, h->stream>>>(P<float4>(ws.qstate),
                                                                       P<float4>(ws.turn_attend), Q * H / 4);
    h->launches++;
    KC_CHECK(tc_gemm<kc::tc::kEpiRelu>(h, P<float>(ws.qstate), Q, m0 + 3, P<float>(ws.mh)));
    KC_CHECK(tc_gemm<kc::tc::kEpiResid>(h, P<float>(ws.mh), Q, m0 + 4, P<float>(ws.qstate)));
  }
  KC_CHECK(tc_gemm<kc::tc::kEpiStore>(h, P<float>(ws.qstate), Q, sel_m, P<float>(ws.sq)));
  k_turn_offsets<<<b.frames / 256 + 1, 256, 0, h->stream>>>(P<uint64_t>(ws.q_off), b.frames, row, P<uint64_t>(ws.turn_off));
  h->launches++;
  ask.q = ws.sq.p;
  ask.heads = 1;
  const kc::cache::ScoreArg sa{bank.selector, bank.table, ask, out->p, P<uint64_t>(ws.turn_off), b.mask,
                               kc::cache::scale_by(float(1.0 / std::sqrt(double(d.h))))};
  KC_TRY(kc::cache::launch_scores(sa, h->sms, h->stream, &h->launches), "scores launch");
  const kc_sampling whole{1.0f, 0, 1.0f, 0.0f, nullptr, nullptr, nullptr, nullptr};
  const kc_rows_view rows{out->p, nullptr, nullptr, uint32_t(Q), 0, row, 0, KC_DTYPE_F32, KC_ROWS_SCORES};
  kc_draw_out drawn{};
  drawn.index = out->index;
  drawn.logp = out->logp;
  drawn.p = out->p;
  return draw_rows(h, &rows, sampling ? sampling : &whole, b.uniforms, &drawn);
}

}  // namespace

extern "C" kc_status kc_bank_turn(kc_handle* h, const kc_batch_view* bv, const kc_bank_view* bank_view,
                                  const kc_sampling* sampling, kc_bank_out* out) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  if (!bv || !out || bv->frames == 0) return fail(h, KC_ERR_INVALID_ARG, "batch arguments are incomplete");
  if (!bv->rec_off || !bv->token_ids || !bv->field_roles || !bv->schema_ids || !bv->band_ids)
    return fail(h, KC_ERR_INVALID_ARG, "batch view is incomplete");
  if (!aligned(bv->token_ids, 16) || !aligned(bv->rec_off, 8))
    return fail(h, KC_ERR_INVALID_ARG, "token_ids must be 16-byte aligned and rec_off 8-byte aligned");
  if (bv->schema_allow || bv->band_allow)
    return fail(h, KC_ERR_INVALID_ARG, "a cache keeps no schemas or bands: a turn takes an explicit mask");
  if (!aligned(out->p, 4) || !aligned(out->index, 4) || !aligned(out->logp, 4) || !aligned(bv->mask, 4))
    return fail(h, KC_ERR_INVALID_ARG, "a turn's outputs and mask must be 4-byte aligned");
  if (!aligned(bv->uniforms, 8)) return fail(h, KC_ERR_INVALID_ARG, "uniforms must be 8-byte aligned");
  if (sampling) KC_CHECK(check_sampling(h, sampling, false));
  Bank bank;
  try {
    KC_CHECK(check_bank(h, bank_view, bv->frames, &bank));
  } catch (const std::bad_alloc&) {
    return fail(h, KC_ERR_CAPACITY, "out of host memory for the bank's caches");
  }
  DevBatch b;
  b.frames = bv->frames; b.records = bv->records; b.rec_off = bv->rec_off;
  b.token_ids = bv->token_ids; b.field_roles = bv->field_roles; b.schema_ids = bv->schema_ids;
  b.band_ids = bv->band_ids; b.uniforms = bv->uniforms; b.word_ids = bv->word_ids; b.word_alpha = bv->word_alpha;
  b.mask = bv->mask;
  kc::FrameTotals tot;
  // whatever the call answers, its arrays are the caller's again: nothing that it
  // queued is left to run
  auto over = [&](kc_status s) {
    if (s) (void)wait_stream(h);
    return s;
  };
  KC_CHECK(over(pack_batch(h, h->ws, b, &tot)));
  if (tot.q && (!out->p || out->q_capacity < tot.q))
    return over(fail(h, KC_ERR_CAPACITY, "the output rows are fewer than the turn's questions"));
  for (;;) {
    KC_CHECK(over(turn_pass(h, b, tot, bank, sampling, out)));
    KC_TRY(cudaMemcpyAsync(h->h_err, h->d_err, sizeof(int), cudaMemcpyDeviceToHost, h->stream), "readback");
    KC_TRY(wait_stream(h), "turn");
    const int e = *h->h_err;
    if (e & kc::tc::kErrTimeout)
      return fail(h, KC_ERR_TIMEOUT, "a tensor-core pipeline wait expired; the turn was not completed");
    if (!(e & kc::tc::kErrOverflow)) break;
    // activations left the split's range: again at a smaller scale (what was
    // appended is written over)
    if (h->sa <= -24) return fail(h, KC_ERR_NONFINITE, "the activations leave the range of the split products");
    h->sa -= 6;
  }
  out->total_q = tot.q;
  out->total_r = tot.r;
  if (h->profiling) prof_collect(h);
  return KC_OK;
}
