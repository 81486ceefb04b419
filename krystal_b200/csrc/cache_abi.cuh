// cache_abi.cuh — the C ABI of the bank cache (kc_cache_*): argument checks and
// the launchers of cache_store.cu and cache_attend*.cu.
#pragma once

namespace {

static_assert(kc::cache::kI8 == KC_CACHE_I8 && kc::cache::kE4M3 == KC_CACHE_E4M3 && kc::cache::kPage == KC_CACHE_PAGE &&
              kc::cache::kMaxBlocks * KC_CACHE_PAGE == KC_CACHE_MAX_SELECT, "the header's cache is the kernels'");

kc_status check_cache(kc_handle* h, const kc_cache_view* v, kc::cache::Store* c) {
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the cache view is null");
  if (v->format != KC_CACHE_I8 && v->format != KC_CACHE_E4M3)
    return fail(h, KC_ERR_INVALID_ARG, "a cache holds i8 or e4m3 codes");
  if (v->head_dim != 32 && v->head_dim != 64 && v->head_dim != 128)
    return fail(h, KC_ERR_CAPACITY, "a cache's head_dim is 32, 64 or 128");
  if (v->kv_heads == 0 || v->kv_heads > 128) return fail(h, KC_ERR_CAPACITY, "a cache has 1 to 128 kv_heads");
  if (v->pages == 0) return fail(h, KC_ERR_INVALID_ARG, "a cache without pages");
  if (!v->storage || !aligned(v->storage, 16))
    return fail(h, KC_ERR_INVALID_ARG, "a cache's storage must be there and 16-byte aligned");
  if (v->bytes < kc_cache_bytes(v->pages, v->kv_heads, v->head_dim))
    return fail(h, KC_ERR_CAPACITY, "the storage is smaller than kc_cache_bytes(pages, kv_heads, head_dim)");
  c->cells = static_cast<uint8_t*>(v->storage);
  c->bounds = reinterpret_cast<float*>(c->cells + uint64_t(v->pages) * v->kv_heads * 2 * kc::cache::cell_bytes(v->head_dim));
  c->pages = v->pages;
  c->heads = v->kv_heads;
  c->dim = v->head_dim;
  c->format = v->format;
  return KC_OK;
}

kc_status check_table(kc_handle* h, const kc_page_table* v, kc::cache::Table* t) {
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the page table is null");
  if (v->sequences && (!v->lengths || (v->pitch && !v->pages)))
    return fail(h, KC_ERR_INVALID_ARG, "a page table needs its pages and lengths");
  if (!aligned(v->pages, 4) || !aligned(v->lengths, 4))
    return fail(h, KC_ERR_INVALID_ARG, "the pages and lengths must be 4-byte aligned");
  const uint64_t most = std::min<uint64_t>(uint64_t(v->pitch) * KC_CACHE_PAGE, 0xffffffc0u);
  if (v->max_length > most) return fail(h, KC_ERR_INVALID_ARG, "max_length is longer than the table's pages");
  t->table = v->pages;
  t->lengths = v->lengths;
  t->seqs = v->sequences;
  t->pitch = v->pitch;
  t->max_len = v->max_length ? v->max_length : uint32_t(most);
  return KC_OK;
}

kc_status check_element(kc_handle* h, int32_t dtype, uintptr_t* size) {
  if (dtype != KC_DTYPE_F32 && dtype != KC_DTYPE_F16 && dtype != KC_DTYPE_BF16)
    return fail(h, KC_ERR_INVALID_ARG, "rows and questions are f32, f16 or bf16");
  *size = dtype == KC_DTYPE_F32 ? 4 : 2;
  return KC_OK;
}

kc_status cache_rows(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table, const kc_cache_rows* v,
                     const uint32_t* starts, bool write) {
  kc::cache::Store c;
  kc::cache::Table t;
  KC_CHECK(check_cache(h, cache, &c));
  KC_CHECK(check_table(h, table, &t));
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the rows are null");
  uintptr_t size;
  KC_CHECK(check_element(h, v->dtype, &size));
  const uint64_t width = uint64_t(c.heads) * c.dim;
  if (v->rows && (write ? !v->keys || !v->values : !v->keys && !v->values))
    return fail(h, KC_ERR_INVALID_ARG, write ? "a write needs keys and values" : "a read needs keys or values");
  if (v->pitch && v->pitch < width)
    return fail(h, KC_ERR_INVALID_ARG, "the rows' pitch is smaller than kv_heads * head_dim");
  if (!v->row_off && v->rows != t.seqs)
    return fail(h, KC_ERR_INVALID_ARG, "without row_off there is one row a sequence");
  if (!aligned(v->keys, size) || !aligned(v->values, size) || !aligned(v->row_off, 8) || !aligned(starts, 4))
    return fail(h, KC_ERR_INVALID_ARG, "rows, their offsets and starts must be aligned to their type");
  if (v->rows >> 31) return fail(h, KC_ERR_CAPACITY, "a call takes at most 2147483647 rows");
  const kc::cache::Rows r{v->keys, v->values, v->row_off, starts, v->rows, v->pitch ? v->pitch : width, v->dtype};
  if (write) KC_TRY(kc::cache::launch_write(c, t, r, h->sms, h->stream, &h->launches), "cache write launch");
  else KC_TRY(kc::cache::launch_read(c, t, r, h->sms, h->stream, &h->launches), "cache read launch");
  return KC_OK;
}

// Questions over a checked cache.
kc_status check_ask(kc_handle* h, const kc_question_view* v, const kc::cache::Store& c, const kc::cache::Table& t,
                    kc::cache::Ask* a) {
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the questions are null");
  uintptr_t size;
  KC_CHECK(check_element(h, v->dtype, &size));
  if (v->heads == 0 || v->heads % c.heads || v->heads > 1024)
    return fail(h, KC_ERR_INVALID_ARG, "heads must be a multiple of kv_heads, at most 1024");
  const uint64_t width = uint64_t(v->heads) * c.dim;
  if (v->pitch && v->pitch < width)
    return fail(h, KC_ERR_INVALID_ARG, "the questions' pitch is smaller than heads * head_dim");
  if (!v->q_off && v->questions != t.seqs)
    return fail(h, KC_ERR_INVALID_ARG, "without q_off there is one question a sequence");
  if (v->questions && !v->q) return fail(h, KC_ERR_INVALID_ARG, "the questions have no values");
  if (!aligned(v->q, size) || !aligned(v->q_off, 8))
    return fail(h, KC_ERR_INVALID_ARG, "questions and their offsets must be aligned to their type");
  if (uint64_t(v->questions) * v->heads > 0x7fffffffull)
    return fail(h, KC_ERR_CAPACITY, "a call takes at most 2147483647 heads of questions");
  a->q = v->q;
  a->off = v->q_off;
  a->questions = v->questions;
  a->heads = v->heads;
  a->max_q = !v->q_off ? 1 : v->max_questions ? std::min(v->max_questions, v->questions) : v->questions;
  a->pitch = v->pitch ? v->pitch : width;
  a->dtype = v->dtype;
  return KC_OK;
}

// What a launch answered; too many units are the caller's bound on the questions.
kc_status launched(kc_handle* h, cudaError_t e, const char* what) {
  if (e == cudaErrorInvalidConfiguration)
    return fail(h, KC_ERR_CAPACITY, "sequences times max_questions leave the launch's range: bound one sequence's questions");
  KC_TRY(e, what);
  return KC_OK;
}

kc_status check_scale(kc_handle* h, float scale, uint32_t dim, kc::cache::Scale* out) {
  if (!std::isfinite(scale)) return fail(h, KC_ERR_INVALID_ARG, "scale must be finite");
  *out = kc::cache::scale_by(scale != 0.0f ? scale : float(1.0 / std::sqrt(double(dim))));
  return KC_OK;
}

}  // namespace

extern "C" {

uint64_t kc_cache_bytes(uint32_t pages, uint32_t kv_heads, uint32_t head_dim) {
  return uint64_t(pages) * kv_heads * (2 * uint64_t(kc::cache::cell_bytes(head_dim)) + 8 * uint64_t(head_dim));
}

kc_status kc_cache_write(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table, const kc_cache_rows* rows) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  return cache_rows(h, cache, table, rows, nullptr, true);
}

kc_status kc_cache_read(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table, const uint32_t* starts,
                        const kc_cache_rows* rows) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  return cache_rows(h, cache, table, rows, starts, false);
}

kc_status kc_cache_blocks(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table,
                          const kc_question_view* questions, uint32_t count, uint32_t recent, uint32_t* blocks) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  kc::cache::BlockArg a{};
  KC_CHECK(check_cache(h, cache, &a.c));
  KC_CHECK(check_table(h, table, &a.t));
  KC_CHECK(check_ask(h, questions, a.c, a.t, &a.a));
  if (count == 0) return fail(h, KC_ERR_INVALID_ARG, "a selection takes at least one block");
  if (recent > count) return fail(h, KC_ERR_INVALID_ARG, "recent blocks are among the count: at most count");
  if (a.t.max_len > KC_CACHE_MAX_SELECT)
    return fail(h, KC_ERR_CAPACITY, "blocks are selected over at most KC_CACHE_MAX_SELECT rows a sequence");
  if (a.a.questions && (!blocks || !aligned(blocks, 4)))
    return fail(h, KC_ERR_INVALID_ARG, "the blocks must be there and 4-byte aligned");
  a.count = count;
  a.recent = recent;
  a.blocks = blocks;
  return launched(h, kc::cache::launch_blocks(a, h->sms, h->stream, &h->launches), "block selection launch");
}

uint64_t kc_cache_attend_workspace(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table,
                                   const kc_question_view* questions, uint32_t block_count) {
  if (!h) return 0;
  std::lock_guard<std::mutex> lk(h->mu);
  kc::cache::AttendArg a{};
  if (check_cache(h, cache, &a.c) || check_table(h, table, &a.t) || check_ask(h, questions, a.c, a.t, &a.a)) return 0;
  a.block_count = block_count;
  return kc::cache::plan_attend(a, h->sms) * 4;
}

kc_status kc_cache_attend(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table,
                          const kc_question_view* questions, const kc_attend_view* v) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  kc::cache::AttendArg a{};
  KC_CHECK(check_cache(h, cache, &a.c));
  KC_CHECK(check_table(h, table, &a.t));
  KC_CHECK(check_ask(h, questions, a.c, a.t, &a.a));
  if (!v) return fail(h, KC_ERR_INVALID_ARG, "the attention view is null");
  const uint64_t width = uint64_t(a.a.heads) * a.c.dim;
  if (a.a.questions && !v->out) return fail(h, KC_ERR_INVALID_ARG, "attention needs an output");
  if (v->out_pitch && v->out_pitch < width)
    return fail(h, KC_ERR_INVALID_ARG, "the output's pitch is smaller than heads * head_dim");
  if (v->out && v->out == questions->q) return fail(h, KC_ERR_INVALID_ARG, "attention does not write over its questions");
  if (v->mask && !v->mask_off) return fail(h, KC_ERR_INVALID_ARG, "a mask needs its offsets");
  if ((v->blocks != nullptr) != (v->block_count != 0))
    return fail(h, KC_ERR_INVALID_ARG, "a list of blocks needs its count, and a count its list");
  if (!aligned(v->out, a.a.dtype == KC_DTYPE_F32 ? 4 : 2) || !aligned(v->lse, 4) || !aligned(v->mask, 4) ||
      !aligned(v->mask_off, 8) || !aligned(v->blocks, 4) || !aligned(v->workspace, 16))
    return fail(h, KC_ERR_INVALID_ARG, "an attention's arrays must be aligned to their type, its workspace to 16 bytes");
  KC_CHECK(check_scale(h, v->scale, a.c.dim, &a.scale));
  a.out = v->out;
  a.out_pitch = v->out_pitch ? v->out_pitch : width;
  a.lse = v->lse;
  a.mask = v->mask;
  a.mask_off = v->mask_off;
  a.blocks = v->blocks;
  a.block_count = v->block_count;
  const uint64_t need = kc::cache::plan_attend(a, h->sms) * 4;
  if (need && (!v->workspace || v->workspace_bytes < need))
    return fail(h, KC_ERR_CAPACITY, "the workspace is smaller than kc_cache_attend_workspace");
  a.work = static_cast<float*>(v->workspace);
  return launched(h, kc::cache::launch_attend(a, h->sms, h->stream, &h->launches), "attention launch");
}

kc_status kc_cache_scores(kc_handle* h, const kc_cache_view* cache, const kc_page_table* table,
                          const kc_question_view* questions, const uint64_t* off, const float* mask, float scale,
                          float* scores) {
  if (!h) return fail(nullptr, KC_ERR_INVALID_ARG, "handle is null");
  std::lock_guard<std::mutex> lk(h->mu);
  DeviceGuard dg(h->device);
  kc::cache::ScoreArg a{};
  KC_CHECK(check_cache(h, cache, &a.c));
  KC_CHECK(check_table(h, table, &a.t));
  KC_CHECK(check_ask(h, questions, a.c, a.t, &a.a));
  if (a.a.heads != 1) return fail(h, KC_ERR_CAPACITY, "pointer scores are taken over one head");
  if (a.a.questions && (!off || !scores)) return fail(h, KC_ERR_INVALID_ARG, "scores need their offsets and an output");
  if (!aligned(off, 8) || !aligned(mask, 4) || !aligned(scores, 4))
    return fail(h, KC_ERR_INVALID_ARG, "scores, mask and offsets must be aligned to their type");
  KC_CHECK(check_scale(h, scale, a.c.dim, &a.scale));
  a.scores = scores;
  a.off = off;
  a.mask = mask;
  return launched(h, kc::cache::launch_scores(a, h->sms, h->stream, &h->launches), "scores launch");
}

}  // extern "C"
