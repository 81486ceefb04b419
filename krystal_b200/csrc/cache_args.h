// cache_args.h — the bank cache's storage, and the arguments of its kernels and
// their launchers (cache_store.cu, cache_attend_*.cu), which krystal_cuda.cu
// calls for the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cmath>

namespace kc {
namespace cache {

constexpr int kI8 = 0, kE4M3 = 1;            // KC_CACHE_* of the C ABI
constexpr uint32_t kPage = 64, kCell = 32;   // rows of a page, rows of a cell
constexpr uint32_t kNone = 0xffffffffu;
constexpr float kBlocked = -1e29f;           // a mask entry at or below it (or NaN) shuts a row out
constexpr float kShut = -1e30f;              // the score of a row that is shut out
constexpr uint32_t kMaxBlocks = 25600;       // pages a sequence may have where blocks are selected (200 KB of keys)

// A cell: keys [32][dim] and values [32][dim], 8 bits each, then 32 f32 key
// scales and 32 f32 value scales.
__host__ __device__ constexpr uint32_t cell_bytes(uint32_t dim) { return kCell * (2 * dim + 8); }

// The storage: cells [pages][heads][2], then bounds [pages][heads][2][dim] f32
// (the smallest, then the largest of the page's stored keys).
struct Store {
  uint8_t* cells;
  float* bounds;
  uint32_t pages, heads, dim;
  int format;
};

// Sequence s holds lengths[s] rows in the pages table[s * pitch ..].
struct Table {
  const uint32_t *table, *lengths;
  uint32_t seqs, pitch;
  uint32_t max_len;  // what longer sequences count as; at most pitch * 64
};

// Rows to write or to read: sequence s has rows off[s] .. off[s + 1] - 1 (off
// null: row s). They are the sequence's last, or (starts) those from starts[s] on.
struct Rows {
  void *keys, *values;
  const uint64_t* off;
  const uint32_t* starts;
  uint64_t rows, pitch;
  int dtype;  // kF32 / kF16 / kBF16 of policy_args.h
};

// Questions [questions][heads][dim]; sequence s asks off[s] .. off[s + 1] - 1
// (off null: question s).
struct Ask {
  const void* q;
  const uint64_t* off;
  uint32_t questions, heads, max_q;
  uint64_t pitch;
  int dtype;
};

// What scores are multiplied by: m 2^e, |m| in [1/2, 1).
struct Scale {
  float m;
  int e;
};
inline Scale scale_by(float x) {
  Scale s;
  s.m = std::frexp(x, &s.e);
  return s;
}

struct AttendArg {
  Store c;
  Table t;
  Ask a;
  void* out;
  uint64_t out_pitch;
  float* lse;
  const float* mask;        // sequence s's [Q_s, R_s] block at mask_off[s]
  const uint64_t* mask_off;
  const uint32_t* blocks;   // [questions][kv heads][block_count], or null: every block
  uint32_t block_count;
  Scale scale;
  float* work;              // partial results of split sequences
  uint32_t splits;          // parts a sequence's rows are cut into at most (1: none)
  uint32_t chunk;           // blocks of a part
};

struct ScoreArg {
  Store c;
  Table t;
  Ask a;
  float* scores;            // sequence s's [Q_s, R_s] block at off[s]
  const uint64_t* off;
  const float* mask;        // laid out like scores, or null
  Scale scale;
};

struct BlockArg {
  Store c;
  Table t;
  Ask a;
  uint32_t count, recent;
  uint32_t* blocks;         // [questions][kv heads][count]
};

// By question type (cache_attend_f32.cu, cache_attend_f16.cu, cache_attend_bf16.cu).
cudaError_t attend_f32(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t attend_f16(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t attend_bf16(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t scores_f32(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t scores_f16(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t scores_bf16(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches);

cudaError_t prepare_store();
cudaError_t prepare_f32();
cudaError_t prepare_f16();
cudaError_t prepare_bf16();

// What the kernels need once on each device (the current one).
cudaError_t prepare();

cudaError_t launch_write(const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t launch_read(const Store& c, const Table& t, const Rows& r, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t launch_blocks(const BlockArg& a, int sms, cudaStream_t s, uint64_t* launches);
cudaError_t launch_scores(const ScoreArg& a, int sms, cudaStream_t s, uint64_t* launches);

// How a call's sequences are cut, and the workspace (floats) that takes; fills
// a.splits and a.chunk.
uint64_t plan_attend(AttendArg& a, int sms);
cudaError_t launch_attend(const AttendArg& a, int sms, cudaStream_t s, uint64_t* launches);

}  // namespace cache
}  // namespace kc
