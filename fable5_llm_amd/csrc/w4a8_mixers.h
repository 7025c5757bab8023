// Declarations of the mixers between a step's sites: attention over a paged
// key-value cache (w4a8_attend.hip), the cache's pages (w4a8_kv.hip) and the
// gated delta rule (w4a8_delta.hip), shared with the C ABI (w4a8_abi.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace w4a8 {

// element types of activations and caches (W4A8_DT_*)
enum Dtype { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2, DT_I16 = 3 };
inline int dtype_size(int d) { return d == DT_F32 ? 4 : 2; }

// bits of the context's error word
constexpr int kErrKvRange = 32;    // a sequence, position or page outside the cache
constexpr int kErrKvFull = 64;     // too few free pages
constexpr int kErrKvList = 128;    // a sequence listed twice, or a child not empty
constexpr int kErrDelta = 256;     // a state slot or a prompt's bounds
constexpr int kKvSkip = 1 << 30;   // never in the word: the call comes behind a refused one

// 16-byte loads and stores that pass the caches by: data read or written once
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 load16_nt(const void *p) {
  return __builtin_nontemporal_load((const u32x4 *)p);
}
__device__ __forceinline__ void store16_nt(void *p, u32x4 v) {
  __builtin_nontemporal_store(v, (u32x4 *)p);
}

// A paged cache.  pool: [pages][layers][keys, values][kv heads][page tokens]
// [head dim], so that a page holds every layer's rows of its tokens and is
// copied as one block, and a head's rows of one page are one run of memory.
// refs[page]: sequences that hold it, 0 if free.  tables[seq][max_pages]: the
// pages of sequence seq, ceil(lens[seq] / page tokens) of them in use.
struct KvCache {
  uint8_t *pool;
  int32_t *refs, *tables, *lens;
  int32_t *scratch;           // kv_scratch_words(seqs, pages) words, marks zero
  int32_t *err;               // the context's error word, and how often it was taken
  int32_t pages, seqs, max_pages, lg_page;
  int32_t layers, heads, dim, esize, dtype;
  int64_t page_bytes;
  __host__ __device__ int32_t page() const { return 1 << lg_page; }
};
// scratch: a head of kKvHead words, a mark and a job per sequence, two words
// per page
constexpr int kKvHead = 64;
inline size_t kv_scratch_words(int64_t seqs, int64_t pages) {
  return kKvHead + 2 * (size_t)seqs + 2 * (size_t)pages;
}
// word of scratch that a refused reserve or fork leaves: 1 + how often the
// error word had been taken.  Until the next time, calls that change the cache
// do nothing: those behind the refused one count on it (an append without
// positions would overwrite the token before).
constexpr int kKvStop = 2;
__device__ __forceinline__ bool kv_stopped(const KvCache &kv) {
  return kv.scratch[kKvStop] == kv.err[1] + 1;
}
hipError_t launch_kv_extend(const KvCache &kv, const int32_t *seqs, const int32_t *counts,
                            int32_t n, hipStream_t s);
hipError_t launch_kv_fork(const KvCache &kv, const int32_t *parents, const int32_t *children,
                          int32_t n, hipStream_t s);
hipError_t launch_kv_free(const KvCache &kv, const int32_t *seqs, int32_t n, hipStream_t s);
hipError_t launch_kv_compact(const KvCache &kv, int num_cu, hipStream_t s);
hipError_t launch_kv_copy(const KvCache &kv, const int32_t *src, const int32_t *dst, int32_t n,
                          int num_cu, hipStream_t s);
struct KvAppend {
  const void *k, *v;            // [n][heads][dim], strides in elements
  int64_t k_token, k_head, v_token, v_head;
  const int32_t *seqs, *pos;    // pos null: each sequence's last token
  int32_t n, layer, dtype;
  float unit;                   // DT_I16: the value of one step
};
hipError_t launch_kv_append(const KvCache &kv, const KvAppend &a, hipStream_t s);

struct Attend {
  const void *q;                // [rows][hq][dim], strides in elements
  void *out;
  int64_t q_row, q_head, out_row, out_head;
  const int32_t *seqs, *upto;   // upto null: every token of the sequence
  float *part;                  // [rows][hq][splits][dim], then {max, sum} [rows][hq][splits]
  int32_t rows, hq, layer, splits, dtype;
  float scale;                  // of the scores, log2(e) included
  float out_unit;               // DT_I16: 1 / the value of one step of out
};
constexpr int kAttendChunk = 128;   // least tokens of a split
int attend_splits(const KvCache &kv, int64_t rows, int64_t hq, int num_cu);
int64_t attend_workspace(const KvCache &kv, int64_t rows, int64_t hq, int num_cu);
hipError_t launch_attend(const KvCache &kv, const Attend &a, hipStream_t s);

// The gated delta rule: q, k [tokens][hk][dk], v, out [tokens][hv][dv], g and
// beta [tokens][hv], state [slots][hv][dk][dv].
struct Delta {
  const void *q, *k, *v;
  const float *g, *beta;
  float *state;
  void *out;
  const int32_t *slots;         // null: row i's state is slot i
  const int32_t *cu;            // null: one token per row
  void *ws;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, g_token, beta_token, out_token,
      out_head;
  int32_t tokens, rows, hk, hv, dk, dv, nslots, dtype, norm, fresh;
  float scale, eps;
  float unit, out_unit;         // DT_I16: the value of a step of q, k, v; 1 / that of out
  int32_t *err;
  int32_t claimed;              // one token per row: the rows' slots lie in out (launch_delta)
};
constexpr int64_t kDeltaStride = 1 << 23;   // of v's and out's tokens, whole prompts
int64_t delta_workspace(int64_t tokens, int64_t rows, int64_t hk, int64_t hv, int64_t dk,
                        int dtype);
hipError_t launch_delta(Delta d, int num_cu, hipStream_t s);

}  // namespace w4a8
