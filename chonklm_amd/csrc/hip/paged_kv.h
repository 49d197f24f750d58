// The quantised, paged K/V cache: writing, reading back, attention of one new
// token a row (paged_kv.hip). The page format is chonk.h's.
#pragma once

#include <hip/hip_runtime.h>

#include "prefill.h"

namespace chonk {

enum KvFault : int32_t { KVF_SEQ = 1, KVF_POS = 2, KVF_PAGE = 4 };

struct KvCache {
  uint8_t* pages;
  const int32_t* table;   // [n_seqs][max_pages]
  int32_t* fault;         // KvFault bits of rows that were refused, or null
  int32_t type, kv_heads, hd, n_pages, n_seqs, max_pages;
};

// Bytes of one kv head's K (or V) in a page: codes, then scales.
constexpr int kv_code_bytes(int type, int hd) {
  return kKvPage * (type == CHONK_KV_F16 ? 2 * hd : type == CHONK_KV_Q8 ? hd : hd / 2);
}
constexpr int kv_part_bytes(int type, int hd) {
  return kv_code_bytes(type, hd) + (type == CHONK_KV_F16 ? 0 : kKvPage * (hd / 32) * 2);
}
constexpr bool kv_type_ok(int type) { return type == CHONK_KV_F16 || type == CHONK_KV_Q8 || type == CHONK_KV_Q4; }
constexpr bool kv_hd_ok(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

// Sequence and position of a row; a negative sequence leaves the row out.
struct KvPlace {
  const int32_t *seq, *pos;  // [rows], or null: seq0, p0 + row
  int32_t seq0, p0;
};

struct KvAppendArgs {
  KvCache c;
  KvPlace at;
  PartSum q, k, v;        // fp32 rows (K-split partial sums, their ld not read); q.p null: k and v alone
  const _Float16 *q16, *k16, *v16;  // fp16 rows instead
  void* q_out;            // rows of the input's type
  int64_t q_ld, k_ld, v_ld, qo_ld;  // elements from row to row
  int32_t rows, heads, f16;
  const float *qn_w, *kn_w;
  double eps;
  const float2* rope;     // [rope_n][rope_dim / 2], or null
  int32_t rope_dim, rope_n, interleaved;
};

struct KvReadArgs {
  KvCache c;
  KvPlace at;
  void *k, *v;            // either may be null
  int64_t row_ld, head_ld;
  int32_t rows, f16;
};

struct KvAttendArgs {
  KvCache c;
  const int32_t *seq;     // [rows]
  const int32_t *len;     // [rows] positions a row may see
  int32_t len_add;        // added to len (rows' positions given instead: 1)
  const void* q;
  void* out;
  int64_t q_ld, o_ld;
  int32_t rows, heads, f16, window;
  // set by the launcher: rows are cut into at most `want` segments, joined from part, unless the
  // longest has at most `whole` half pages (many: or the rows are about as long as each other)
  int32_t split, want, whole, many;
  float scale;
  float* part;
};

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s);
hipError_t launch_kv_read(const KvReadArgs& a, hipStream_t s);
// Floats of workspace that launch_kv_attend needs for these rows.
int64_t kv_attend_floats(const KvCache& c, int rows, int heads);
hipError_t launch_kv_attend(const KvAttendArgs& a, hipStream_t s);

}  // namespace chonk
