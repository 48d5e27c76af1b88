// Paged cache: parameter blocks and index arithmetic shared by the kernels,
// the host launcher and (the arithmetic alone, as plain C++) the CPU tests.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define C2H_HD __host__ __device__
#else
#define C2H_HD
#endif

namespace c2h {

// Element types (include/c2h.h).
enum PagedType : int { PT_F32 = 0, PT_F16 = 1, PT_BF16 = 30, PT_E4M3 = 100 };
C2H_HD constexpr int type_bytes(int t) { return t == PT_F32 ? 4 : t == PT_E4M3 ? 1 : 2; }

// What a kernel found wrong, or-ed into a pinned word that c2h_sync reads.
enum PagedErr : int { PERR_LENGTH = 1, PERR_PAGE = 2, PERR_START = 4 };

constexpr int PAGED_MIN_PAGE = 8;      // a lane's four rows of V lie in one page
constexpr int PAGED_MAX_PAGE = 1024;
// A launch's work-items stay below 2^32, at most 256 per token, per (session,
// head) and 1024 per row.
constexpr int MAX_TOKENS = (1 << 24) - 1, MAX_SESSION_HEADS = (1 << 24) - 1, MAX_NORM_ROWS = (1 << 22) - 1;
constexpr int PAGED_MAX_LEN = 1 << 23; // a position and a chunk's end beyond it (chunk_units) fit 32 bits
constexpr int ATTN_HEADS = 16;         // query heads of a workgroup: columns of the matrix instruction
constexpr int ATTN_CHUNKS = 1024;      // chunks that a batch is cut into
constexpr int ATTN_MANY_ROWS = 2048;   // rows from which the join takes several a workgroup
constexpr int ATTN_WGS = 512;          // workgroups that take them in turn

// The positions [lo, hi) that a session of `len` positions attends, `window`
// of them at most (0: all).
struct Span {
  int lo, hi;
};
C2H_HD inline Span attended(int len, int window) {
  return Span{window > 0 && len > window ? len - window : 0, len};
}
// A span is cut into chunks of whole units, of the positions that the four
// waves of a workgroup take in one step.  Chunks begin at multiples of their
// size from the span's first position rounded down to a multiple of 4, so that
// four positions a lane reads together lie in one page; the first chunk's
// begin at s.lo.
constexpr int SPAN_ALIGN = 4;
C2H_HD inline int chunk_base(Span s, int chunk, int i) { return (s.lo & ~(SPAN_ALIGN - 1)) + i * chunk; }
C2H_HD inline int units_of(Span s, int unit) { return (s.hi - (s.lo & ~(SPAN_ALIGN - 1)) + unit - 1) / unit; }
// Chunks of a session: at least one, which writes the row of an empty one.
C2H_HD inline int chunks_of(int units, int chunk_units) {
  const int n = (units + chunk_units - 1) / chunk_units;
  return n > 1 ? n : 1;
}
// Tiles of 16 positions in a wave's step: 16 KB of keys and values, at most
// four tiles and at least one.
C2H_HD constexpr int attn_tiles(int type, int hd) {
  const int t = 512 / (hd * type_bytes(type));
  return t < 1 ? 1 : t > 4 ? 4 : t;
}
C2H_HD constexpr int attn_hd(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
C2H_HD constexpr int attn_unit(int type, int head_dim) { return 64 * attn_tiles(type, attn_hd(head_dim)); }
// Units per chunk: a batch of `units` in all, in each of n_rows (KV head, head
// tile) rows, as about ATTN_CHUNKS equal chunks; no more than the longest
// session has of the smallest unit, so that a chunk's positions (at most 2^25)
// fit 32 bits however large the batch.
C2H_HD inline int chunk_units(int64_t units, int n_rows) {
  const int64_t c = (units * n_rows + ATTN_CHUNKS - 1) / ATTN_CHUNKS, most = PAGED_MAX_LEN / 64;
  return (int)(c < 1 ? 1 : c < most ? c : most);
}
// Chunks (of one row) that any batch of sessions of up to max_units can come
// to: about ATTN_CHUNKS / n_rows, and a partial one per session.
inline int64_t chunks_bound(int n_seqs, int n_rows, int max_units) {
  const int64_t even = ATTN_CHUNKS / n_rows + 1 + n_seqs, all = (int64_t)n_seqs * (max_units > 1 ? max_units : 1);
  return even < all ? even : all;
}
// A wave's lanes hold the pages from page p0 on, one each, enough for its
// steps at base, base + unit, ... before the one returned.
C2H_HD inline int first_step_beyond(int p0, int page_shift, int base, int step, int unit) {
  const int limit = (p0 + 64) << page_shift;
  return base + ((limit - step - base) / unit + 1) * unit;
}

C2H_HD inline bool length_ok(int len, int max_len) { return len >= 0 && len <= max_len; }
C2H_HD inline bool page_ok(int page, int n_pages) { return (uint32_t)page < (uint32_t)n_pages; }

// Position of the i-th token of a call, the token `i` of tokens
// [start, end) that are the last ones of a session of `len` positions; < 0
// if the session does not hold that many.
C2H_HD inline int64_t token_pos(int len, int64_t i, int64_t end) { return (int64_t)len - (end - i); }

struct PagedKV {
  char* k;
  char* v;
  int64_t page_stride, token_stride, head_stride;  // bytes
  const float* k_scale;
  const float* v_scale;
  int n_pages, page_shift, n_kv_heads, head_dim;
};
struct PagedBatch {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  int n_seqs, max_len;
};
struct HeadRows {
  char* data;
  int64_t token_stride, head_stride;  // bytes
};

struct PagedAttnParams {
  PagedKV kv;
  PagedBatch b;
  HeadRows q, out;
  int type;        // of q and out
  int n_heads, group, n_tiles;  // query heads, per KV head, workgroups of ATTN_HEADS of them
  int window;
  int n_rows;                   // n_kv_heads * n_tiles
  int grid;                     // workgroups
  float scale_log2;             // scale * log2(e)
  float* part_o;   // [chunks_bound][n_heads][head_dim]: sums of a chunk
  float* part_ml;  // [chunks_bound][n_heads][2]: its maximum (log2) and total
  int32_t* info;   // [n_seqs][2]: a session's first chunk, and its chunks (null: one each)
  int* err;
};

struct RopeTab {
  int rot_dim, layout;
  float mscale;
  double turns[128];
};
constexpr int ROPE_TOKENS = 4;  // tokens of a workgroup, one wave's to place each
struct RopeParams {
  HeadRows q, qo, k, v;
  PagedKV kv;
  PagedBatch b;
  const int32_t* token_start;
  const int32_t* positions;  // where there is no cache
  int n_tokens, n_q, n_kv;   // heads per token
  int head_dim;
  int tok;                   // tokens per workgroup
  int runs;                  // pairs of runs per head, and the divisions by it and by the heads
  uint32_t runs_magic, rows_magic;
  int* err;
  RopeTab rope;
};

// c2h_rmsnorm_q8k_dev
struct NormQ8Params {
  const char* x;
  const char* r;
  char* sum;
  int64_t x_stride, r_stride, sum_stride;  // bytes
  const float* w;
  float* y;
  int64_t y_stride;  // floats
  uint8_t* q8k;
  float eps;
  int n_rows, cols;
};

#ifdef __HIPCC__
// Launches on `stream`; arguments checked by the entry points.
void launch_paged_attn(const PagedAttnParams& P, int cache_type, hipStream_t stream);
void launch_rope(const RopeParams& P, int type, int cache_type, bool cached, hipStream_t stream);
void launch_norm_q8(const NormQ8Params& P, int type, hipStream_t stream);
#endif

}  // namespace c2h
