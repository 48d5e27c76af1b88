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
constexpr int ATTN_HEADS = 16;         // query heads of a workgroup: columns of the matrix instruction
constexpr int ATTN_MAX_CHUNK = 1024;   // positions of a workgroup
constexpr int ATTN_TAB = ATTN_MAX_CHUNK / PAGED_MIN_PAGE + 1;  // pages a chunk can touch

// The positions [lo, hi) that a session of `len` positions attends, `window`
// of them at most (0: all).
struct Span {
  int lo, hi;
};
C2H_HD inline Span attended(int len, int window) {
  return Span{window > 0 && len > window ? len - window : 0, len};
}
// The span's chunks begin at multiples of `chunk` from its first position
// rounded down to a multiple of 4, so that four positions a lane reads
// together lie in one page; the first chunk's begin at s.lo.
constexpr int SPAN_ALIGN = 4;
C2H_HD inline int chunk_base(Span s, int chunk, int i) { return (s.lo & ~(SPAN_ALIGN - 1)) + i * chunk; }
C2H_HD inline int chunks_of(Span s, int chunk) {
  return (int)(((int64_t)s.hi - (s.lo & ~(SPAN_ALIGN - 1)) + chunk - 1) / chunk);
}
// Chunks of the longest span of a launch: sessions of at most max_len.
C2H_HD inline int most_chunks(int max_len, int window, int chunk) {
  return window > 0 && window < max_len ? chunks_of(Span{0, window + SPAN_ALIGN - 1}, chunk) : chunks_of(Span{0, max_len}, chunk);
}

// Positions per workgroup for a batch of n_rows (session, KV head, head
// tile) rows whose spans are at most `span`.
inline int attn_chunk(int64_t n_rows, int span) {
  int chunk = ATTN_MAX_CHUNK;
  while (chunk > 128 && n_rows * ((span + chunk - 1) / chunk) < 1024) chunk /= 2;
  return chunk;
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
  int chunk, n_chunks;          // positions per workgroup; chunks of the longest session
  float scale_log2;             // scale * log2(e)
  float* part_o;   // [n_seqs][n_heads][n_chunks][head_dim], where n_chunks > 1
  float* part_ml;  // [n_seqs][n_heads][n_chunks][2]: running maximum (log2) and sum
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
