// Operators for many sessions: rotary positions, the paged cache's append
// and its attention (include/c2h.h describes them; none has a counterpart in
// the reference).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "c2h_device.h"
#include "c2h_paged.h"

namespace c2h {

namespace {

// ------------------------------------------------------------ element types

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <class To, class From>
__device__ __forceinline__ To as(From v) {
  return __builtin_bit_cast(To, v);
}

// Two floats as 16-bit numbers of the product's type, rounded to nearest even.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return as<uint32_t>(v);
  } else {
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return as<uint32_t>(v);
  }
}
template <bool BF>
__device__ __forceinline__ float unpack(uint32_t v, int i) {
  if constexpr (BF) return __uint_as_float(i ? v & 0xffff0000u : v << 16);
  return (float)as<f16x2>(v)[i];
}
// Saturating: finite values and infinities beyond 448 store as +-448, NaN
// stays NaN.
__device__ __forceinline__ float e4m3_range(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }
__device__ __forceinline__ uint32_t e4m3_bits4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(a), e4m3_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(c), e4m3_range(d), lo, true);
}

// Errors are rare: one system-scope or into pinned host memory.
__device__ __forceinline__ void report(int* err, int what) {
  __hip_atomic_fetch_or(err, what, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// ------------------------------------------------------ rotation and append

// cos and sin of pos * f_i, times mscale: the angle in turns in 64 bits, of
// which the nearest whole number leaves |fraction| <= 1/2 exactly.
__device__ __forceinline__ float2 cos_sin(const RopeTab& r, int i, int pos) {
  const double t = (double)pos * r.turns[i];
  const float x = (float)(2.0 * (t - __builtin_rint(t)));
  float s, c;
  sincospif(x, &s, &c);
  return make_float2(c * r.mscale, s * r.mscale);
}

// Where a call's token goes: its position, and the byte offset of its slot
// in the pool; false if it goes nowhere.  One whole wave: its lanes look for
// the last session that starts at or before t, 64 starts a round, and the last
// round brings the session's end and length with its start.
__device__ __forceinline__ bool place(const RopeParams& P, int t, int* pos, int64_t* off) {
  const int lane = threadIdx.x & 63;
  int s = t, len;
  int64_t end = (int64_t)t + 1;
  if (P.token_start) {
    int lo = 0, n = P.b.n_seqs;
    while (n > 64) {
      const int step = (n + 63) >> 6;
      const bool before = lane * step < n && P.token_start[lo + lane * step] <= t;
      const int skip = max((int)__popcll(__ballot(before)) - 1, 0) * step;
      lo += skip;
      n = min(step, n - skip);
    }
    const int mine = lo + min(lane, n - 1);
    const int first = P.token_start[mine], after = P.token_start[mine + 1], held = P.b.lens[mine];
    const int at = max((int)__popcll(__ballot(lane < n && first <= t)) - 1, 0);
    s = lo + at;
    end = __builtin_amdgcn_readlane(after, at);
    len = __builtin_amdgcn_readlane(held, at);
    if (t >= end) return false;
  } else {
    len = P.b.lens[s];
  }
  if (len == 0) return false;
  const int64_t p = token_pos(len, t, end);
  if (!length_ok(len, P.b.max_len) || p < 0) {
    if (lane == 0) report(P.err, length_ok(len, P.b.max_len) ? PERR_START : PERR_LENGTH);
    return false;
  }
  const int page = P.b.table[s * P.b.table_stride + (p >> P.kv.page_shift)];
  if (!page_ok(page, P.kv.n_pages)) {
    if (lane == 0) report(P.err, PERR_PAGE);
    return false;
  }
  *pos = (int)p;
  *off = page * P.kv.page_stride + (p & ((1 << P.kv.page_shift) - 1)) * P.kv.token_stride;
  return true;
}

// VEC neighbouring elements as they lie in memory, and as floats.
template <int T, int VEC>
struct Run {
  static constexpr int DW = VEC * type_bytes(T) / 4;
  uint32_t w[DW];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (DW % 4 == 0) {
#pragma unroll
      for (int i = 0; i < DW; i += 4) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(p + 4 * i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else if constexpr (DW == 2) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (DW % 4 == 0) {
#pragma unroll
      for (int i = 0; i < DW; i += 4) *reinterpret_cast<u32x4*>(p + 4 * i) = u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]};
    } else if constexpr (DW == 2) {
      *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    } else {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = T == PT_F32 ? __uint_as_float(w[i % DW]) : unpack<T == PT_BF16>(w[i / 2 % DW], i & 1);
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < DW; ++i) {
      if constexpr (T == PT_F32)
        w[i] = __float_as_uint(x[i]);
      else if constexpr (T == PT_E4M3)
        w[i] = e4m3_bits4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      else
        w[i] = pack2<T == PT_BF16>(x[2 * i], x[2 * i + 1]);
    }
  }
};

// A workgroup takes P.tok consecutive tokens, up to four.  A wave finds a
// token's place and fills its cosines and sines (one 64-bit angle per pair and
// token, in LDS for all heads); then every thread moves pairs of VEC-element
// runs: the two halves of VEC rotated pairs in the half layout, neighbours
// elsewhere, 16 bytes a load at 16 bits.  The first pair's loads are issued
// before the angles, which they do not wait for.
// Bound by memory: 16,384 tokens of 32 heads of 128 (268 MB) 50.4 us, 5.3
// TB/s, where a thread per pair with angles of its own took 151; 92 MB of
// prompts into e4m3 23.5 us, 3.9 TB/s, of which the chain of loads before a
// workgroup's first store (session, page) is the rest.  A step of few tokens
// is that chain: 2.7 us for a rotation, 4.6 for 256 sessions' append.
template <int T, int CT, bool CACHED, int VEC>
__global__ void __launch_bounds__(256) k_rope(RopeParams P) {
  __shared__ float2 cs[ROPE_TOKENS][128];
  __shared__ int64_t slot[ROPE_TOKENS];  // the token's offset in the pool; < 0: none
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t0 = blockIdx.x * P.tok, tok = min(P.tok, P.n_tokens - t0);
  const RopeTab& R = P.rope;
  const int rows = P.n_q + 2 * P.n_kv, items = tok * rows * P.runs;
  const int half = R.rot_dim / 2;

  // pair `it` of runs: its token, row, and the elements its runs begin at
  // (b < 0: only one run)
  struct Item {
    int tt, row, a, b;
    bool turn;
  };
  auto item = [&](int it) {
    Item x;
    const int q = P.runs == 1 ? it : (int)__umulhi((uint32_t)it, P.runs_magic), c = it - q * P.runs;
    x.tt = rows == 1 ? q : (int)__umulhi((uint32_t)q, P.rows_magic);
    x.row = q - x.tt * rows;
    x.turn = x.row < P.n_q + P.n_kv;
    const int e = 2 * c * VEC;
    if (x.turn && R.layout == 0) {
      x.turn = c * VEC < half;
      x.a = x.turn ? c * VEC : e;  // half and rot_dim are whole runs: the copied ones go on at 2 c
      x.b = x.turn ? x.a + half : x.a + VEC;
    } else {
      x.a = e;
      x.b = e + VEC;
    }
    if (x.b >= P.head_dim) x.b = -1;
    return x;
  };
  auto source = [&](const Item& x) {
    const bool is_q = x.row < P.n_q, is_v = x.row >= P.n_q + P.n_kv;
    const HeadRows& S = is_q ? P.q : is_v ? P.v : P.k;
    const int h = is_q ? x.row : is_v ? x.row - P.n_q - P.n_kv : x.row - P.n_q;
    return S.data + (t0 + x.tt) * S.token_stride + h * S.head_stride;
  };
  Item x = item(min(tid, items - 1));
  Run<T, VEC> ra, rb;
  auto load = [&](const Item& y) {
    const char* p = source(y);
    ra.load(p + y.a * type_bytes(T));
    rb.load(p + max(y.b, 0) * type_bytes(T));
  };
  load(x);

  for (int tt = wave; tt < tok; tt += 4) {
    int pos = 0;
    int64_t off = 0;
    if constexpr (CACHED) {
      if (!place(P, t0 + tt, &pos, &off)) off = -1;
      if (lane == 0) slot[tt] = off;
    } else {
      pos = P.positions[t0 + tt];
    }
    for (int i = lane; i < half; i += 64) cs[tt][i] = cos_sin(R, i, pos);
  }
  __syncthreads();

  for (int it = tid; it < items; it += 256) {
    float a[VEC], b[VEC];
    ra.get(a);
    rb.get(b);
    const Item y = x;
    if (it + 256 < items) {
      x = item(it + 256);
      load(x);
    }
    const float2* c = cs[y.tt];
    if (y.turn && R.layout == 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 f = c[y.a + i];
        const float u = a[i] * f.x - b[i] * f.y, v = a[i] * f.y + b[i] * f.x;
        a[i] = u;
        b[i] = v;
      }
    } else if (y.turn) {
      auto turn = [&](float(&z)[VEC], int at) {
        if (at < 0 || at >= R.rot_dim) return;  // rot_dim is whole runs
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const float2 f = c[(at + i) >> 1];
          const float u = z[i] * f.x - z[i + 1] * f.y, v = z[i] * f.y + z[i + 1] * f.x;
          z[i] = u;
          z[i + 1] = v;
        }
      };
      turn(a, y.a);
      turn(b, y.b);
    }
    const bool is_q = y.row < P.n_q, is_v = y.row >= P.n_q + P.n_kv;
    if constexpr (CACHED) {
      const int64_t off = slot[y.tt];
      if (off < 0) continue;
      if (!is_q) {
        const int h = is_v ? y.row - P.n_q - P.n_kv : y.row - P.n_q;
        char* dst = (is_v ? P.kv.v : P.kv.k) + off + h * P.kv.head_stride;
        if constexpr (CT == PT_E4M3) {
          const float* sc = is_v ? P.kv.v_scale : P.kv.k_scale;
          if (sc) {
            const float d = sc[h];
#pragma unroll
            for (int i = 0; i < VEC; ++i) a[i] /= d, b[i] /= d;
          }
        }
        Run<CT, VEC> w;
        w.set(a);
        w.store(dst + y.a * type_bytes(CT));
        w.set(b);
        if (y.b >= 0) w.store(dst + y.b * type_bytes(CT));
        continue;
      }
    }
    char* dst = P.qo.data + (t0 + y.tt) * P.qo.token_stride + y.row * P.qo.head_stride;
    Run<T, VEC> w;
    w.set(a);
    w.store(dst + y.a * type_bytes(T));
    w.set(b);
    if (y.b >= 0) w.store(dst + y.b * type_bytes(T));
  }
}

// --------------------------------------------------------------- attention
//
// One token per session, so every key and value is used once per query head:
// at 16 heads per KV head 8 operations per byte of a 16-bit pool, far below
// what the matrix units do per byte of HBM.  The kernel's work is to keep
// loads in flight, so a wave runs on its own: registers hold its keys and
// values, nothing of them passes through LDS, and it meets the other waves
// once, at its end.
//
//   scores   S[position][head] = K Q^T: a matrix instruction takes the rows
//            of K as a lane loads them (16 bytes of one position per lane);
//            Q lies in LDS in the instruction's order.
//   softmax  running maximum and sum per head in 32 bits.  S leaves lane l
//            with head l % 16 and positions 4 (l / 16) + i, which is how the
//            next product takes P: no value moves between lanes.
//   output   O^T[dim][head] = V^T P^T.  Lane l loads the same elements
//            (16 bytes, at l % 16) of the four positions 4 (l / 16) + i, so
//            its four registers hold a 4-position column of each element, and
//            the columns that the instruction wants come from byte permutes
//            within the lane.  Tile t of a row is then every (elements per
//            lane)-th element, which the epilogue undoes.
//
// 16-bit parts: queries and probabilities of 32 bits are split into 16-bit
// summands (hi = round(x), next = round(x - hi), ...), one matrix
// instruction each.  Three bf16 or two f16 parts carry 24 and 22 bits: all
// that 32-bit outputs show.  Two bf16 parts of P (2^-17) stay below a
// 16-bit output's own rounding.  f16 parts are kept in f16's normal range by
// powers of two: Q by its head's largest element, P by 2^15 (P <= 1 against
// the running maximum), which cancels in O / sum.

// The next part of four numbers, which become what it leaves unless it is the
// last.  INF: an infinite part leaves nothing (rather than the NaN of
// inf - inf); probabilities are finite.
template <bool BF, bool INF>
__device__ __forceinline__ u32x2 part4(float (&a)[4], bool last) {
  const u32x2 v = {pack2<BF>(a[0], a[1]), pack2<BF>(a[2], a[3])};
  if (!last)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float rest = a[i] - unpack<BF>(v[i >> 1], i & 1);
      a[i] = INF && __builtin_isinf(a[i]) ? 0.0f : rest;
    }
  return v;
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as<bf16x8>(a), as<bf16x8>(b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(as<f16x8>(a), as<f16x8>(b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x2 a, u32x2 b, f32x4 c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as<i16x4>(a), as<i16x4>(b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x16f16(as<f16x4>(a), as<f16x4>(b), c, 0, 0, 0);
}

// Four e4m3 as four f16 (exact).
__device__ __forceinline__ u32x2 e4m3_to_f16(uint32_t v) {
  return u32x2{as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v, 1.0f, false)),
               as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v, 1.0f, true))};
}

// Over the four lanes l % 16 of a wave.
__device__ __forceinline__ float max_of_rows(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_rows(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ f32x4 load4(int t, const char* p) {
  if (t == PT_F32) return *reinterpret_cast<const f32x4*>(p);
  const u32x2 u = *reinterpret_cast<const u32x2*>(p);
  if (t == PT_BF16) return f32x4{unpack<true>(u.x, 0), unpack<true>(u.x, 1), unpack<true>(u.y, 0), unpack<true>(u.y, 1)};
  return f32x4{unpack<false>(u.x, 0), unpack<false>(u.x, 1), unpack<false>(u.y, 0), unpack<false>(u.y, 1)};
}
__device__ __forceinline__ void store4(int t, char* p, f32x4 v) {
  if (t == PT_F32)
    *reinterpret_cast<f32x4*>(p) = v;
  else if (t == PT_BF16)
    *reinterpret_cast<u32x2*>(p) = u32x2{pack2<true>(v.x, v.y), pack2<true>(v.z, v.w)};
  else
    *reinterpret_cast<u32x2*>(p) = u32x2{pack2<false>(v.x, v.y), pack2<false>(v.z, v.w)};
}

// exp2(m - mu) where m may be -inf (nothing summed: 0).
__device__ __forceinline__ float weight(float m, float mu) { return __builtin_amdgcn_exp2f(m - mu); }
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

constexpr float MINUS_INF = -__builtin_inff();

// A load of keys or values.  They are used once: where a head's tokens lie
// back to back in a page (STREAM) they bypass the last-level cache, 8 x 32,768
// positions of f16 in pages of 64 in 163 us for 183, 128 sessions of e4m3 44.3
// for 46.0.  Where heads alternate within a page other workgroups soon read
// the neighbouring bytes, and plain loads are the faster ones (32 sessions of
// 8,192, 8 KV heads of e4m3: 101 us for 110).
template <bool STREAM, class T>
__device__ __forceinline__ T load_kv(const char* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  return *reinterpret_cast<const T*>(p);
}

// CT: the pool's type; HD: head_dim rounded up to 64, 128 or 256; FULL:
// head_dim == HD; PRECISE: the 32-bit split above (for outputs or queries
// that need it).
template <int CT, int HD, bool FULL, bool PRECISE>
struct Attn {
  static constexpr int ES = type_bytes(CT);
  static constexpr bool F32 = CT == PT_F32, BF = CT == PT_BF16, F8 = CT == PT_E4M3;
  static constexpr int KC = HD * ES / 64;              // 16-byte loads of a key per lane
  static constexpr int VB = HD * ES / 16 < 16 ? HD * ES / 16 : 16;  // bytes of a value load
  static constexpr int VW = VB / 4, VE = VB / ES;      // its dwords, its elements
  static constexpr int NV = HD * ES / 16 / VB;         // loads of a value per lane
  static constexpr int NO = HD / 16;                   // output tiles: NV * VE
  static constexpr int NT = attn_tiles(CT, HD), STEP = 16 * NT, UNIT = 4 * STEP;
  static_assert(UNIT == attn_unit(CT, HD), "the host's units");
  static constexpr int NQ = F32 ? 1 : PRECISE ? (BF ? 3 : 2) : 1;
  static constexpr int NP = F32 ? 1 : BF && PRECISE ? 3 : 2;
  static constexpr int FR = F32 ? HD / 16 : HD / 32;   // 16-byte fragments of a query per lane
  static constexpr float BIAS = F32 || BF ? 0.0f : 15.0f;
  static constexpr int DB = HD < 128 ? HD : 128;       // elements that waves join at a time
  static constexpr int OROW = DB + 4;
  static constexpr int Q_BYTES = NQ * FR * 1024, O_BYTES = 4 * 16 * OROW * 4;
  static constexpr int LDS = Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES;
};

// Sum over the lanes up to this one.
__device__ __forceinline__ int scan_of_wave(int x) {
  x += dpp0_i<0x111>(x);  // row_shr:1
  x += dpp0_i<0x112>(x);
  x += dpp0_i<0x114>(x);
  x += dpp0_i<0x118>(x);
  x += dpp0_i<DPP_BCAST15, 0xa>(x);
  x += dpp0_i<DPP_BCAST31, 0xc>(x);
  return x;
}

// How a batch is cut, found by every wave from the lengths: the host does not
// know them, and a grid over max_len would start a workgroup per chunk that a
// session could have (64 sessions of 30 to 8,000: most of them empty).  Lane l
// looks after sessions [l * per, (l + 1) * per).
struct Cut {
  int per, units;   // units: positions of a chunk, in units
  int len;          // per == 1: the lane's length
  int upto;         // chunks of the sessions up to this lane's last
  int total;
};
template <int UNIT>
__device__ __forceinline__ int session_units(int len, int max_len, int window) {
  return units_of(attended(length_ok(len, max_len) ? len : 0, window), UNIT);
}
template <int UNIT>
__device__ __forceinline__ Cut cut_batch(const int32_t* lens, int n_seqs, int max_len, int window, int n_rows,
                                         bool split) {
  const int lane = threadIdx.x & 63;
  Cut c{(n_seqs + 63) >> 6, 1, 0, 0, n_seqs};
  if (!split) return c;  // no session is longer than a unit
  auto units_at = [&](int len) { return session_units<UNIT>(len, max_len, window); };
  if (c.per == 1) {
    c.len = lane < n_seqs ? lens[lane] : 0;
    c.units = chunk_units(__builtin_amdgcn_readlane(scan_of_wave(units_at(c.len)), 63), n_rows);
    c.upto = scan_of_wave(lane < n_seqs ? chunks_of(units_at(c.len), c.units) : 0);
  } else {
    // eight lengths of the lane's at a time, loaded together
    int v[8];
    auto load8 = [&](int k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = lens[min(lane * c.per + k + i, n_seqs - 1)];
    };
    auto sum8 = [&](int k, auto of) {
      int sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += k + i < c.per && lane * c.per + k + i < n_seqs ? of(v[i]) : 0;
      return sum;
    };
    int mine = 0, n = 0;  // below 2^31: 1024 sessions of 2^17 units
    for (int k = 0; k < c.per; k += 8) {
      load8(k);
      mine += sum8(k, units_at);
    }
    int64_t units = 0;
    for (int m = 0; m < 64; ++m) units += __builtin_amdgcn_readlane(mine, m);
    c.units = chunk_units(units, n_rows);
    for (int k = 0; k < c.per; k += 8) {
      if (c.per > 8) load8(k);
      n += sum8(k, [&](int len) { return chunks_of(units_at(len), c.units); });
    }
    c.upto = scan_of_wave(n);
  }
  c.total = __builtin_amdgcn_readlane(c.upto, 63);
  return c;
}

// One new token per session: workgroups take chunks in turn, a chunk's steps
// go round its four waves, and a row of one chunk is written here, others'
// parts are joined by k_paged_join.
// Bound by memory where there is much to read: 8 sessions of 32,768 positions,
// 16/8 heads of 128, f16 in pages of 64 (1,059 MB) 163 us, 6.5 TB/s, what a
// plain streaming read of 4 GiB reaches.  Smaller calls lose to the chain
// length -> page -> keys at the start of a workgroup's chunks, of a few steps
// each: 64 sessions of 30 to 8,000, 12/2 heads, bf16 (92 MB) 18.7 us, 4.9 TB/s
// (a plain read of 100 MB: 5.6); 128 of up to 4,096, 16/2 heads, e4m3 (161 MB)
// 39.8 us, 4.1 TB/s.  One session of 41 positions, 5.0 us, and one of 4,096,
// 7.8 us, are that chain.  The matrix units are busy 8 %, the VALU 20 to 37 %.
// 16 KB a wave and two workgroups to a CU keep 32 MB in flight, more than the
// memory's latency times its rate; 512 workgroups and 1,024 chunks took 21.2
// us where 512 chunks took 25.1 and 2,048 24.6 (64 sessions, with the join).
// More than 16 query heads to a KV head are tiles of 16, a workgroup each that
// reads the keys and values again: 400 MB in 145 us at 24/1 heads of 128 for
// 83 at 16/1, and in 143 (plain loads) and 167 us (streamed ones, which the
// second tile does not find in the cache) at 40/2 heads of 64 for 85 and 80 at
// 14/2.
//
// The leading arguments arrive in registers at wave start (kernel-argument
// preload).  shape: log2 of the page size; from bit 4: whether sessions can
// have several chunks; from bit 5: n_tiles; from bit 14: n_kv_heads.
// The block P is read where it is used, through its place in the kernel's
// arguments: kept in registers over the loop, its fields spill.
struct AttnLead {
  const int32_t *lens, *table;
  int64_t table_stride;
  int max_len, window;
  uint32_t shape;
  int n_seqs;
};
static_assert(sizeof(AttnLead) % alignof(PagedAttnParams) == 0, "P follows the leading arguments");
using Args = const __attribute__((address_space(4))) PagedAttnParams*;
template <int CT, int HD, bool FULL, bool PRECISE, bool STREAM>
__global__ void __launch_bounds__(256, HD == 256 && (CT == PT_F32 || !FULL) ? 1 : 2)
    k_paged_attn(const int32_t* lens, const int32_t* table, int64_t table_stride, int max_len, int window, uint32_t shape,
                 int n_seqs, PagedAttnParams P) {
  using A = Attn<CT, HD, FULL, PRECISE>;
  constexpr int KC = A::KC, NT = A::NT, NV = A::NV, VW = A::VW, VE = A::VE, NO = A::NO, FR = A::FR, NQ = A::NQ, NP = A::NP;
  constexpr bool BF = A::BF;
  __shared__ __align__(16) char lds[A::LDS];
  __shared__ float mul[16], wm[4][16], wl[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, j = lane >> 4;
  auto fresh = [&]() {
    auto* lead = (const __attribute__((address_space(4))) AttnLead*)__builtin_amdgcn_kernarg_segment_ptr();
    Args a = (Args)(lead + 1), b;
    asm volatile("" : "=s"(b) : "0"(a));
    return b;
  };
  const int shift = shape & 15, n_tiles = (shape >> 5) & 511, n_rows = (shape >> 14) * n_tiles;
  const bool split = shape & 16;
  // One field of each cache line of the block, loaded together with the lengths: the reads
  // further down then hit (1x4096 10.43 -> 10.09 us, 64 ragged sessions 22.0 -> 21.5, 128 of
  // e4m3 43.7 -> 43.3).
  const int near0 = P.kv.n_pages, near1 = P.n_heads, near2 = P.b.n_seqs;
  const float* near3 = P.part_o;
  const Cut cut = cut_batch<A::UNIT>(lens, n_seqs, max_len, window, n_rows, split);
  asm volatile("" ::"s"(near0), "s"(near1), "s"(near2), "s"(near3));
  const int csize = cut.units * A::UNIT, items = cut.total * n_rows;

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
  // the item's session and chunk
  Args args = fresh();
  const int unit = item / n_rows, row = item - unit * n_rows;
  int s = unit, chunk = 0, len = 0;
  if (!split) {
    len = lens[s];
  } else {
    const int owner = __popcll(__ballot(cut.upto <= unit));
    chunk = unit - (owner ? __builtin_amdgcn_readlane(cut.upto, owner - 1) : 0);
    s = owner;
    len = __builtin_amdgcn_readlane(cut.len, owner);
    if (cut.per > 1) {
      len = 0;
      for (s = owner * cut.per; s < min((owner + 1) * cut.per, n_seqs); s += 64) {  // 64 at a time; one of them has it
        const bool mine = s + lane < n_seqs && s + lane < (owner + 1) * cut.per;
        const int one = mine ? lens[s + lane] : 0;
        const int upto = scan_of_wave(mine ? chunks_of(session_units<A::UNIT>(one, max_len, window), cut.units) : 0);
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (chunk < all) {
          const int at = __popcll(__ballot(upto <= chunk));
          chunk -= at ? __builtin_amdgcn_readlane(upto, at - 1) : 0;
          len = __builtin_amdgcn_readlane(one, at);
          s += at;
          break;
        }
        chunk -= all;
      }
      s = min(s, n_seqs - 1);
    }
  }
  const bool ok = length_ok(len, max_len);
  const Span span = attended(ok ? len : 0, window);
  const int n = chunks_of(units_of(span, A::UNIT), cut.units);
  const int base0 = chunk_base(span, csize, chunk), c0 = max(base0, span.lo), c1 = min(base0 + csize, span.hi);
  const int last = c1 - 1;
  if (split && row == 0 && chunk == 0 && tid == 0) {
    args->info[2 * s] = unit;
    args->info[2 * s + 1] = n;
  }
  // lane i holds page p0 + i, and the next 64 that the wave's steps come to
  // are on their way
  const int first = base0 + wave * A::STEP;  // the wave's steps: first, first + UNIT, ...
  int p0 = c0 >> shift, beyond = first_step_beyond(p0, shift, first, A::STEP, A::UNIT);
  auto held_pages = [&](int from) { return from + lane <= last >> shift && c1 > c0; };
  auto load_pages = [&](int from) { return held_pages(from) ? table[s * table_stride + from + lane] : 0; };
  const int page = load_pages(p0);
  int next_page = beyond < c1 ? load_pages(beyond >> shift) : 0;

  const int kvh = n_tiles == 1 ? row : row / n_tiles;
  const int h0 = kvh * args->group + (row - kvh * n_tiles) * ATTN_HEADS;
  const int nh = min(ATTN_HEADS, (kvh + 1) * args->group - h0);
  const int hd = FULL ? HD : args->kv.head_dim;
  constexpr int EPT = HD / 16;  // elements of the queries that a thread brings
  const int qhead = tid >> 4, qd0 = (tid & 15) * EPT;
  f32x4 q[EPT / 4];
#pragma unroll
  for (int g = 0; g < EPT / 4; ++g) {
    const bool have = qhead < nh && (FULL || qd0 + 4 * g < hd);
    q[g] = have ? load4(args->type, args->q.data + s * args->q.token_stride + (h0 + qhead) * args->q.head_stride +
                                    (int64_t)(qd0 + 4 * g) * (args->type == PT_F32 ? 4 : 2))
                : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  bool fail = !ok || __any(held_pages(p0) && !page_ok(page, args->kv.n_pages));
  int64_t page_off = page * args->kv.page_stride + kvh * args->kv.head_stride;

  u32x4 K[NT][KC];
  uint32_t V[NT][4][NV][VW];
  const int rowb = hd * A::ES, mask = (1 << shift) - 1;
  const uint32_t ts = (uint32_t)args->kv.token_stride;  // below 2^31
  // Positions outside [c0, c1) are read as the nearest inside, and masked
  // in the scores; elements past head_dim as the row's first, against zeros
  // of Q and into output tiles that are not stored.
  int from = c0, to = last;
  auto inside = [&](int pos) { return min(max(pos, from), to); };
  auto page_of = [&](int pos) {
    const int at = ((pos >> shift) - p0) * 4;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)page_off);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)(page_off >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
  };
  auto in_page = [&](int pos) { return (int64_t)((uint64_t)(uint32_t)(pos & mask) * ts); };
  auto load_k = [&](int base) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int pos = inside(base + 16 * t + r);
      const char* row = args->kv.k + page_of(pos) + in_page(pos);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        int off = c * 64 + j * 16;
        if constexpr (!FULL) off = off < rowb ? off : 0;
        K[t][c] = load_kv<STREAM, u32x4>(row + off);
      }
    }
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // one page holds those of the four positions that are inside
      const int first = base + 16 * t + 4 * j;
      const char* at = args->kv.v + page_of(inside(first));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* row = at + in_page(inside(first + i));
#pragma unroll
        for (int b = 0; b < NV; ++b) {
          int off = b * 16 * A::VB + r * A::VB;
          if constexpr (!FULL) off = off < rowb ? off : 0;
          if constexpr (VW == 4) {
            const u32x4 v = load_kv<STREAM, u32x4>(row + off);
#pragma unroll
            for (int w = 0; w < 4; ++w) V[t][i][b][w] = v[w];
          } else if constexpr (VW == 2) {
            const u32x2 v = load_kv<STREAM, u32x2>(row + off);
            V[t][i][b][0] = v.x;
            V[t][i][b][1] = v.y;
          } else {
            V[t][i][b][0] = load_kv<STREAM, uint32_t>(row + off);
          }
        }
      }
    }
  };
  const bool work = !fail && first < c1;
  if (work) {
    load_k(first);
    load_v(first);
  }

  // the queries, split into the parts of the product
  __syncthreads();  // the item before is done with LDS
  {
    int e = 0;
    if constexpr (A::BIAS != 0.0f) {
      float top = 0.0f;
#pragma unroll
      for (int g = 0; g < EPT / 4; ++g)
        top = fmaxf(fmaxf(top, fmaxf(fabsf(q[g].x), fabsf(q[g].y))), fmaxf(fabsf(q[g].z), fabsf(q[g].w)));
#pragma unroll
      for (int m = 1; m < 16; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
      if (top > 0.0f && top < __builtin_inff()) {
        e = 14 + 127 - (int)(__float_as_uint(top) >> 23);
        e = min(max(e, -115), 100);
      }
    }
    if ((tid & 15) == 0) {
      const float ks = A::F8 && args->kv.k_scale ? args->kv.k_scale[kvh] : 1.0f;
      mul[qhead] = ldexpf(args->scale_log2 * ks, -e);
    }
#pragma unroll
    for (int g = 0; g < EPT / 4; ++g) {
      const int d = qd0 + 4 * g;
      if constexpr (A::F32) {
        *reinterpret_cast<f32x4*>(lds + ((d >> 4) * 64 + ((d >> 2) & 3) * 16 + qhead) * 16) = q[g];
      } else {
        const int f = A::F8 ? 2 * (d >> 6) + ((d >> 3) & 1) : d >> 5, jj = A::F8 ? (d >> 4) & 3 : (d >> 3) & 3;
        char* at = lds + (f * 64 + jj * 16 + qhead) * 16 + ((d >> 2) & 1) * 8;
        float a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = A::BIAS != 0.0f ? ldexpf(q[g][i], e) : q[g][i];
#pragma unroll
        for (int p = 0; p < NQ; ++p) {
          *reinterpret_cast<u32x2*>(at + p * FR * 1024) = part4<BF, true>(a, p + 1 == NQ);
        }
      }
    }
  }
  __syncthreads();
  const float smul = mul[r];

  f32x4 o[NO];
#pragma unroll
  for (int t = 0; t < NO; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = MINUS_INF, l = 0.0f;

  if (work) {
    for (int base = first; base < c1; base += A::UNIT) {
      const int next = base + A::UNIT;
      // scores
      f32x4 S[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) S[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < NQ; ++p)
#pragma unroll
        for (int f = 0; f < FR; ++f) {
          const u32x4 q = *reinterpret_cast<const u32x4*>(lds + ((p * FR + f) * 64 + lane) * 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (A::F32) {
              const f32x4 a = as<f32x4>(K[t][f]), b = as<f32x4>(q);
#pragma unroll
              for (int i = 0; i < 4; ++i) S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], S[t], 0, 0, 0);
            } else if constexpr (A::F8) {
              const u32x2 lo = e4m3_to_f16(K[t][f / 2][(f & 1) * 2]), hi = e4m3_to_f16(K[t][f / 2][(f & 1) * 2 + 1]);
              S[t] = mfma32<BF>(u32x4{lo.x, lo.y, hi.x, hi.y}, q, S[t]);
            } else {
              S[t] = mfma32<BF>(K[t][f], q, S[t]);
            }
          }
        }
      if (next == beyond && next < c1) {
        Args pool = fresh();
        p0 = beyond >> shift;
        if (__any(held_pages(p0) && !page_ok(next_page, pool->kv.n_pages))) {
          fail = true;
          break;
        }
        page_off = next_page * pool->kv.page_stride + kvh * pool->kv.head_stride;
        beyond = first_step_beyond(p0, shift, next, A::STEP, A::UNIT);
        next_page = beyond < c1 ? load_pages(beyond >> shift) : 0;
      }
      if (next >= c1) from = to = max(base, c0);  // no next step: one row, unused
      load_k(next);
      // softmax
      const uint32_t at = (uint32_t)(base + 4 * j - c0), held = (uint32_t)(c1 - c0);
      float top = MINUS_INF;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S[t][i] = at + (16 * t + i) < held ? S[t][i] * smul : MINUS_INF;
          top = fmaxf(top, S[t][i]);
        }
      if (__any(top > m)) {
        const float mn = fmaxf(m, max_of_rows(top)), a = weight(m, finite_max(mn));
        m = mn;
        l *= a;
#pragma unroll
        for (int t = 0; t < NO; ++t) o[t] *= a;
      }
      const float mb = finite_max(m) - A::BIAS;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S[t][i] = __builtin_amdgcn_exp2f(S[t][i] - mb);
          l += S[t][i];
        }
      // output
      if constexpr (A::F32) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < NV; ++b)
#pragma unroll
              for (int w = 0; w < VW; ++w)
                o[b * VE + w] =
                    __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(V[t][i][b][w]), S[t][i], o[b * VE + w], 0, 0, 0);
      } else {
        u32x2 p[NT][NP];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float a[4] = {S[t][0], S[t][1], S[t][2], S[t][3]};
#pragma unroll
          for (int q = 0; q < NP; ++q) p[t][q] = part4<BF, false>(a, q + 1 == NP);
        }
#pragma unroll
        for (int b = 0; b < NV; ++b)
#pragma unroll
          for (int w = 0; w < VE / 2; ++w) {  // elements 2w and 2w + 1 of the load
            u32x2 col[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              uint32_t x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (A::F8)
                  x[i] = e4m3_to_f16(V[t][i][b][w / 2])[w & 1];
                else
                  x[i] = V[t][i][b][w];
              }
              col[t][0] = u32x2{__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u)};
              col[t][1] = u32x2{__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f32x4& acc = o[b * VE + 2 * w + h];
#pragma unroll
              for (int q = 0; q < NP; ++q) {
                if constexpr (NT % 2 == 0) {
#pragma unroll
                  for (int t = 0; t < NT; t += 2)
                    acc = mfma32<BF>(u32x4{col[t][h].x, col[t][h].y, col[t + 1][h].x, col[t + 1][h].y},
                                     u32x4{p[t][q].x, p[t][q].y, p[t + 1][q].x, p[t + 1][q].y}, acc);
                } else {
#pragma unroll
                  for (int t = 0; t < NT; ++t) acc = mfma16<BF>(col[t][h], p[t][q], acc);
                }
              }
            }
          }
      }
      load_v(next);
    }
    l = sum_of_rows(l);
  }

  Args at_end = fresh();
  // A bad page or length: the wave's total is NaN, and so is the row.
  if (fail) {
    m = MINUS_INF;
    l = __builtin_nanf("");
    if (lane == 0) report(at_end->err, ok ? PERR_PAGE : PERR_LENGTH);
  }

  // the waves' sums, brought to their common maximum, DB elements at a time
  if (lane < 16) {
    wm[wave][r] = m;
    wl[wave][r] = l;
  }
  float* os = reinterpret_cast<float*>(lds);
  const float vs = A::F8 && at_end->kv.v_scale ? at_end->kv.v_scale[kvh] : 1.0f;
#pragma unroll
  for (int d0 = 0; d0 < HD; d0 += A::DB) {
    __syncthreads();  // the queries, or the elements before, are read
    if (r < nh) {
#pragma unroll
      for (int t = 0; t < NO; t += 4) {
        // tiles t .. t+3 of load b: elements row * VE + t % VE + 0 .. 3 of its 16 VE
        const int b = t / VE;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = b * 16 * VE + (4 * j + i) * VE + t % VE - d0;
          if (d >= 0 && d < A::DB)
            *reinterpret_cast<f32x4*>(os + (wave * 16 + r) * A::OROW + d) =
                f32x4{o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]};
        }
      }
    }
    __syncthreads();
    for (int it = tid; it < nh * (A::DB / 4); it += 256) {
      const int head = it / (A::DB / 4), d = (it % (A::DB / 4)) * 4;
      if (!FULL && d0 + d >= hd) continue;
      const float top = fmaxf(fmaxf(wm[0][head], wm[1][head]), fmaxf(wm[2][head], wm[3][head])), mu = finite_max(top);
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float a = weight(wm[w][head], mu);
        total += wl[w][head] * a;
        sum += *reinterpret_cast<const f32x4*>(os + (w * 16 + head) * A::OROW + d) * a;
      }
      if (n == 1) {
        const float inv = total == 0.0f ? 0.0f : vs / total;
        store4(at_end->type, at_end->out.data + s * at_end->out.token_stride + (h0 + head) * at_end->out.head_stride +
                           (int64_t)(d0 + d) * (at_end->type == PT_F32 ? 4 : 2), sum * inv);
      } else {
        const int64_t part = (int64_t)unit * at_end->n_heads + h0 + head;
        *reinterpret_cast<f32x4*>(at_end->part_o + part * hd + d0 + d) = sum * vs;
        if (d0 + d == 0) {
          at_end->part_ml[part * 2] = top;
          at_end->part_ml[part * 2 + 1] = total;
        }
      }
    }
  }
  }
}

// Joins the chunks of a row: the sums brought to the common maximum (3.5 us
// for 16 rows of 32 chunks, 5 us for 768 or 2,048 rows of a few; a join in the
// first launch, by the row's last workgroup, was slower: 26.7 us in all for 22
// at 64 sessions).  One
// workgroup per row; HDP / 4 threads hold the row's elements, and 1024 / HDP
// groups of them take every so-manieth chunk.
template <int HDP>
__global__ void __launch_bounds__(256) k_paged_join(const int32_t* info, const float* part_o, const float* part_ml,
                                                    PagedAttnParams P) {
  constexpr int LANES = HDP / 4, GROUPS = 256 / LANES, AHEAD = 4;
  __shared__ __align__(16) float part[GROUPS][HDP + 4];
  __shared__ float tmp[4];
  const int head = blockIdx.x, s = blockIdx.y, hd = P.kv.head_dim, tid = threadIdx.x;
  const int g = tid / LANES, d = (tid % LANES) * 4, dc = min(d, hd - 4);
  const int n = info[2 * s + 1];
  if (n <= 1) return;
  const int64_t first = (int64_t)info[2 * s] * P.n_heads + head;
  auto ml = [&](int i) { return *reinterpret_cast<const float2*>(part_ml + (first + (int64_t)i * P.n_heads) * 2); };
  auto sums = [&](int i) { return *reinterpret_cast<const f32x4*>(part_o + (first + (int64_t)i * P.n_heads) * hd + dc); };
  float2 x[AHEAD];
  f32x4 v[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = min(g + k * GROUPS, n - 1);
    x[k] = ml(i);
    v[k] = sums(i);
  }
  float m = MINUS_INF;
  for (int i = tid; i < n; i += 256) m = fmaxf(m, ml(i).x);
  for (int k = 32; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
  if ((tid & 63) == 0) tmp[tid >> 6] = m;
  __syncthreads();
  const float mu = finite_max(fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3])));
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  float l = 0.0f;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (g + k * GROUPS < n) {
      const float w = weight(x[k].x, mu);
      l += x[k].y * w;
      a += v[k] * w;
    }
  for (int i = g + AHEAD * GROUPS; i < n; i += GROUPS) {
    const float2 y = ml(i);
    const float w = weight(y.x, mu);
    l += y.y * w;
    a += sums(i) * w;
  }
  *reinterpret_cast<f32x4*>(&part[g][d]) = a;
  if (d == 0) part[g][HDP] = l;
  __syncthreads();
  if (g == 0 && d < hd) {
    l = 0.0f;
    a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      a += *reinterpret_cast<const f32x4*>(&part[i][d]);
      l += part[i][HDP];
    }
    // no weight at all: zeros, but the NaN of a bad table stays
    store4(P.type, P.out.data + s * P.out.token_stride + head * P.out.head_stride + (int64_t)d * (P.type == PT_F32 ? 4 : 2),
           l == 0.0f ? a * 0.0f : a / l);
  }
}

// The same for batches of many rows, most of a few chunks or one: HDP / 4
// threads to a row, nothing shared between them.  From 2,048 rows (128
// sessions of e4m3: 43.7 us in all for 45.0; 500 sessions of 20 to 900, 8,000
// rows: 33.2 for 35.4); at 768 rows of up to 30 chunks the row's one thread
// group is the slower one (25.0 for 22.1).
template <int HDP>
__global__ void __launch_bounds__(256) k_paged_join_rows(const int32_t* info, const float* part_o, const float* part_ml, int rows,
                                                         PagedAttnParams P) {
  constexpr int LANES = HDP / 4, ROWS = 256 / LANES, AHEAD = 4;
  const int row = blockIdx.x * ROWS + threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4, hd = P.kv.head_dim;
  if (row >= rows || d >= hd) return;
  const int s = row / P.n_heads, head = row - s * P.n_heads;
  const int2 where = *reinterpret_cast<const int2*>(info + 2 * s);
  const int n = where.y;
  if (n <= 1) return;
  const int64_t first = (int64_t)where.x * P.n_heads + head;
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  float m = MINUS_INF, l = 0.0f;
  for (int i0 = 0; i0 < n; i0 += AHEAD) {
    float2 x[AHEAD];
    f32x4 v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t part = first + (int64_t)min(i0 + k, n - 1) * P.n_heads;
      x[k] = *reinterpret_cast<const float2*>(part_ml + part * 2);
      v[k] = *reinterpret_cast<const f32x4*>(part_o + part * hd + d);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i0 + k >= n) x[k] = make_float2(MINUS_INF, 0.0f), v[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      top = fmaxf(top, x[k].x);
    }
    const float mu = finite_max(top), was = weight(m, mu);
    a *= was;
    l *= was;
    m = top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float w = weight(x[k].x, mu);
      a += v[k] * w;
      l += x[k].y * w;
    }
  }
  // no weight at all: zeros, but the NaN of a bad table stays
  store4(P.type, P.out.data + s * P.out.token_stride + head * P.out.head_stride + (int64_t)d * (P.type == PT_F32 ? 4 : 2),
         l == 0.0f ? a * 0.0f : a / l);
}

template <int CT, int HD, bool FULL, bool PRECISE, bool STREAM>
void launch_attn_as(const PagedAttnParams& P, hipStream_t st) {
  const uint32_t shape = (uint32_t)P.kv.page_shift | (P.info ? 16u : 0u) | (uint32_t)P.n_tiles << 5 | (uint32_t)P.kv.n_kv_heads << 14;
  hipLaunchKernelGGL((k_paged_attn<CT, HD, FULL, PRECISE, STREAM>), dim3(P.grid), dim3(256), 0, st, P.b.lens, P.b.table,
                     P.b.table_stride, P.b.max_len, P.window, shape, P.b.n_seqs, P);
  if (!P.info) return;
  const int rows = P.n_heads * P.b.n_seqs;
  if (rows >= ATTN_MANY_ROWS)
    hipLaunchKernelGGL(k_paged_join_rows<HD>, dim3((rows + 1023 / HD) / (1024 / HD)), dim3(256), 0, st, P.info, P.part_o,
                       P.part_ml, rows, P);
  else
    hipLaunchKernelGGL(k_paged_join<HD>, dim3(P.n_heads, P.b.n_seqs), dim3(256), 0, st, P.info, P.part_o, P.part_ml, P);
}

// Queries and outputs that a single 16-bit part holds take the shorter
// split: the pool's own type, and either 16-bit type on f16 and e4m3 pools
// (a bf16 query fits f16's bits once its range is brought in).  Widths that
// fill no template take the longer split and plain loads whatever the types,
// one kernel a pool type and template: the second product is hidden behind the
// loads there too (400 MB of bf16, heads' tokens back to back: 10/5 heads of 80
// 84 us with bf16 rows and with f32, 6/2 of 96 79, 8/4 of 192 94; full widths
// of 128 and 256 83 and 75).
template <int CT, int HD>
void launch_attn_hd(const PagedAttnParams& P, hipStream_t st) {
  if (P.kv.head_dim != HD) return launch_attn_as<CT, HD, false, true, false>(P, st);
  const bool stream = P.kv.token_stride == HD * type_bytes(CT);
  if constexpr (CT != PT_F32) {
    if (CT == PT_BF16 ? P.type == PT_BF16 : P.type != PT_F32)
      return stream ? launch_attn_as<CT, HD, true, false, true>(P, st) : launch_attn_as<CT, HD, true, false, false>(P, st);
  }
  return stream ? launch_attn_as<CT, HD, true, true, true>(P, st) : launch_attn_as<CT, HD, true, true, false>(P, st);
}
template <int CT>
void launch_attn_t(const PagedAttnParams& P, hipStream_t st) {
  if (P.kv.head_dim <= 64)
    launch_attn_hd<CT, 64>(P, st);
  else if (P.kv.head_dim <= 128)
    launch_attn_hd<CT, 128>(P, st);
  else
    launch_attn_hd<CT, 256>(P, st);
}

}  // namespace

void launch_paged_attn(const PagedAttnParams& P, int cache_type, hipStream_t st) {
  switch (cache_type) {
    case PT_F32: launch_attn_t<PT_F32>(P, st); break;
    case PT_F16: launch_attn_t<PT_F16>(P, st); break;
    case PT_BF16: launch_attn_t<PT_BF16>(P, st); break;
    default: launch_attn_t<PT_E4M3>(P, st); break;
  }
}

namespace {
template <int T, int CT, bool CACHED>
void launch_rope_as(RopeParams P, hipStream_t st) {
  // the halves of a rotated head are whole runs of 8 elements, or of 4
  const bool narrow = P.rope.layout == 0 && P.rope.rot_dim % 16 != 0;
  const int vec = narrow ? 4 : 8;
  const int rows = P.n_q + 2 * P.n_kv;
  P.runs = (P.head_dim / vec + 1) / 2;
  // x / d = (x * ceil(2^32 / d)) >> 32 for x up to 4 * rows * runs, far below 2^32 / d
  P.runs_magic = (uint32_t)(((1ull << 32) + P.runs - 1) / P.runs);
  P.rows_magic = (uint32_t)(((1ull << 32) + rows - 1) / rows);
  // two items a thread once there are enough workgroups: 16,384 tokens of 32
  // heads (256 items each) 50.4 us by two tokens, 53.2 by four, 53.8 by one;
  // prompts into a pool of 2 KV heads (160 items) 24.7, 23.5 and 29.1
  P.tok = std::min({std::max(P.n_tokens / 1024, 1), (511 + rows * P.runs) / (rows * P.runs), ROPE_TOKENS});
  const dim3 grid((P.n_tokens + P.tok - 1) / P.tok);
  if (narrow)
    hipLaunchKernelGGL((k_rope<T, CT, CACHED, 4>), grid, dim3(256), 0, st, P);
  else
    hipLaunchKernelGGL((k_rope<T, CT, CACHED, 8>), grid, dim3(256), 0, st, P);
}
template <int T>
void launch_rope_t(const RopeParams& P, int cache_type, bool cached, hipStream_t st) {
  if (!cached)
    launch_rope_as<T, T, false>(P, st);
  else if (cache_type == PT_F32)
    launch_rope_as<T, PT_F32, true>(P, st);
  else if (cache_type == PT_F16)
    launch_rope_as<T, PT_F16, true>(P, st);
  else if (cache_type == PT_BF16)
    launch_rope_as<T, PT_BF16, true>(P, st);
  else
    launch_rope_as<T, PT_E4M3, true>(P, st);
}
}  // namespace

void launch_rope(const RopeParams& P, int type, int cache_type, bool cached, hipStream_t st) {
  if (type == PT_F32)
    launch_rope_t<PT_F32>(P, cache_type, cached, st);
  else if (type == PT_F16)
    launch_rope_t<PT_F16>(P, cache_type, cached, st);
  else
    launch_rope_t<PT_BF16>(P, cache_type, cached, st);
}

}  // namespace c2h
