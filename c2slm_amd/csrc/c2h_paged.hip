// Operators for many sessions: rotary positions, the paged cache's append
// and its attention (include/c2h.h describes them; none has a counterpart in
// the reference).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "c2h_paged.h"

namespace c2h {

namespace {

// ------------------------------------------------------------ element types

template <int T>
__device__ __forceinline__ float load_as_f32(const char* p, int64_t i) {
  if constexpr (T == PT_F32) {
    return reinterpret_cast<const float*>(p)[i];
  } else if constexpr (T == PT_F16) {
    return (float)reinterpret_cast<const _Float16*>(p)[i];
  } else if constexpr (T == PT_BF16) {
    return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  } else {
    return __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(p)[i], 0);
  }
}

// Round to nearest even; NaN stays NaN.
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  const __bf16 b = (__bf16)x;
  return (uint32_t)__builtin_bit_cast(uint16_t, b);
}
// Saturating: finite values and infinities beyond 448 store as +-448.
__device__ __forceinline__ uint32_t e4m3_bits(float x) {
  const float c = x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 0xffu;
}

template <int T>
__device__ __forceinline__ void store_f32(char* p, int64_t i, float x) {
  if constexpr (T == PT_F32) {
    reinterpret_cast<float*>(p)[i] = x;
  } else if constexpr (T == PT_F16) {
    reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
  } else if constexpr (T == PT_BF16) {
    reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)bf16_bits(x);
  } else {
    reinterpret_cast<uint8_t*>(p)[i] = (uint8_t)e4m3_bits(x);
  }
}
__device__ __forceinline__ float load_type(int t, const char* p, int64_t i) {
  return t == PT_F32 ? load_as_f32<PT_F32>(p, i) : t == PT_F16 ? load_as_f32<PT_F16>(p, i) : load_as_f32<PT_BF16>(p, i);
}
__device__ __forceinline__ void store_type(int t, char* p, int64_t i, float x) {
  if (t == PT_F32)
    store_f32<PT_F32>(p, i, x);
  else if (t == PT_F16)
    store_f32<PT_F16>(p, i, x);
  else
    store_f32<PT_BF16>(p, i, x);
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
// in the pool; false if it goes nowhere.
__device__ bool place(const RopeParams& P, int t, int* pos, int64_t* off) {
  int s = t;
  int64_t end = (int64_t)t + 1;
  if (P.token_start) {
    int lo = 0, hi = P.b.n_seqs;  // the last session that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (P.token_start[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    s = lo;
    end = P.token_start[s + 1];
    if (t >= end) return false;
  }
  const int len = P.b.lens[s];
  if (len == 0) return false;
  const int64_t p = token_pos(len, t, end);
  if (!length_ok(len, P.b.max_len) || p < 0) {
    report(P.err, length_ok(len, P.b.max_len) ? PERR_START : PERR_LENGTH);
    return false;
  }
  const int page = P.b.table[s * P.b.table_stride + (p >> P.kv.page_shift)];
  if (!page_ok(page, P.kv.n_pages)) {
    report(P.err, PERR_PAGE);
    return false;
  }
  *pos = (int)p;
  *off = page * P.kv.page_stride + (p & ((1 << P.kv.page_shift) - 1)) * P.kv.token_stride;
  return true;
}

// One workgroup per token, a thread per pair (or copied element).
template <int T, int CT, bool CACHED>
__global__ void __launch_bounds__(256) k_rope(RopeParams P) {
  const int t = blockIdx.x;
  int pos;
  int64_t off = 0;
  if constexpr (CACHED) {
    if (!place(P, t, &pos, &off)) return;
  } else {
    pos = P.positions[t];
  }
  const RopeTab& R = P.rope;
  const int half = R.rot_dim / 2, rows = P.n_q + 2 * P.n_kv, per = P.head_dim - half;
  for (int it = threadIdx.x; it < rows * per; it += 256) {
    const int row = it / per, i = it % per;
    const bool is_q = row < P.n_q, is_v = row >= P.n_q + P.n_kv;
    const int h = is_q ? row : (row - P.n_q) % P.n_kv;
    const HeadRows& S = is_q ? P.q : is_v ? P.v : P.k;
    const char* src = S.data + t * S.token_stride + h * S.head_stride;
    char* dst;
    float mul = 1.0f;
    if (is_q)
      dst = P.qo.data + t * P.qo.token_stride + h * P.qo.head_stride;
    else if constexpr (CACHED) {
      dst = (is_v ? P.kv.v : P.kv.k) + off + h * P.kv.head_stride;
      const float* sc = is_v ? P.kv.v_scale : P.kv.k_scale;
      if (CT == PT_E4M3 && sc) mul = sc[h];
    } else
      dst = P.ko.data + t * P.ko.token_stride + h * P.ko.head_stride;
    const int a = i < half ? (R.layout == 0 ? i : 2 * i) : i + half, b = i < half ? (R.layout == 0 ? i + half : 2 * i + 1) : a;
    float x = load_as_f32<T>(src, a), y = load_as_f32<T>(src, b);
    if (i < half && !is_v) {
      const float2 cs = cos_sin(R, i, pos);
      const float u = x * cs.x - y * cs.y, v = x * cs.y + y * cs.x;
      x = u;
      y = v;
    }
    if (CACHED && !is_q) {
      store_f32<CT>(dst, a, CT == PT_E4M3 ? x / mul : x);
      if (b != a) store_f32<CT>(dst, b, CT == PT_E4M3 ? y / mul : y);
    } else {
      store_f32<T>(dst, a, x);
      if (b != a) store_f32<T>(dst, b, y);
    }
  }
}

// --------------------------------------------------------------- attention

__device__ __forceinline__ float wg_reduce(float v, float* tmp, bool is_max) {
  for (int m = 32; m > 0; m >>= 1) {
    const float o = __shfl_xor(v, m);
    v = is_max ? fmaxf(v, o) : v + o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  return is_max ? fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3])) : (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
}

// One workgroup per (chunk, query head, session): scores of the chunk by a
// thread per position, then the weighted sum by a thread per element.
template <int CT>
__global__ void __launch_bounds__(256) k_paged_attn(PagedAttnParams P) {
  __shared__ float sc[ATTN_MAX_CHUNK], qs[256], tmp[4];
  __shared__ int tab[ATTN_TAB], bad;
  const int chunk = blockIdx.x % P.n_chunks, head = blockIdx.x / P.n_chunks % P.n_heads, s = blockIdx.x / P.n_chunks / P.n_heads;
  const int tid = threadIdx.x, hd = P.kv.head_dim, kvh = head / P.group;
  const int len = P.b.lens[s];
  const bool ok = length_ok(len, P.b.max_len);
  const Span span = attended(ok ? len : 0, P.window);
  const int n = max(chunks_of(span, P.chunk), 1);
  if (chunk >= n) return;
  const int c0 = span.lo + chunk * P.chunk, c1 = min(c0 + P.chunk, span.hi), p0 = c0 >> P.kv.page_shift;
  if (tid == 0) bad = 0;
  __syncthreads();
  if (c1 > c0)
    for (int i = tid; i <= ((c1 - 1) >> P.kv.page_shift) - p0; i += 256) {
      tab[i] = P.b.table[s * P.b.table_stride + p0 + i];
      if (!page_ok(tab[i], P.kv.n_pages)) bad = 1;
    }
  for (int d = tid; d < hd; d += 256)
    qs[d] = load_type(P.type, P.q.data + s * P.q.token_stride + head * P.q.head_stride, d);
  __syncthreads();
  char* out = P.out.data + s * P.out.token_stride + head * P.out.head_stride;
  const bool fail = bad || !ok;
  float m = -__builtin_inff(), l = 0.0f;
  if (!fail) {
    const float ks = CT == PT_E4M3 && P.kv.k_scale ? P.kv.k_scale[kvh] : 1.0f;
    auto slot = [&](int p) {
      return tab[(p >> P.kv.page_shift) - p0] * P.kv.page_stride + (p & ((1 << P.kv.page_shift) - 1)) * P.kv.token_stride +
             kvh * P.kv.head_stride;
    };
    for (int p = c0 + tid; p < c1; p += 256) {
      const char* row = P.kv.k + slot(p);
      float a = 0.0f;
      for (int d = 0; d < hd; ++d) a = __builtin_fmaf(qs[d], load_as_f32<CT>(row, d), a);
      sc[p - c0] = a * (P.scale_log2 * ks);
      m = fmaxf(m, sc[p - c0]);
    }
    m = wg_reduce(m, tmp, true);
    const float mu = m == -__builtin_inff() ? 0.0f : m;
    for (int p = c0 + tid; p < c1; p += 256) {
      sc[p - c0] = __builtin_amdgcn_exp2f(sc[p - c0] - mu);
      l += sc[p - c0];
    }
    l = wg_reduce(l, tmp, false);
    __syncthreads();
    for (int d = tid; d < hd; d += 256) {
      float a = 0.0f;
      for (int p = c0; p < c1; ++p) a = __builtin_fmaf(sc[p - c0], load_as_f32<CT>(P.kv.v + slot(p), d), a);
      const float vs = CT == PT_E4M3 && P.kv.v_scale ? P.kv.v_scale[kvh] : 1.0f;
      if (n == 1)
        store_type(P.type, out, d, l == 0.0f ? 0.0f : a / l * vs);
      else
        P.part_o[(((int64_t)s * P.n_heads + head) * P.n_chunks + chunk) * hd + d] = a * vs;
    }
  } else {
    if (tid == 0) report(P.err, ok ? PERR_PAGE : PERR_LENGTH);
    for (int d = tid; d < hd; d += 256) {
      if (n == 1)
        store_type(P.type, out, d, __builtin_nanf(""));
      else
        P.part_o[(((int64_t)s * P.n_heads + head) * P.n_chunks + chunk) * hd + d] = __builtin_nanf("");
    }
  }
  if (n > 1 && tid == 0) {
    float* ml = P.part_ml + (((int64_t)s * P.n_heads + head) * P.n_chunks + chunk) * 2;
    ml[0] = m;
    ml[1] = l;
  }
}

// Joins the chunks of a row: the sums brought to the common maximum.
__global__ void __launch_bounds__(256) k_paged_join(PagedAttnParams P) {
  const int head = blockIdx.x % P.n_heads, s = blockIdx.x / P.n_heads, hd = P.kv.head_dim;
  const int len = P.b.lens[s];
  const int n = chunks_of(attended(length_ok(len, P.b.max_len) ? len : 0, P.window), P.chunk);
  if (n <= 1) return;
  const int64_t row = ((int64_t)s * P.n_heads + head) * P.n_chunks;
  float m = -__builtin_inff(), l = 0.0f;
  for (int i = 0; i < n; ++i) m = fmaxf(m, P.part_ml[(row + i) * 2]);
  const float mu = m == -__builtin_inff() ? 0.0f : m;
  for (int i = 0; i < n; ++i) l += P.part_ml[(row + i) * 2 + 1] * __builtin_amdgcn_exp2f(P.part_ml[(row + i) * 2] - mu);
  for (int d = threadIdx.x; d < hd; d += 256) {
    float a = 0.0f;
    for (int i = 0; i < n; ++i)
      a += P.part_o[(row + i) * hd + d] * __builtin_amdgcn_exp2f(P.part_ml[(row + i) * 2] - mu);
    store_type(P.type, P.out.data + s * P.out.token_stride + head * P.out.head_stride, d, l == 0.0f ? a * 0.0f : a / l);
  }
}

}  // namespace

void launch_paged_attn(const PagedAttnParams& P, int cache_type, hipStream_t st) {
  const dim3 grid(P.n_chunks * P.n_heads * P.b.n_seqs), block(256);
  switch (cache_type) {
    case PT_F32: hipLaunchKernelGGL(k_paged_attn<PT_F32>, grid, block, 0, st, P); break;
    case PT_F16: hipLaunchKernelGGL(k_paged_attn<PT_F16>, grid, block, 0, st, P); break;
    case PT_BF16: hipLaunchKernelGGL(k_paged_attn<PT_BF16>, grid, block, 0, st, P); break;
    default: hipLaunchKernelGGL(k_paged_attn<PT_E4M3>, grid, block, 0, st, P); break;
  }
  if (P.n_chunks > 1) hipLaunchKernelGGL(k_paged_join, dim3(P.n_heads * P.b.n_seqs), block, 0, st, P);
}

namespace {
template <int T>
void launch_rope_t(const RopeParams& P, int cache_type, bool cached, hipStream_t st) {
  const dim3 grid(P.n_tokens), block(256);
  if (!cached)
    hipLaunchKernelGGL((k_rope<T, T, false>), grid, block, 0, st, P);
  else if (cache_type == PT_F32)
    hipLaunchKernelGGL((k_rope<T, PT_F32, true>), grid, block, 0, st, P);
  else if (cache_type == PT_F16)
    hipLaunchKernelGGL((k_rope<T, PT_F16, true>), grid, block, 0, st, P);
  else if (cache_type == PT_BF16)
    hipLaunchKernelGGL((k_rope<T, PT_BF16, true>), grid, block, 0, st, P);
  else
    hipLaunchKernelGGL((k_rope<T, PT_E4M3, true>), grid, block, 0, st, P);
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
