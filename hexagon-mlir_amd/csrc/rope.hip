// Rotary positions and the append to the paged key-value cache, in one launch:
// q -> rotated q, k -> rotated k in its cache row, v -> its cache row; and the same with a
// norm of each query and key head before the rotation.
//
// Bound by memory: every element of q, k and v is read once and written once (8192 tokens,
// 32 + 8 heads of 128, bf16: 206 MB in 40 us, 5.1 TB/s; a copy of 1 GiB runs at 5.3); a
// pair takes two products and two fmas.  A group of threads serves one token. A thread
// keeps one chunk of the rotated dims (eight pairs, or four neighbouring ones) and walks
// the heads with it, so it loads its cosines and sines once per token and not once per
// head; the q heads, the k heads and then the v chunks are one sequence of 16-byte loads
// and stores, at any element address.
#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

struct HeadsArg {
  const void* p;
  int64_t ts, hs;
};

struct RopeArgs {
  HeadsArg q, qo, k, v;
  void *kc, *vc;
  int64_t kps, khs, kts, vps, vhs, vts;
  const int32_t* positions;
  const float* cos_sin;
  const int32_t* slots;
  int64_t ld_cs, max_pos;
  uint32_t nslots, page_size;
  int tokens, hq, hkv, dim, rot;
  int tt;          // threads of a token
  int rchunks;     // chunks of a head's rotated dims
  int chunks;      // and of its other dims
};

constexpr int kChunk = 8;  // 16-bit elements of a vector

template <typename T>
__device__ __forceinline__ RawVec<T> load_n(const T* p, int n) {
  return n == kChunk ? load_any(p) : load_tail(p, 0, n, T(0));
}
// Rows of the cache go past the caches, which then keep the inputs of large calls (8192
// tokens, 32 + 8 heads of 128: 41.2 -> 40.4 us; 16 + 16 heads of 64: 26.2 -> 20.9; 1024
// tokens 7.2 -> 6.9); q stays in them for the attention that follows (nontemporal too,
// 42.2, 25.6 and 5.9).
template <bool CACHED, typename T>
__device__ __forceinline__ void store_n(T* p, RawVec<T> v, int n) {
  if (n == kChunk && !CACHED) store_any(p, v);
  else if (n == kChunk) *reinterpret_cast<AnyVec<T>*>(p) = v;
  else store_tail(p, 0, n, v);
}
// n of M floats (M a multiple of 4, n at least 1), the rest unspecified.
template <int M>
__device__ __forceinline__ void load_floats(const float* p, int n, float (&f)[M]) {
  if (n == M) {
#pragma unroll
    for (int i = 0; i < M; i += 4) {
      const RawVec<float> v = load_any(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < M; ++e) f[e] = p[min(e, n - 1)];
  }
}

template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeArgs a) {
  const int t = blockIdx.x * (256 / a.tt) + static_cast<int>(threadIdx.x) / a.tt;
  const int i = static_cast<int>(threadIdx.x) % a.tt;
  if (t >= a.tokens) return;
  const uint32_t slot = static_cast<uint32_t>(a.slots[t]);  // negative ones pass nslots too
  const bool stored = slot < a.nslots;
  const int64_t page = stored ? slot / a.page_size : 0;
  const int64_t off = stored ? slot % a.page_size : 0;
  T* kc = static_cast<T*>(a.kc) + page * a.kps + off * a.kts;
  T* vc = static_cast<T*>(a.vc) + page * a.vps + off * a.vts;

  const int per = a.tt / a.chunks;  // heads at a time
  const int c = i % a.chunks;
  int h = i / a.chunks;
  if (h < per) {
    const int half = a.rot / 2;
    const bool turned = c < a.rchunks;
    // The chunk's elements lo[0, n) and, of the half-split pairs, lo + half.
    const int lo = turned ? c * kChunk : a.rot + (c - a.rchunks) * kChunk;
    const int n = min(kChunk, (turned ? (PAIRS ? a.rot : half) : a.dim) - lo);
    constexpr int M = PAIRS ? kChunk / 2 : kChunk;  // pairs of a chunk
    float cs[M], sn[M];
    if (turned) {
      const int32_t p = a.positions[t];
      const bool good = p >= 0 && p < a.max_pos;
      const float* row = a.cos_sin + (good ? p : 0) * a.ld_cs + (PAIRS ? lo / 2 : lo);
      load_floats(row, PAIRS ? n / 2 : n, cs);
      load_floats(row + half, PAIRS ? n / 2 : n, sn);
      if (!good) {
#pragma unroll
        for (int e = 0; e < M; ++e) cs[e] = sn[e] = __builtin_nanf("");
      }
    }
    for (; h < a.hq + a.hkv; h += per) {
      const bool isq = h < a.hq;
      if (!isq && !stored) break;
      const T* src = isq ? static_cast<const T*>(a.q.p) + t * a.q.ts + h * a.q.hs
                         : static_cast<const T*>(a.k.p) + t * a.k.ts + (h - a.hq) * a.k.hs;
      T* dst = isq ? static_cast<T*>(const_cast<void*>(a.qo.p)) + t * a.qo.ts + h * a.qo.hs
                   : kc + (h - a.hq) * a.khs;
      RawVec<T> x = load_n(src + lo, n);
      if (turned) {
        if constexpr (PAIRS) {
#pragma unroll
          for (int e = 0; e < M; ++e) {
            const float u = tof(x[2 * e]), w = tof(x[2 * e + 1]);
            x[2 * e] = fromf<T>(fmaf(u, cs[e], -(w * sn[e])));
            x[2 * e + 1] = fromf<T>(fmaf(w, cs[e], u * sn[e]));
          }
        } else {
          RawVec<T> y = load_n(src + lo + half, n);
#pragma unroll
          for (int e = 0; e < kChunk; ++e) {
            const float u = tof(x[e]), w = tof(y[e]);
            x[e] = fromf<T>(fmaf(u, cs[e], -(w * sn[e])));
            y[e] = fromf<T>(fmaf(w, cs[e], u * sn[e]));
          }
          if (isq) store_n<true>(dst + lo + half, y, n);
          else store_n<false>(dst + lo + half, y, n);
        }
      }
      if (isq) store_n<true>(dst + lo, x, n);
      else store_n<false>(dst + lo, x, n);
    }
  }
  if (!stored) return;
  const int vch = a.dim / kChunk;
  for (int j = i; j < a.hkv * vch; j += a.tt) {
    const int hv = j / vch, d = (j - hv * vch) * kChunk;
    const T* src = static_cast<const T*>(a.v.p) + t * a.v.ts + hv * a.v.hs + d;
    store_n<false>(vc + hv * a.vhs + d, load_any(src), kChunk);
  }
}

typedef float v8f32 __attribute__((ext_vector_type(8)));

// The norms of the heads in front of it: gamma and beta rows of a head, `hs` apart.
struct HeadNorm {
  const void *gamma, *beta;
  int64_t hs;
  float eps;
  int kind;
};
struct NormRopeArgs : RopeArgs {
  HeadNorm nq, nk;
  int lanes;  // of a head: a power of two, its chunks and up
};

// The sum over the aligned group of `lanes` lanes (1 to 64) that this one is in.
__device__ __forceinline__ float group_sum(float v, int lanes) {
  if (lanes > 1) v += dpp<kDppQuadXor1>(v);
  if (lanes > 2) v += dpp<kDppQuadXor2>(v);
  if (lanes > 4) v += dpp<kDppRowHalfMirror>(v);
  if (lanes > 8) v += dpp<kDppRowMirror>(v);
  if (lanes > 16) v += __shfl_xor(v, 16, 64);
  if (lanes > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

// A head's norm, its rotation and its store in one pass over it: the lanes of a head, a
// power of two, keep its chunks in registers as fp32 from the load to the one rounding
// and share the statistics by DPP sums (LayerNorm: the mean, then the squares around it).
// Bound by memory as above: 8192 tokens, 32 + 8 heads of 128, bf16, 206 MB in 39.9 us,
// 5.2 TB/s, what the rotation without norms takes.  (The next head's loads issued before this
// one's sums: 68 us with 128 threads a token, for 45.7.)
template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void norm_rope_append_kernel(NormRopeArgs a) {
  const int t = blockIdx.x * (256 / a.tt) + static_cast<int>(threadIdx.x) / a.tt;
  const int i = static_cast<int>(threadIdx.x) % a.tt;
  if (t >= a.tokens) return;
  const uint32_t slot = static_cast<uint32_t>(a.slots[t]);  // negative ones pass nslots too
  const bool stored = slot < a.nslots;
  const int64_t page = stored ? slot / a.page_size : 0;
  const int64_t off = stored ? slot % a.page_size : 0;
  T* kc = static_cast<T*>(a.kc) + page * a.kps + off * a.kts;
  T* vc = static_cast<T*>(a.vc) + page * a.vps + off * a.vts;

  const int per = a.tt / a.lanes;  // heads at a time
  const int c = i % a.lanes;
  const int half = a.rot / 2;
  const bool turned = c < a.rchunks;
  const bool two = !PAIRS && turned;  // of the half-split pairs, lo + half too
  const int lo = turned ? c * kChunk : a.rot + (c - a.rchunks) * kChunk;
  const int n = c < a.chunks ? min(kChunk, (turned ? (PAIRS ? a.rot : half) : a.dim) - lo) : 0;
  constexpr int M = PAIRS ? kChunk / 2 : kChunk;  // pairs of a chunk
  float cs[M], sn[M];
  if (turned) {
    const int32_t p = a.positions[t];
    const bool good = p >= 0 && p < a.max_pos;
    const float* row = a.cos_sin + (good ? p : 0) * a.ld_cs + (PAIRS ? lo / 2 : lo);
    load_floats(row, PAIRS ? n / 2 : n, cs);
    load_floats(row + half, PAIRS ? n / 2 : n, sn);
    if (!good) {
#pragma unroll
      for (int e = 0; e < M; ++e) cs[e] = sn[e] = __builtin_nanf("");
    }
  }
  const int heads = stored ? a.hq + a.hkv : a.hq;
  const float count = 1.0f / static_cast<float>(a.dim);
  // Every lane of a wave takes every turn: the sums need them all.
  for (int h0 = 0; h0 < heads; h0 += per) {
    const int h = h0 + i / a.lanes;
    const bool on = h < heads && n > 0;
    const bool isq = h < a.hq;
    const int hh = isq ? h : h - a.hq;
    const HeadNorm nm = isq ? a.nq : a.nk;
    const T* src = isq ? static_cast<const T*>(a.q.p) + t * a.q.ts + hh * a.q.hs
                       : static_cast<const T*>(a.k.p) + t * a.k.ts + hh * a.k.hs;
    T* dst = isq ? static_cast<T*>(const_cast<void*>(a.qo.p)) + t * a.qo.ts + hh * a.qo.hs
                 : kc + hh * a.khs;
    RawVec<T> rx = RawVec<T>(T(0)), ry = rx, gx = rx, gy = rx, bx = rx, by = rx;
    if (on) {
      rx = load_n(src + lo, n);
      if (two) ry = load_n(src + lo + half, n);
      if (nm.gamma) {
        const T* g = static_cast<const T*>(nm.gamma) + hh * nm.hs + lo;
        gx = load_n(g, n);
        if (two) gy = load_n(g + half, n);
      }
      if (nm.beta) {
        const T* g = static_cast<const T*>(nm.beta) + hh * nm.hs + lo;
        bx = load_n(g, n);
        if (two) by = load_n(g + half, n);
      }
    }
    // (load_n leaves zeros past n.)
    v8f32 x = __builtin_convertvector(rx, v8f32), y = __builtin_convertvector(ry, v8f32);
    if (nm.kind == HXM_NORM_LAYER) {
      float mean = 0.0f;
#pragma unroll
      for (int e = 0; e < kChunk; ++e) mean += x[e] + y[e];
      mean = group_sum(mean, a.lanes) * count;
#pragma unroll
      for (int e = 0; e < kChunk; ++e) {
        x[e] = e < n ? x[e] - mean : 0.0f;
        y[e] = two && e < n ? y[e] - mean : 0.0f;
      }
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < kChunk; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
    ss = group_sum(ss, a.lanes) * count;
    if (!on) continue;
    if (nm.kind != HXM_NORM_NONE) {
      const float r = 1.0f / sqrtf(ss + nm.eps);
      x *= r, y *= r;
      if (nm.gamma) {
        x *= __builtin_convertvector(gx, v8f32);
        if (!PAIRS) y *= __builtin_convertvector(gy, v8f32);
      }
      if (nm.beta) {
        x += __builtin_convertvector(bx, v8f32);
        if (!PAIRS) y += __builtin_convertvector(by, v8f32);
      }
    }
    if (turned) {
      v8f32 u;
      if constexpr (PAIRS) {
#pragma unroll
        for (int e = 0; e < M; ++e) {
          u[2 * e] = fmaf(x[2 * e], cs[e], -(x[2 * e + 1] * sn[e]));
          u[2 * e + 1] = fmaf(x[2 * e + 1], cs[e], x[2 * e] * sn[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < M; ++e) {
          u[e] = fmaf(x[e], cs[e], -(y[e] * sn[e]));
          y[e] = fmaf(y[e], cs[e], x[e] * sn[e]);
        }
        const RawVec<T> oy = __builtin_convertvector(y, RawVec<T>);
        if (isq) store_n<true>(dst + lo + half, oy, n);
        else store_n<false>(dst + lo + half, oy, n);
      }
      x = u;
    }
    const RawVec<T> ox = __builtin_convertvector(x, RawVec<T>);
    if (isq) store_n<true>(dst + lo, ox, n);
    else store_n<false>(dst + lo, ox, n);
  }
  if (!stored) return;
  const int vch = a.dim / kChunk;
  for (int j = i; j < a.hkv * vch; j += a.tt) {
    const int hv = j / vch, d = (j - hv * vch) * kChunk;
    const T* src = static_cast<const T*>(a.v.p) + t * a.v.ts + hv * a.v.hs + d;
    store_n<false>(vc + hv * a.vhs + d, load_any(src), kChunk);
  }
}

}  // namespace

hxm_status check_heads(const char* op, const char* what, const hxm_heads* h, int64_t tokens,
                       int64_t heads, int64_t dim, bool written) {
  if (!h || (tokens > 0 && heads > 0 && !h->data))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s null %s", op, what);
  if (!stride_ok(h->token_stride) || !stride_ok(h->head_stride))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s %s strides %lld, %lld", op, what,
                (long long)h->token_stride, (long long)h->head_stride);
  const int64_t n[2] = {tokens, heads}, s[2] = {h->token_stride, h->head_stride};
  if (written && !strides_disjoint(n, s, 2, dim))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s %s rows share elements", op, what);
  return HXM_OK;
}

bool heads_same(const hxm_heads* out, const hxm_heads* in, int64_t tokens, int64_t heads) {
  return out->data == in->data && (out->token_stride == in->token_stride || tokens == 1) &&
         (out->head_stride == in->head_stride || heads == 1);
}

bool heads_apart(const hxm_heads* out, int64_t out_heads, const hxm_heads* in, int64_t in_heads,
                 int64_t tokens, int64_t dim) {
  const uintptr_t o = reinterpret_cast<uintptr_t>(out->data),
                  i = reinterpret_cast<uintptr_t>(in->data);
  if (matrices_disjoint(o, out->token_stride, i, in->token_stride, tokens,
                        (out_heads - 1) * out->head_stride + dim,
                        (in_heads - 1) * in->head_stride + dim, 2))
    return true;
  // Heads of one between heads of the other.  A stride along one token or one head is none.
  if ((tokens > 1 && out->token_stride != in->token_stride) ||
      (out_heads > 1 && in_heads > 1 && out->head_stride != in->head_stride))
    return false;
  const int64_t n[2] = {tokens, out_heads > in_heads ? out_heads : in_heads};
  const int64_t s[2] = {out->token_stride, out_heads > 1 ? out->head_stride : in->head_stride};
  return twins_disjoint(o, i, n, s, 2, dim, 2);
}

// Keys and values apart: whole buffers, parts of each page, or rows side by side at equal
// strides.
static bool keys_values_apart(const hxm_kv_cache* c) {
  const uintptr_t k = reinterpret_cast<uintptr_t>(c->k), v = reinterpret_cast<uintptr_t>(c->v);
  auto page_span = [&](int64_t head_stride, int64_t token_stride) {
    const __int128 span = static_cast<__int128>(c->heads - 1) * head_stride +
                          static_cast<__int128>(c->page_size - 1) * token_stride + c->dim;
    return span < INT64_MAX ? static_cast<int64_t>(span) : INT64_MAX;
  };
  if (matrices_disjoint(k, c->k_page_stride, v, c->v_page_stride, c->pages,
                        page_span(c->k_head_stride, c->k_token_stride),
                        page_span(c->v_head_stride, c->v_token_stride), 2))
    return true;
  const int64_t n[3] = {c->pages, c->heads, c->page_size};
  const int64_t ks[3] = {c->k_page_stride, c->k_head_stride, c->k_token_stride},
                vs[3] = {c->v_page_stride, c->v_head_stride, c->v_token_stride};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && ks[i] != vs[i]) return false;
  return twins_disjoint(k, v, n, ks, 3, c->dim, 2);
}

bool layers_apart(const hxm_kv_cache* c, int64_t layers, int64_t kls, int64_t vls) {
  const int64_t n[4] = {layers, c->pages, c->heads, c->page_size};
  const int64_t ks[4] = {kls, c->k_page_stride, c->k_head_stride, c->k_token_stride},
                vs[4] = {vls, c->v_page_stride, c->v_head_stride, c->v_token_stride};
  if (!strides_disjoint(n, ks, 4, c->dim) || !strides_disjoint(n, vs, 4, c->dim)) return false;
  auto layer_span = [&](const int64_t* s) {
    __int128 span = c->dim;
    for (int i = 1; i < 4; ++i) span += static_cast<__int128>(n[i] - 1) * s[i];
    return span < INT64_MAX ? static_cast<int64_t>(span) : INT64_MAX;
  };
  const uintptr_t k = reinterpret_cast<uintptr_t>(c->k), v = reinterpret_cast<uintptr_t>(c->v);
  if (matrices_disjoint(k, kls, v, vls, layers, layer_span(ks), layer_span(vs), 2)) return true;
  for (int i = 0; i < 4; ++i)
    if (n[i] > 1 && ks[i] != vs[i]) return false;
  return layer_twins_disjoint(k, v, n, ks, c->dim, 2);
}

hxm_status check_kv_cache(const char* op, const hxm_kv_cache* c, bool written) {
  if (!c || !c->k || !c->v)
    return fail(HXM_INVALID_ARG, "invalid-argument: %s null cache", op);
  if (c->pages < 1 || c->page_size < 1 || c->heads < 1 || c->dim < 1)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: %s cache of %lld pages, %lld tokens, %lld heads, %lld dims", op,
                (long long)c->pages, (long long)c->page_size, (long long)c->heads,
                (long long)c->dim);
  if (c->dim % 8 != 0 || c->dim > 256)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: %s head dim %lld is not a multiple of 8 up to 256", op,
                (long long)c->dim);
  if (c->pages > INT32_MAX / c->page_size || c->heads > 65535)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: %s cache of %lld pages of %lld tokens, %lld heads", op,
                (long long)c->pages, (long long)c->page_size, (long long)c->heads);
  const int64_t n[3] = {c->pages, c->heads, c->page_size};
  const int64_t s[2][3] = {{c->k_page_stride, c->k_head_stride, c->k_token_stride},
                           {c->v_page_stride, c->v_head_stride, c->v_token_stride}};
  for (const auto& st : s) {
    if (!stride_ok(st[0]) || !stride_ok(st[1]) || !stride_ok(st[2]))
      return fail(HXM_INVALID_ARG, "invalid-argument: %s cache strides %lld, %lld, %lld", op,
                  (long long)st[0], (long long)st[1], (long long)st[2]);
    if (written && !strides_disjoint(n, st, 3, c->dim))
      return fail(HXM_INVALID_ARG, "invalid-argument: %s cache rows share elements", op);
  }
  if (written && !keys_values_apart(c))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s keys and values share elements", op);
  return HXM_OK;
}

// The arguments of an append checked, and as the kernels take them.
static hxm_status rope_args(const char* op, const hxm_heads* q, const hxm_heads* q_out,
                            int64_t q_heads, const hxm_heads* k, const hxm_heads* v,
                            const int32_t* positions, const float* cos_sin, int64_t ld_cos_sin,
                            int64_t max_pos,
                            int64_t rot_dim, int32_t interleaved, const int32_t* slots,
                            const hxm_kv_cache* cache, int64_t tokens, int32_t dtype,
                            RopeArgs& a) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: %s takes f16 or bf16 (got %d)",
                op, dtype);
  hxm_status st = check_kv_cache(op, cache, true);
  if (st != HXM_OK) return st;
  const int64_t dim = cache->dim, hkv = cache->heads;
  if (tokens < 0 || q_heads < 0)
    return fail(HXM_INVALID_ARG, "invalid-argument: %s tokens=%lld q_heads=%lld", op,
                (long long)tokens, (long long)q_heads);
  if (tokens > INT32_MAX / 2 || q_heads > 65535)
    return fail(HXM_UNSUPPORTED_SHAPE, "tile-alignment: %s tokens=%lld q_heads=%lld", op,
                (long long)tokens, (long long)q_heads);
  if (rot_dim < 0 || rot_dim > dim || rot_dim % 2 != 0)
    return fail(HXM_INVALID_ARG, "invalid-argument: %s rot_dim=%lld of %lld dims", op,
                (long long)rot_dim, (long long)dim);
  if ((st = check_heads(op, "k", k, tokens, hkv, dim, false)) != HXM_OK) return st;
  if ((st = check_heads(op, "v", v, tokens, hkv, dim, false)) != HXM_OK) return st;
  if (q_heads > 0) {
    if ((st = check_heads(op, "q", q, tokens, q_heads, dim, false)) != HXM_OK) return st;
    if ((st = check_heads(op, "q_out", q_out, tokens, q_heads, dim, true)) != HXM_OK)
      return st;
  }
  if (rot_dim > 0 && (max_pos < 1 || !stride_ok(ld_cos_sin) || ld_cos_sin < rot_dim))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s max_pos=%lld ld_cos_sin=%lld", op,
                (long long)max_pos, (long long)ld_cos_sin);
  if (tokens > 0 && (!slots || (rot_dim > 0 && (!positions || !cos_sin))))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: %s null slots, positions or cos_sin", op);
  if (q_heads > 0 && tokens > 0) {
    if ((!heads_same(q_out, q, tokens, q_heads) &&
         !heads_apart(q_out, q_heads, q, q_heads, tokens, dim)) ||
        !heads_apart(q_out, q_heads, k, hkv, tokens, dim) ||
        !heads_apart(q_out, q_heads, v, hkv, tokens, dim))
      return fail(HXM_INVALID_ARG,
                  "invalid-argument: %s q_out overlaps q (without being it), k or v", op);
  }
  if (q_heads > 0) {
    a.q = {q->data, q->token_stride, q->head_stride};
    a.qo = {q_out->data, q_out->token_stride, q_out->head_stride};
  }
  a.k = {k->data, k->token_stride, k->head_stride};
  a.v = {v->data, v->token_stride, v->head_stride};
  a.kc = cache->k, a.vc = cache->v;
  a.kps = cache->k_page_stride, a.khs = cache->k_head_stride, a.kts = cache->k_token_stride;
  a.vps = cache->v_page_stride, a.vhs = cache->v_head_stride, a.vts = cache->v_token_stride;
  a.positions = positions, a.cos_sin = cos_sin, a.slots = slots;
  a.ld_cs = ld_cos_sin, a.max_pos = max_pos;
  a.nslots = static_cast<uint32_t>(cache->pages * cache->page_size);
  a.page_size = static_cast<uint32_t>(cache->page_size);
  a.tokens = static_cast<int>(tokens), a.hq = static_cast<int>(q_heads);
  a.hkv = static_cast<int>(hkv), a.dim = static_cast<int>(dim), a.rot = static_cast<int>(rot_dim);
  a.rchunks = static_cast<int>(ceil_div(interleaved ? rot_dim : rot_dim / 2, kChunk));
  a.chunks = a.rchunks + static_cast<int>(ceil_div(dim - rot_dim, kChunk));
  return HXM_OK;
}

}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_rope_append(const hxm_heads* q, const hxm_heads* q_out, int64_t q_heads,
                                      const hxm_heads* k, const hxm_heads* v,
                                      const int32_t* positions, const float* cos_sin,
                                      int64_t ld_cos_sin, int64_t max_pos, int64_t rot_dim,
                                      int32_t interleaved, const int32_t* slots,
                                      const hxm_kv_cache* cache, int64_t tokens, int32_t dtype,
                                      void* stream) {
  RopeArgs a{};
  hxm_status st = rope_args("rope_append", q, q_out, q_heads, k, v, positions, cos_sin, ld_cos_sin,
                            max_pos, rot_dim, interleaved, slots, cache, tokens, dtype, a);
  if (st != HXM_OK || (st = require_device(nullptr)) != HXM_OK) return st;
  if (tokens == 0) return ok();
  // Threads of a token: one for each chunk it has, a power of two from 64 to
  // a workgroup's 256, or 128 once the tokens fill the chip that way (a head has at
  // most 33 chunks).  32 + 8 heads of 128: 8192 tokens 42.7 us with 256, 41.2 with 128, 46
  // with 64; 64 tokens 5.2, 5.5, 6.8.
  a.tt = 64;
  const int most = tokens >= 2048 ? 128 : 256;
  while (a.tt < most && a.tt < a.chunks * (a.hq + a.hkv)) a.tt *= 2;
  const int64_t groups = ceil_div(tokens, 256 / a.tt);
  if ((st = check_grid("rope append", groups, 256)) != HXM_OK) return st;
  const unsigned g = static_cast<unsigned>(groups);
  hipStream_t s = as_stream(stream);
  if (dtype == HXM_F16)
    interleaved ? rope_append_kernel<_Float16, true><<<g, 256, 0, s>>>(a)
                : rope_append_kernel<_Float16, false><<<g, 256, 0, s>>>(a);
  else
    interleaved ? rope_append_kernel<__bf16, true><<<g, 256, 0, s>>>(a)
                : rope_append_kernel<__bf16, false><<<g, 256, 0, s>>>(a);
  return check_launch("rope append");
}

extern "C" hxm_status hxm_norm_rope_append(const hxm_heads* q, const hxm_heads* q_out,
                                           int64_t q_heads, const hxm_heads* k, const hxm_heads* v,
                                           const hxm_head_norm* q_norm, const hxm_head_norm* k_norm,
                                           const int32_t* positions, const float* cos_sin,
                                           int64_t ld_cos_sin, int64_t max_pos, int64_t rot_dim,
                                           int32_t interleaved, const int32_t* slots,
                                           const hxm_kv_cache* cache, int64_t tokens, int32_t dtype,
                                           void* stream) {
  NormRopeArgs a{};
  hxm_status st = rope_args("norm_rope_append", q, q_out, q_heads, k, v, positions, cos_sin,
                            ld_cos_sin, max_pos, rot_dim, interleaved, slots, cache, tokens, dtype,
                            a);
  if (st != HXM_OK) return st;
  for (const bool isq : {true, false}) {
    if (isq && q_heads == 0) continue;
    const hxm_head_norm* m = isq ? q_norm : k_norm;
    if (!m || m->kind < HXM_NORM_NONE || m->kind > HXM_NORM_LAYER || !(m->eps >= 0.0f) ||
        !stride_ok(m->head_stride) || (m->head_stride > 0 && m->head_stride < cache->dim) ||
        (m->kind == HXM_NORM_NONE && (m->gamma || m->beta)))
      return fail(HXM_INVALID_ARG, "invalid-argument: norm_rope_append norm of %s",
                  isq ? "q" : "k");
    (isq ? a.nq : a.nk) = HeadNorm{m->gamma, m->beta, m->head_stride, m->eps, m->kind};
  }
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (tokens == 0) return ok();
  a.lanes = 1;
  while (a.lanes < a.chunks) a.lanes *= 2;
  // Threads of a token: as rope_append, and one wave where the tokens fill the chip that way
  // (32 + 8 heads of 128: 8192 tokens 39.9 us with 64, 45.7 with 128, 60 with 256; 4096 19.4,
  // 20.4, 24.9; 2048 12.9, 11.7, 14.6; 1024 12.1, 9.5, 9.0; 64 8.7, 6.4, 5.3; 64 + 8 of 128: 8192
  // 61, 65, 79, 2048 19.4, 17.1, 19.1, 64 12.9, 8.7, 6.5; 16 + 16 of 256: 76, 77, 81, 20.6, 19.3,
  // 19.4, 13.0, 8.2, 5.8; 8 + 8 of 64: 13.0 each, 5.9, 4.4).
  a.tt = 64;
  const int most = tokens >= 4096 ? 64 : tokens >= 2048 ? 128 : 256;
  while (a.tt < most && a.tt < a.lanes * (a.hq + a.hkv)) a.tt *= 2;
  const int64_t groups = ceil_div(tokens, 256 / a.tt);
  if ((st = check_grid("norm rope append", groups, 256)) != HXM_OK) return st;
  const unsigned g = static_cast<unsigned>(groups);
  hipStream_t s = as_stream(stream);
  if (dtype == HXM_F16)
    interleaved ? norm_rope_append_kernel<_Float16, true><<<g, 256, 0, s>>>(a)
                : norm_rope_append_kernel<_Float16, false><<<g, 256, 0, s>>>(a);
  else
    interleaved ? norm_rope_append_kernel<__bf16, true><<<g, 256, 0, s>>>(a)
                : norm_rope_append_kernel<__bf16, false><<<g, 256, 0, s>>>(a);
  return check_launch("norm rope append");
}
