// Rotary positions and the append to the paged key-value cache, in one launch:
// q -> rotated q, k -> rotated k in its cache row, v -> its cache row.
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

}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_rope_append(const hxm_heads* q, const hxm_heads* q_out, int64_t q_heads,
                                      const hxm_heads* k, const hxm_heads* v,
                                      const int32_t* positions, const float* cos_sin,
                                      int64_t ld_cos_sin, int64_t max_pos, int64_t rot_dim,
                                      int32_t interleaved, const int32_t* slots,
                                      const hxm_kv_cache* cache, int64_t tokens, int32_t dtype,
                                      void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: rope_append takes f16 or bf16 (got %d)",
                dtype);
  hxm_status st = check_kv_cache("rope_append", cache, true);
  if (st != HXM_OK) return st;
  const int64_t dim = cache->dim, hkv = cache->heads;
  if (tokens < 0 || q_heads < 0)
    return fail(HXM_INVALID_ARG, "invalid-argument: rope_append tokens=%lld q_heads=%lld",
                (long long)tokens, (long long)q_heads);
  if (tokens > INT32_MAX / 2 || q_heads > 65535)
    return fail(HXM_UNSUPPORTED_SHAPE, "tile-alignment: rope_append tokens=%lld q_heads=%lld",
                (long long)tokens, (long long)q_heads);
  if (rot_dim < 0 || rot_dim > dim || rot_dim % 2 != 0)
    return fail(HXM_INVALID_ARG, "invalid-argument: rope_append rot_dim=%lld of %lld dims",
                (long long)rot_dim, (long long)dim);
  if ((st = check_heads("rope_append", "k", k, tokens, hkv, dim, false)) != HXM_OK) return st;
  if ((st = check_heads("rope_append", "v", v, tokens, hkv, dim, false)) != HXM_OK) return st;
  if (q_heads > 0) {
    if ((st = check_heads("rope_append", "q", q, tokens, q_heads, dim, false)) != HXM_OK) return st;
    if ((st = check_heads("rope_append", "q_out", q_out, tokens, q_heads, dim, true)) != HXM_OK)
      return st;
  }
  if (rot_dim > 0 && (max_pos < 1 || !stride_ok(ld_cos_sin) || ld_cos_sin < rot_dim))
    return fail(HXM_INVALID_ARG, "invalid-argument: rope_append max_pos=%lld ld_cos_sin=%lld",
                (long long)max_pos, (long long)ld_cos_sin);
  if (tokens > 0 && (!slots || (rot_dim > 0 && (!positions || !cos_sin))))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: rope_append null slots, positions or cos_sin");
  if (q_heads > 0 && tokens > 0) {
    if ((!heads_same(q_out, q, tokens, q_heads) &&
         !heads_apart(q_out, q_heads, q, q_heads, tokens, dim)) ||
        !heads_apart(q_out, q_heads, k, hkv, tokens, dim) ||
        !heads_apart(q_out, q_heads, v, hkv, tokens, dim))
      return fail(HXM_INVALID_ARG,
                  "invalid-argument: rope_append q_out overlaps q (without being it), k or v");
  }
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (tokens == 0) return ok();
  RopeArgs a{};
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
