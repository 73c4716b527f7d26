// Attention of one new token per sequence over the paged key-value cache.
//
// Bound by memory: the keys and values of a sequence are read once per key
// head, 4 * dim bytes a token, against 4 * dim * group operations.  The group of
// query heads that shares a key head is the 16-wide side of the MFMAs (padded
// with zeros), so one read serves the whole group.
//
// A wave takes 32 tokens at a time.  With K as the left operand and Q^T as the
// right one, S^T = K Q^T leaves lane (g, c) = (lane / 16, lane % 16) the scores of
// head c; the rows of the two 16-token products are assigned so that they are
// those of tokens 8g .. 8g+7.  That is how O^T = V^T P^T wants P^T as its right
// operand: the probabilities go from the first product to the second in the
// registers they are in, and running maximum, sum and output of a head live
// in the lanes of one column.  V's left operand has tokens along a lane's
// registers: a lane loads the 8 tokens x dim/16 dims whose transpose it needs
// (whole rows per 16 lanes) and transposes them in registers with byte permutes.
// No LDS until the waves of a workgroup are joined.
//
// The running maximum moves only when a score passes it by more than 2^8 in
// the exponent's base 2: exp2(s - m) stays far below fp32's limit, and the
// output is rescaled a few times per sequence and not per tile.  f16
// probabilities are scaled by 2^7 on the way into the product, so that with
// those 8 binary orders of headroom they stay below 65504 and the smallest
// normal one is 2^-21 of the largest.
#include <type_traits>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kTile = 32;       // tokens of a wave's step
constexpr int kHeads = 16;      // query heads of a workgroup
constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;  // of the running maximum, in powers of two

struct AttnArgs {
  const void* q;
  void* out;
  const void* kc;
  const void* vc;
  const int32_t* table;
  const int32_t* lens;
  float* lse;
  int64_t q_ts, q_hs, o_ts, o_hs;
  int64_t kps, khs, kts, vps, vhs, vts;
  int64_t ld_table, capacity;  // tokens a table row holds
  uint32_t pages, page_size;
  int hkv, group, tiles, dim, window;
  float scale;
};

template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef v8f16 V;
  static constexpr float kShift = 7.0f;
  static __device__ __forceinline__ v4f32 mfma(V a, V b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<__bf16> {
  typedef v8bf16 V;
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ v4f32 mfma(V a, V b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// 16 or 8 bytes at any element address.
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t any2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Keys and values of a 32-token tile as a lane holds them.
template <int DT>
struct Tile {
  static constexpr int KK = DT / 32;  // K steps of the first product
  static constexpr int VW = DT / 32;  // dwords of a token's DT / 16 value dims
  v4u32_t k[2][KK];
  uint32_t v[8][VW];
};

__device__ __forceinline__ float shfl_xor(float v, int m) { return __shfl_xor(v, m, 64); }

// D_FULL: dim == DT, no dims to mask.  P8: page_size a multiple of 8, so that 8
// aligned tokens share a page.
template <typename T, int DT, bool D_FULL, bool P8>
__global__ __launch_bounds__(kWaves * 64) void paged_attention_kernel(AttnArgs a) {
  using F = Frag<T>;
  using V8 = typename F::V;
  constexpr int KK = Tile<DT>::KK, VW = Tile<DT>::VW, VE = DT / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  int id = blockIdx.x;
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int hk = id % a.hkv, b = id / a.hkv;
  const int rows = min(kHeads, a.group - tile * kHeads);  // query heads here
  const int h0 = hk * a.group + tile * kHeads;
  const int D = D_FULL ? DT : a.dim;

  const int32_t len = a.lens[b];
  const bool over = len > a.capacity;
  const int n = over ? 0 : max(len, 0);
  const int lo = a.window > 0 ? max(0, n - a.window) : 0;
  const int32_t* table = a.table + b * a.ld_table;

  V8 qf[KK];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_ts + (h0 + min(c, rows - 1)) * a.q_hs;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const int d = k * 32 + g * 8;
      const bool in = c < rows && (D_FULL || d < D);
      const v4u32_t w = *reinterpret_cast<const any4*>(q + (D_FULL || d < D ? d : 0));
      qf[k] = __builtin_bit_cast(V8, in ? w : v4u32_t(0u));
    }
  }
  const T* kbase = static_cast<const T*>(a.kc) + hk * a.khs;
  const T* vbase = static_cast<const T*>(a.vc) + hk * a.vhs;

  // The cache row of a token: false when its page number is out of range (row 0
  // is read instead).
  auto locate = [&](int tok, int64_t* page, int64_t* off) {
    const uint32_t p = static_cast<uint32_t>(tok) / a.page_size;
    const uint32_t id = static_cast<uint32_t>(table[p]);
    *off = static_cast<uint32_t>(tok) - p * a.page_size;
    const bool good = id < a.pages;
    *page = good ? id : 0;
    return good;
  };

  float m = -__builtin_huge_valf(), l = 0.0f;
  v4f32 acc[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] = v4f32(0.0f);
  const float scale2 = a.scale * kLog2e;

  for (int base = (lo & ~(kTile - 1)) + wave * kTile; base < n; base += kWaves * kTile) {
    // Tokens outside [lo, n) are read as the nearest one inside.
    auto inside = [&](int tok) { return min(max(tok, lo), n - 1); };
    Tile<DT> t;
    bool kgood[2];
    const T* krow[2];
    const T* vrow[8];
    if constexpr (P8) {
      // The 8 tokens of a group: their page once, rows a stride apart.  A group
      // that the range cuts takes its tokens one by one.
      int64_t page, off;
      const int kt = base + 8 * (c >> 2), vt = base + 8 * g;
      const bool good = locate(inside(kt), &page, &off);
      const int64_t koff = off - (inside(kt) - kt);  // of the group's first token
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kgood[u] = good;
        const int64_t o = koff + inside(kt + 4 * u + (c & 3)) - kt;
        krow[u] = kbase + page * a.kps + o * a.kts;
      }
      locate(inside(vt), &page, &off);
      const int64_t voff = off - (inside(vt) - vt);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        vrow[j] = vbase + page * a.vps + (voff + inside(vt + j) - vt) * a.vts;
    } else {
      int64_t page, off;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kgood[u] = locate(inside(base + 8 * (c >> 2) + 4 * u + (c & 3)), &page, &off);
        krow[u] = kbase + page * a.kps + off * a.kts;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        locate(inside(base + 8 * g + j), &page, &off);
        vrow[j] = vbase + page * a.vps + off * a.vts;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const int d = k * 32 + g * 8;
        const v4u32_t w = *reinterpret_cast<const any4*>(krow[u] + (D_FULL || d < D ? d : 0));
        t.k[u][k] = D_FULL || d < D ? w : v4u32_t(0u);
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (DT == 64) {
        const u32x2 w = *reinterpret_cast<const any2*>(vrow[j] + (D_FULL || 4 * c < D ? 4 * c : 0));
        t.v[j][0] = w[0], t.v[j][1] = w[1];
      } else {
#pragma unroll
        for (int s = 0; s < DT / 128; ++s) {
          const int d = 128 * s + 8 * c;
          const v4u32_t w = *reinterpret_cast<const any4*>(vrow[j] + (D_FULL || d < D ? d : 0));
#pragma unroll
          for (int x = 0; x < 4; ++x) t.v[j][4 * s + x] = w[x];
        }
      }
    }

    // S^T: the scores of head c at tokens base + 8g + 4u + i.
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      v4f32 d = v4f32(0.0f);
#pragma unroll
      for (int k = 0; k < KK; ++k) d = F::mfma(__builtin_bit_cast(V8, t.k[u][k]), qf[k], d);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * u + i] = d[i] * scale2;
    }
    // A token on a bad page poisons its sequence.  The lane that loaded token 8g
    // + 4u + i is lane 4g + i (of any 16).
    bool bad = !kgood[0] || !kgood[1];
    if (__any(bad)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = __builtin_nanf("");
    }
    if (base < lo || base + kTile > n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = base + 8 * g + j;
        const bool in = tok >= lo && tok < n;
        s[j] = in ? s[j] : -__builtin_huge_valf();
        // 0 * V must be 0 for what lies in the cache there.
#pragma unroll
        for (int x = 0; x < VW; ++x) t.v[j][x] = in ? t.v[j][x] : 0u;
      }
    }
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, shfl_xor(top, 16));
      top = fmaxf(top, shfl_xor(top, 32));
      const float mn = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(m - (mn == -__builtin_huge_valf() ? 0.0f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] *= alpha;
    }
    const float ref = (m == -__builtin_huge_valf() ? 0.0f : m) - F::kShift;
    V8 p;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = __builtin_amdgcn_exp2f(s[j] - ref);
      l += e;
      p[j] = fromf<T>(e);
    }
    // O^T: dims of this lane's transposed 8-token columns.
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      v4u32_t col;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        col[w] = __builtin_amdgcn_perm(t.v[2 * w + 1][e / 2], t.v[2 * w][e / 2],
                                       e & 1 ? 0x07060302u : 0x05040100u);
      acc[e] = F::mfma(__builtin_bit_cast(V8, col), p, acc[e]);
    }
  }

  // Joins the waves: outputs [wave][head][dim] with their maximum and sum.
  constexpr int PITCH = DT + 4;
  __shared__ __align__(16) float so[kWaves][kHeads][PITCH];
  __shared__ float sm[kWaves][kHeads], sl[kWaves][kHeads];
  l += shfl_xor(l, 16);
  l += shfl_xor(l, 32);
  if (g == 0) sm[wave][c] = m, sl[wave][c] = l;
  // acc[e][i] is dim VE' * (4g + i) + e' of head c, VE' = min(VE, 8).
  constexpr int VC = VE < 8 ? VE : 8;
#pragma unroll
  for (int e = 0; e < VE; e += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f32 w;
#pragma unroll
      for (int x = 0; x < 4; ++x) w[x] = acc[e + x][i];
      *reinterpret_cast<v4f32*>(&so[wave][c][(e / 8) * 128 + VC * (4 * g + i) + e % 8]) = w;
    }
  __syncthreads();
  const bool nothing = n == 0;
  for (int x = threadIdx.x; x < rows * D; x += kWaves * 64) {
    const int h = x / D, d = x - h * D;
    float M = sm[0][h];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm[w][h]);
    const float ref = M == -__builtin_huge_valf() ? 0.0f : M;
    float o = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][h] - ref);
      o = fmaf(f, so[w][h][d], o);
      L = fmaf(f, sl[w][h], L);
    }
    o = over ? __builtin_nanf("") : nothing ? 0.0f : o / L;
    static_cast<T*>(a.out)[b * a.o_ts + (h0 + h) * a.o_hs + d] = fromf<T>(o);
    if (d == 0 && a.lse)
      a.lse[static_cast<int64_t>(b) * a.hkv * a.group + h0 + h] =
          over ? __builtin_nanf("")
               : nothing ? -__builtin_huge_valf()
                         : (M + (__builtin_amdgcn_logf(L) - F::kShift)) * 0.6931471805599453f;
  }
}

template <typename T, int DT>
hxm_status launch_attention(const AttnArgs& a, int64_t groups, hipStream_t stream) {
  const unsigned n = static_cast<unsigned>(groups);
  const bool full = a.dim == DT, p8 = a.page_size % 8 == 0;
  if (full && p8) paged_attention_kernel<T, DT, true, true><<<n, kWaves * 64, 0, stream>>>(a);
  else if (full) paged_attention_kernel<T, DT, true, false><<<n, kWaves * 64, 0, stream>>>(a);
  else if (p8) paged_attention_kernel<T, DT, false, true><<<n, kWaves * 64, 0, stream>>>(a);
  else paged_attention_kernel<T, DT, false, false><<<n, kWaves * 64, 0, stream>>>(a);
  return check_launch("paged attention");
}

template <typename T>
hxm_status launch_attention_dim(const AttnArgs& a, int64_t groups, hipStream_t stream) {
  if (a.dim <= 64) return launch_attention<T, 64>(a, groups, stream);
  if (a.dim <= 128) return launch_attention<T, 128>(a, groups, stream);
  return launch_attention<T, 256>(a, groups, stream);
}

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_paged_attention(const hxm_heads* q, const hxm_heads* out,
                                          int64_t q_heads, const hxm_kv_cache* cache,
                                          const int32_t* block_table, int64_t ld_table,
                                          int64_t table_pages, const int32_t* seq_lens,
                                          int64_t batch, float scale, int64_t window, float* lse,
                                          int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE,
                "unsupported-dtype: paged_attention takes f16 or bf16 (got %d)", dtype);
  hxm_status st = check_kv_cache("paged_attention", cache, false);
  if (st != HXM_OK) return st;
  if (batch < 0 || q_heads < 1 || q_heads % cache->heads != 0 || window < 0)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: paged_attention batch=%lld, %lld query heads over %lld, "
                "window=%lld",
                (long long)batch, (long long)q_heads, (long long)cache->heads, (long long)window);
  if (q_heads > 65535 || batch > INT32_MAX / 65536)
    return fail(HXM_UNSUPPORTED_SHAPE, "tile-alignment: paged_attention batch=%lld, %lld heads",
                (long long)batch, (long long)q_heads);
  if ((st = check_heads("paged_attention", "q", q, batch, q_heads, cache->dim, false)) != HXM_OK ||
      (st = check_heads("paged_attention", "out", out, batch, q_heads, cache->dim, true)) != HXM_OK)
    return st;
  if (batch > 0 && !heads_same(out, q, batch, q_heads) &&
      !heads_apart(out, q_heads, q, q_heads, batch, cache->dim))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: paged_attention out overlaps q without being it");
  if (table_pages < 0 || table_pages > INT32_MAX || !stride_ok(ld_table) ||
      (batch > 1 && ld_table < table_pages) ||
      (batch > 0 && (!seq_lens || (table_pages > 0 && !block_table))))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: paged_attention table of %lld pages, ld %lld, or null lengths",
                (long long)table_pages, (long long)ld_table);
  if (!(scale == scale))
    return fail(HXM_INVALID_ARG, "invalid-argument: paged_attention scale is NaN");
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (batch == 0) return ok();
  AttnArgs a{};
  a.q = q->data, a.q_ts = q->token_stride, a.q_hs = q->head_stride;
  a.out = out->data, a.o_ts = out->token_stride, a.o_hs = out->head_stride;
  a.kc = cache->k, a.vc = cache->v;
  a.kps = cache->k_page_stride, a.khs = cache->k_head_stride, a.kts = cache->k_token_stride;
  a.vps = cache->v_page_stride, a.vhs = cache->v_head_stride, a.vts = cache->v_token_stride;
  a.table = block_table, a.lens = seq_lens, a.lse = lse;
  a.ld_table = ld_table, a.capacity = table_pages * cache->page_size;
  a.pages = static_cast<uint32_t>(cache->pages);
  a.page_size = static_cast<uint32_t>(cache->page_size);
  a.hkv = static_cast<int>(cache->heads);
  a.group = static_cast<int>(q_heads / cache->heads);
  a.tiles = static_cast<int>(ceil_div(a.group, kHeads));
  a.dim = static_cast<int>(cache->dim);
  a.window = window > INT32_MAX ? 0 : static_cast<int>(window);
  a.scale = scale;
  const int64_t groups = batch * a.hkv * a.tiles;
  if ((st = check_grid("paged attention", groups, kWaves * 64)) != HXM_OK) return st;
  return dtype == HXM_F16 ? launch_attention_dim<_Float16>(a, groups, as_stream(stream))
                          : launch_attention_dim<__bf16>(a, groups, as_stream(stream));
}
