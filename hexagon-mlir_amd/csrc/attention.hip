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
#include <algorithm>
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
constexpr int64_t kTarget = 1024;  // workgroups a batch is split into

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
  float* parts;
  uint32_t* counts;
  int parts_bytes, slot_rows;
  uint32_t pages, page_size;
  FastDiv page_div;
  int batch, hkv, group, tiles, heads, dim, window;  // heads: hkv * tiles
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

__device__ __forceinline__ float shfl_xor(float v, int m) { return __shfl_xor(v, m, 64); }

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  // Row totals by DPP, then the four rows'.
  auto step = [&](auto ctrl) {
    v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v),
                                                           decltype(ctrl)::value, 0xF, 0xF, true));
  };
  step(std::integral_constant<int, kDppQuadXor1>{});
  step(std::integral_constant<int, kDppQuadXor2>{});
  step(std::integral_constant<int, kDppRowHalfMirror>{});
  step(std::integral_constant<int, kDppRowMirror>{});
  const int i = static_cast<int>(v);
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(i, 0)) +
         static_cast<uint32_t>(__builtin_amdgcn_readlane(i, 16)) +
         static_cast<uint32_t>(__builtin_amdgcn_readlane(i, 32)) +
         static_cast<uint32_t>(__builtin_amdgcn_readlane(i, 48));
}

// Sum of v over lanes 0 .. lane.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {
  auto step = [&](auto ctrl) {  // row_shr by 1, 2, 4, 8; zeros come in
    v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v),
                                                           decltype(ctrl)::value, 0xF, 0xF, true));
  };
  step(std::integral_constant<int, 0x111>{});
  step(std::integral_constant<int, 0x112>{});
  step(std::integral_constant<int, 0x114>{});
  step(std::integral_constant<int, 0x118>{});
  const uint32_t r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31),
                 r2 = __builtin_amdgcn_readlane(v, 47);
  return v + (lane >= 16 ? r0 : 0u) + (lane >= 32 ? r1 : 0u) + (lane >= 48 ? r2 : 0u);
}

// A workgroup's piece of the batch.
struct Piece {
  int b;             // sequence, -1: none
  int n, lo;         // its tokens [lo, n)
  int begin, end;    // the piece's, begin a multiple of 32
  int pieces, index; // of the sequence, and this one
  uint32_t slot;     // of its first partial result (pieces > 1)
  bool over;         // longer than its table row
};

// Piece number u of the batch, its sequences in order.  Every wave works it out
// from the lengths (they are on the device: the host cannot), 64 sequences at a
// time; a batch of 64 or fewer reads them once.
__device__ __forceinline__ Piece find_piece(const AttnArgs& a, uint32_t u, int lane) {
  auto length = [&](int b, int* lo, bool* over) {
    const int32_t len = b < a.batch ? a.lens[b] : 0;
    *over = len > a.capacity;
    const int n = *over ? 0 : max(len, 0);
    *lo = a.window > 0 ? max(0, n - a.window) : 0;
    return n;
  };
  auto units = [](int n, int lo) {
    return static_cast<uint32_t>((n - (lo & ~(kTile - 1)) + kTile - 1) / kTile);
  };
  int lo;
  bool over;
  int n = length(lane, &lo, &over);
  uint32_t w = units(n, lo);
  uint64_t total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (b0 > 0) {
      int l2;
      bool o2;
      const int n2 = length(b0 + lane, &l2, &o2);
      w = units(n2, l2);
    }
    // 2^26 units a lane: 64 of them do not fit 32 bits.
    total += wave_sum(w & 0xffffu) + (static_cast<uint64_t>(wave_sum(w >> 16)) << 16);
  }
  const uint32_t piece = static_cast<uint32_t>(
      min(attn_piece(static_cast<int64_t>(total), a.heads, kTarget), int64_t(1) << 30));
  Piece r{};
  r.b = -1;
  uint32_t first = 0, slots = 0;  // pieces and partial slots of the sequences before
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) n = length(b0 + lane, &lo, &over);
    w = units(n, lo);
    const uint32_t c = b0 + lane < a.batch ? max(1u, (w + piece - 1) / piece) : 0u;
    const uint32_t upto = wave_scan(c, lane);
    const uint32_t cs = c > 1 ? c : 0u, upto_s = wave_scan(cs, lane);
    const uint64_t hit = __ballot(u < first + upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto at = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, l)); };
      r.b = b0 + l;
      r.n = static_cast<int>(at(n)), r.lo = static_cast<int>(at(lo));
      r.over = at(over) != 0;
      r.pieces = static_cast<int>(at(c));
      r.index = static_cast<int>(u - (first + at(upto) - at(c)));
      r.slot = slots + at(upto_s) - at(cs);
      r.begin = (r.lo & ~(kTile - 1)) + r.index * static_cast<int>(piece) * kTile;
      r.end = r.index + 1 < r.pieces ? r.begin + static_cast<int>(piece) * kTile : r.n;
      return r;
    }
    first += __builtin_amdgcn_readlane(upto, 63);
    slots += __builtin_amdgcn_readlane(upto_s, 63);
  }
  return r;
}

// D_FULL: dim == DT, no dims to mask.  P8: page_size a multiple of 8, so that 8
// aligned tokens share a page.
template <typename T, int DT, bool D_FULL, bool P8>
__global__ __launch_bounds__(kWaves * 64) void paged_attention_kernel(AttnArgs a) {
  using F = Frag<T>;
  using V8 = typename F::V;
  constexpr int KK = DT / 32;         // K steps of the first product
  constexpr int VW = DT / 32;         // dwords of a token's DT / 16 value dims in a lane
  constexpr int VE = DT / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  const int head = blockIdx.x % a.heads;
  const Piece w = find_piece(a, blockIdx.x / a.heads, lane);
  if (w.b < 0) return;
  const int tile = head % a.tiles, hk = head / a.tiles;
  const int rows = min(kHeads, a.group - tile * kHeads);  // query heads here
  const int h0 = hk * a.group + tile * kHeads;
  const int D = D_FULL ? DT : a.dim;
  const int b = w.b, n = w.n, lo = w.lo;
  const int32_t* table = a.table + b * a.ld_table;

  V8 qf[KK];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_ts + (h0 + min(c, rows - 1)) * a.q_hs;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const int d = k * 32 + g * 8;
      const bool in = c < rows && (D_FULL || d < D);
      const v4u32_t x = *reinterpret_cast<const any4*>(q + (D_FULL || d < D ? d : 0));
      qf[k] = __builtin_bit_cast(V8, in ? x : v4u32_t(0u));
    }
  }
  const T* kbase = static_cast<const T*>(a.kc) + hk * a.khs;
  const T* vbase = static_cast<const T*>(a.vc) + hk * a.vhs;

  // The tokens whose K and V rows a lane loads: keys base + 8 (c / 4) + 4u + c % 4,
  // values base + 8g + j.  Those outside [lo, n) are read as others that are
  // inside, or beside them in their page, and masked below.
  auto inside = [&](int tok) { return min(max(tok, lo), n - 1); };
  auto page_of = [&](int tok) {
    return static_cast<uint32_t>((static_cast<uint64_t>(tok) * a.page_div.mul) >>
                                 a.page_div.shift);
  };
  constexpr int NK = P8 ? 1 : 2, NV = P8 ? 1 : 8;
  struct Pages {  // page numbers of the lane's key and value tokens
    int32_t k[NK], v[NV];
  };
  auto key_token = [&](int base, int u) {
    return P8 ? base + 8 * (c >> 2) : base + 8 * (c >> 2) + 4 * u + (c & 3);
  };
  auto value_token = [&](int base, int j) { return base + 8 * g + (P8 ? 0 : j); };
  auto fetch_pages = [&](int base, Pages& p) {
#pragma unroll
    for (int u = 0; u < NK; ++u) p.k[u] = table[page_of(inside(key_token(base, u)))];
#pragma unroll
    for (int j = 0; j < NV; ++j) p.v[j] = table[page_of(inside(value_token(base, j)))];
  };
  // The offset in its page; of an aligned group of 8, that of its first token.
  auto offset = [&](int tok) {
    const int t = inside(tok);
    const int off = t - static_cast<int>(page_of(t) * a.page_size);
    return P8 ? off & ~7 : off;
  };
  auto row = [&](const T* base, int32_t page, int off, int64_t ps, int64_t ts) {
    const bool good = static_cast<uint32_t>(page) < a.pages;
    return base + (good ? page : 0) * ps + off * ts;
  };

  v4u32_t kt[2][KK];
  uint32_t vt[8][VW];
  auto load_keys = [&](int base, const Pages& p) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int off = offset(key_token(base, u)) + (P8 ? 4 * u + (c & 3) : 0);
      const T* r = row(kbase, p.k[P8 ? 0 : u], off, a.kps, a.kts);
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        const int d = k * 32 + g * 8;
        const v4u32_t x = *reinterpret_cast<const any4*>(r + (D_FULL || d < D ? d : 0));
        kt[u][k] = D_FULL || d < D ? x : v4u32_t(0u);
      }
    }
  };
  auto load_values = [&](int base, const Pages& p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int off = offset(value_token(base, j)) + (P8 ? j : 0);
      const T* r = row(vbase, p.v[P8 ? 0 : j], off, a.vps, a.vts);
      if constexpr (DT == 64) {
        const u32x2 x = *reinterpret_cast<const any2*>(r + (D_FULL || 4 * c < D ? 4 * c : 0));
        vt[j][0] = x[0], vt[j][1] = x[1];
      } else {
#pragma unroll
        for (int s = 0; s < DT / 128; ++s) {
          const int d = 128 * s + 8 * c;
          const v4u32_t x = *reinterpret_cast<const any4*>(r + (D_FULL || d < D ? d : 0));
#pragma unroll
          for (int y = 0; y < 4; ++y) vt[j][4 * s + y] = x[y];
        }
      }
    }
  };

  float m = -__builtin_huge_valf(), l = 0.0f;
  v4f32 acc[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] = v4f32(0.0f);
  const float scale2 = a.scale * kLog2e;

  // One tile; more: its successor's keys are loaded as soon as the scores are
  // made, its values as soon as this tile's are used, into the same registers.
  Pages here, next;
  auto step = [&](int base, auto more) {
    constexpr bool MORE = decltype(more)::value;
    // S^T: the scores of head c at tokens base + 8g + 4u + i.
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      v4f32 d = v4f32(0.0f);
#pragma unroll
      for (int k = 0; k < KK; ++k) d = F::mfma(__builtin_bit_cast(V8, kt[u][k]), qf[k], d);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * u + i] = d[i] * scale2;
    }
    // A token on a bad page poisons its sequence (the lanes' keys are all the
    // tile's tokens).
    bool bad = false;
#pragma unroll
    for (int u = 0; u < NK; ++u) bad |= static_cast<uint32_t>(here.k[u]) >= a.pages;
    const bool poisoned = __any(bad);
    const int after = base + kWaves * kTile;
    if constexpr (MORE) {
      here = next;
      load_keys(after, here);
      fetch_pages(after + kWaves * kTile, next);
    }
    if (poisoned) {
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
        for (int x = 0; x < VW; ++x) vt[j][x] = in ? vt[j][x] : 0u;
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
      for (int x = 0; x < 4; ++x)
        col[x] = __builtin_amdgcn_perm(vt[2 * x + 1][e / 2], vt[2 * x][e / 2],
                                       e & 1 ? 0x07060302u : 0x05040100u);
      acc[e] = F::mfma(__builtin_bit_cast(V8, col), p, acc[e]);
    }
    if constexpr (MORE) load_values(after, here);
  };
  int base = w.begin + wave * kTile;
  if (base < w.end) {
    fetch_pages(base, here);
    load_keys(base, here);
    load_values(base, here);
    fetch_pages(base + kWaves * kTile, next);
    for (; base + kWaves * kTile < w.end; base += kWaves * kTile) step(base, std::true_type{});
    step(base, std::false_type{});
  }

  // Joins the waves: outputs [wave][head][dim] with their maximum and sum.
  constexpr int PITCH = DT + 4;
  __shared__ __align__(16) float so[kWaves][kHeads][PITCH];
  __shared__ float sm[kWaves][kHeads], sl[kWaves][kHeads];
  l += shfl_xor(l, 16);
  l += shfl_xor(l, 32);
  if (g == 0) sm[wave][c] = m, sl[wave][c] = l;
  // acc[e][i] is dim VC * (4g + i) + e of head c (of each 128 dims).
  constexpr int VC = VE < 8 ? VE : 8;
#pragma unroll
  for (int e = 0; e < VE; e += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f32 x;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = acc[e + y][i];
      *reinterpret_cast<v4f32*>(&so[wave][c][(e / 8) * 128 + VC * (4 * g + i) + e % 8]) = x;
    }
  __syncthreads();

  // Output dims 4d .. 4d + 3 of head h from their sums o, relative to maximum M
  // with normaliser L.
  auto finish = [&](int h, int d, v4f32 o, float M, float L) {
    T* out = static_cast<T*>(a.out) + b * a.o_ts + (h0 + h) * a.o_hs + 4 * d;
    const bool nothing = n == 0;
    const float inv = 1.0f / L;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[e] = fromf<T>(w.over ? __builtin_nanf("") : nothing ? 0.0f : o[e] * inv);
    if (d == 0 && a.lse)
      a.lse[static_cast<int64_t>(b) * a.hkv * a.group + h0 + h] =
          w.over ? __builtin_nanf("")
                 : nothing ? -__builtin_huge_valf()
                           : (M + (__builtin_amdgcn_logf(L) - F::kShift)) * 0.6931471805599453f;
  };
  auto finite = [](float M) { return M == -__builtin_huge_valf() ? 0.0f : M; };
  const int d4 = D / 4, items = rows * d4;
  const int slot_floats = a.slot_rows * (a.dim + 2);
  // Partial results: maxima and sums [rows][2], then outputs [rows][dim], of each
  // piece.  Written through to the coherence point and read back from it (sc1):
  // the workgroups of a sequence run on different XCDs, whose L2s do not see
  // each other.
  const __amdgpu_buffer_rsrc_t parts = __builtin_amdgcn_make_buffer_rsrc(
      a.parts, static_cast<short>(0), a.parts_bytes, 0x00020000);
  constexpr int kSc1 = 16;
  const uint32_t slot0 = (w.slot * a.heads + head * static_cast<uint32_t>(w.pieces));
  auto part_at = [&](int s, int word) {
    return (static_cast<uint32_t>(slot0 + s) * static_cast<uint32_t>(slot_floats) +
            static_cast<uint32_t>(word)) * 4u;
  };
  for (int x = threadIdx.x; x < items; x += kWaves * 64) {
    const int h = x / d4, d = x - h * d4;
    float M = sm[0][h];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) M = fmaxf(M, sm[v][h]);
    v4f32 o = v4f32(0.0f);
    float L = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(sm[v][h] - finite(M));
      const v4f32 y = *reinterpret_cast<const v4f32*>(&so[v][h][4 * d]);
      L = fmaf(f, sl[v][h], L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, y[e], o[e]);
    }
    if (w.pieces == 1) {
      finish(h, d, o, M, L);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u32_t, o), parts,
                                             part_at(w.index, 2 * a.slot_rows + h * a.dim + 4 * d),
                                             0, kSc1);
      if (d == 0) {
        const u32x2 ml = {__builtin_bit_cast(uint32_t, M), __builtin_bit_cast(uint32_t, L)};
        __builtin_amdgcn_raw_buffer_store_b64(ml, parts, part_at(w.index, 2 * h), 0, kSc1);
      }
    }
  }
  if (w.pieces == 1) return;

  // The workgroup that arrives last joins the pieces, in their order whichever
  // it is, and clears the counter for the next launch.  Nobody waits.
  __shared__ int last;
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if (threadIdx.x == 0) {
    uint32_t* count = a.counts + static_cast<int64_t>(b) * a.heads + head;
    const uint32_t before =
        __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = before == static_cast<uint32_t>(w.pieces - 1);
    if (last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  // NG groups of threads take consecutive shares of the pieces, eight loads in
  // flight each, and are joined through LDS.
  int NG = 1;
  while (2 * NG * items <= kWaves * 64 && 2 * NG <= w.pieces) NG *= 2;
  const int grp = static_cast<int>(threadIdx.x) / min(items, kWaves * 64);
  const int s_begin = static_cast<int>(static_cast<int64_t>(w.pieces) * grp / NG);
  const int s_end = static_cast<int>(static_cast<int64_t>(w.pieces) * (grp + 1) / NG);
  struct Joined {
    v4f32 o;
    float M, L;
  };
  auto merge = [&](Joined& j, v4f32 o, float M, float L) {
    const float mn = fmaxf(j.M, M);
    const float fa = __builtin_amdgcn_exp2f(j.M - finite(mn));
    const float fb = __builtin_amdgcn_exp2f(M - finite(mn));
    j.M = mn;
    j.L = fmaf(fb, L, fa * j.L);
#pragma unroll
    for (int e = 0; e < 4; ++e) j.o[e] = fmaf(fb, o[e], fa * j.o[e]);
  };
  Joined* shared = reinterpret_cast<Joined*>(&so[0][0][0]);
  static_assert(sizeof(Joined) == 32 && sizeof(so) >= kWaves * 64 * sizeof(Joined), "LDS of a join");
  for (int x = static_cast<int>(threadIdx.x) % min(items, kWaves * 64); x < items && grp < NG;
       x += kWaves * 64) {
    const int h = x / d4, d = x - h * d4;
    Joined j{v4f32(0.0f), -__builtin_huge_valf(), 0.0f};
    for (int s = s_begin; s < s_end; s += 8) {
      v4u32_t o[8];
      u32x2 ml[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int si = min(s + i, s_end - 1);
        o[i] = __builtin_amdgcn_raw_buffer_load_b128(
            parts, part_at(si, 2 * a.slot_rows + h * a.dim + 4 * d), 0, kSc1);
        ml[i] = __builtin_amdgcn_raw_buffer_load_b64(parts, part_at(si, 2 * h), 0, kSc1);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s + i < s_end) {
          const uint32_t mi = ml[i][0], li = ml[i][1];
          merge(j, __builtin_bit_cast(v4f32, o[i]), __builtin_bit_cast(float, mi),
                __builtin_bit_cast(float, li));
        }
    }
    if (NG == 1) finish(h, d, j.o, j.M, j.L);
    else shared[grp * items + x] = j;
  }
  if (NG == 1) return;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < items) {
    const int x = threadIdx.x, h = x / d4, d = x - h * d4;
    Joined j = shared[x];
    for (int k = 1; k < NG; ++k) {
      const Joined o = shared[k * items + x];
      merge(j, o.o, o.M, o.L);
    }
    finish(h, d, j.o, j.M, j.L);
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
  a.page_div = fast_div(a.page_size);
  a.batch = static_cast<int>(batch);
  a.hkv = static_cast<int>(cache->heads);
  a.group = static_cast<int>(q_heads / cache->heads);
  a.tiles = static_cast<int>(ceil_div(a.group, kHeads));
  a.heads = a.hkv * a.tiles;
  a.dim = static_cast<int>(cache->dim);
  a.window = window > INT32_MAX ? 0 : static_cast<int>(window);
  a.scale = scale;
  // Partial results of at most 2 * kTarget pieces, 34 MB for the largest heads,
  // and a counter for each sequence and head, zero between launches.
  a.slot_rows = std::min(a.group, kHeads);
  const int64_t parts = 2 * kTarget * a.slot_rows * (a.dim + 2) * 4;
  const int64_t counts = batch * a.heads * 4;
  void* ws = nullptr;
  hipStream_t s = as_stream(stream);
  if ((st = stream_workspace(s, static_cast<size_t>(counts), &ws, kWsCount)) != HXM_OK) return st;
  a.counts = static_cast<uint32_t*>(ws);
  if ((st = stream_workspace(s, static_cast<size_t>(parts), &ws, kWsLayer)) != HXM_OK) return st;
  a.parts = static_cast<float*>(ws);
  a.parts_bytes = static_cast<int>(parts);
  const int64_t groups = kTarget + batch * a.heads;
  if ((st = check_grid("paged attention", groups, kWaves * 64)) != HXM_OK) return st;
  return dtype == HXM_F16 ? launch_attention_dim<_Float16>(a, groups, s)
                          : launch_attention_dim<__bf16>(a, groups, s);
}
