// Attention of one new token per sequence over the paged key-value cache.
//
// Bound by memory: the keys and values of a sequence are read once per key
// head, 4 * dim bytes a token, against 4 * dim * group operations.  The group of
// query heads that shares a key head is the 16-wide side of the MFMAs (padded
// with zeros), so one read serves a group of up to 16.  Larger ones are read once for every
// 16 of them, by workgroups apart (8 x 32768 tokens, 2 heads of 128: groups of 16 take 41 us,
// 17 and 32 64, 48 94).
//
// A wave takes 32 tokens at a time, in two steps whose data stays in registers.
// S^T = K Q^T, K the left operand, leaves lane (g, c) = (lane / 16, lane % 16)
// scores of head c; the rows of the two 16-token products are assigned so that
// they are those of tokens 4j + g, j < 8.  O^T = V^T P^T wants exactly those of P^T as its
// right operand, so the probabilities go from one product to the other in the lane they
// are in, and running maximum, sum and output of a head live in one column
// of lanes.
//
// Keys and values come in whole rows, 1 KiB of neighbouring bytes an instruction in the
// order of a page, nontemporal: a workgroup reads nothing twice.  (Keys loaded in the operand's
// own layout, 64 bytes of 16 rows an instruction, read every line in two halves, which the
// caches have to join.  With that layout and three pieces a CU, 8 x 32768 tokens, 8 heads of
// 128, took 98 us where this takes 86, 32 x 4096, 4 heads of 256, 65 and 49; but 16 windows of
// 1000 tokens, one head of 64, took 8.6 and take 10.2, 1 x 2000 tokens 9.8 and 11.3: a tile's
// way through LDS is longer than its own loads.)  A lane then holds 8 tokens x dim / 16 dims of V and transposes them in registers
// with byte permutes; K becomes the left operand through the wave's own piece of LDS, where
// row t has its 16-byte chunk q at q ^ t % 16 (of 8 chunks: q ^ t / 2 % 8, two rows to all
// 64 banks), so that neither side meets a bank twice.  The next tile's keys are on their
// way as soon as this one's are in LDS, its values as soon as this one's are used.
//
// The running maximum moves only when a score passes it by more than 2^8 in
// the exponent's base 2: exp2(s - m) stays far below fp32's limit, and the
// output is rescaled a few times per sequence and not per tile.  The probabilities enter
// the second product as two 16-bit halves (22 bits of them in f16, 16 in bf16;
// one half alone added as much to the error as the output's own rounding, and the
// second costs no time that shows: 98.3 against 98.5 us).  f16 ones are scaled by
// 2^7 on the way, so that with those 8 binary orders of headroom they stay below
// 65504 and the smallest normal one is 2^-21 of the largest; the second half, 2^-24 at least, is
// off by up to 2^-32 of the largest, which is more than 22 bits leave of one below 2^-10 of it.
#include <algorithm>
#include <type_traits>

#include "attention_cut.h"
#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kTile = kAttnTile;  // tokens of a wave's step
constexpr int kHeads = 16;        // query heads of a workgroup
constexpr int kWaves = 4;
constexpr int kUnit = kWaves * kTile;
static_assert(kUnit == kAttnUnit, "a unit is one step of all waves");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;  // of the running maximum, in powers of two

// The pieces (kAttnGroups and kAttnFine): one for each CU where the sequences allow it.
// What a workgroup has under way (a tile of each wave) keeps its CU at its share of the
// memory's rate, fewer pieces are fewer to join, and all run at once.  More at once only
// starve each other: with three workgroups a CU, 8 x 32768 tokens, the first to end took 31
// us and the last 79; 32768 tokens of one sequence, 8 heads of 8, 32 us with 256 pieces, 42
// with 768.  Where sequences times heads are more than that, three times as many pieces
// level what their lengths differ by (16 x 8192 tokens at most, 32 heads: 150 us with 2,
// 141 with 3, 143 with 4 and more; 64 x 4096, 8 heads: 81.5, 80.7, 80.7).  A join costs
// about what three units do, so four units are left whole (1 x 300 tokens, 32 heads: 8.8 us
// whole, 10.3 in two; 8 x 500, 8 heads, 10.0 and 10.8); of longer ones pieces of two units are worth it (the least piece two or
// four units, and four or eight left whole: 1 x 700 tokens, 8 heads, 10.8 and 12.2 us; 1 x 2000
// 11.3 and 13.3; 32 x 1000, one head, 10.9 and 14.5; 8 x 32768 the same).

// Waves a SIMD, by the registers of a tile and the output: many short sequences hide each
// other's start.  Rows located one by one need a few registers more, and spill with 128.
constexpr int attn_waves(int dt, bool p8) {
  return dt <= 64 ? (p8 ? 4 : 3) : dt <= 128 ? 2 : 1;
}

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

// D_FULL: dim == DT, no dims to mask (masked all the same: 8 x 32768 tokens, 8 heads of 128,
// 85.4 us for 84; 32 x 4096, 4 heads of 256, 50.6 for 49.4).  P8: page_size a multiple of 8, and
// 8 rows of a page within 2^31 bytes: the tile's four groups of 8 tokens then have one
// page each, whose number and address the scalar unit works out (rows located one by one over
// the same pages of 16 take 94 us for 84, 58.4 for 51.5 at 64 x 4096, 8 heads of 64, and 144
// for 49.4 at 256 dims, where one wave a SIMD waits for each table entry).
template <typename T, int DT, bool D_FULL, bool P8>
__global__ __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(attn_waves(DT, P8)))) void paged_attention_kernel(AttnArgs a) {
  using F = Frag<T>;
  using V8 = typename F::V;
  constexpr int KK = DT / 32;       // K steps of the first product
  constexpr int VW = DT / 32;       // dwords of a token's value dims in a lane
  constexpr int VE = DT / 16;       // and dims
  constexpr int CK = DT / 8;        // 16-byte chunks of a key row
  constexpr int RI = 64 / CK;       // key rows of a load
  constexpr int KI = kTile / RI;    // loads of a tile's keys
  constexpr int PITCH = DT + 4;     // floats of a row of the join
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int g = lane >> 4, c = lane & 15;
  // Keys of the waves' tiles, and after the last one the waves' outputs.
  constexpr int kKeyBytes = kTile * DT * 2, kOutBytes = kHeads * PITCH * 4;
  constexpr int kWaveBytes = kKeyBytes > kOutBytes ? kKeyBytes : kOutBytes;
  __shared__ __align__(16) uint8_t lds[kWaves * kWaveBytes];
  __shared__ float sm[kWaves][kHeads], sl[kWaves][kHeads];
  __shared__ int last;

  const int head = blockIdx.x % a.heads;
  const Piece w = find_piece(a, blockIdx.x / a.heads, lane);
  if (w.b < 0) return;
  const int tile = head % a.tiles, hk = head / a.tiles;
  const int rows = min(kHeads, a.group - tile * kHeads);  // query heads here
  const int h0 = hk * a.group + tile * kHeads;
  const int D = D_FULL ? DT : a.dim;
  const int b = w.b, n = w.n, lo = w.lo;

  // Q^T: dims 32k + 8g .. of head c, zeros for the heads past the last and the dims
  // past D.
  V8 qf[KK];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_ts + (h0 + min(c, rows - 1)) * a.q_hs;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const int d = k * 32 + g * 8;
      const v4u32_t x = *reinterpret_cast<const any4*>(q + (D_FULL || d < D ? d : 0));
      qf[k] = __builtin_bit_cast(V8, c < rows && (D_FULL || d < D) ? x : v4u32_t(0u));
    }
  }
  const T* kbase = static_cast<const T*>(a.kc) + hk * a.khs;
  const T* vbase = static_cast<const T*>(a.vc) + hk * a.vhs;
  // The table is constant memory to this kernel: uniform entries are scalar loads.
  typedef const int32_t __attribute__((address_space(4))) * ConstInts;
  const ConstInts table =
      (ConstInts)(reinterpret_cast<uintptr_t>(a.table + static_cast<int64_t>(b) * a.ld_table));
  auto page_of = [&](int tok) {
    return static_cast<uint32_t>((static_cast<uint64_t>(static_cast<uint32_t>(tok)) *
                                  a.page_div.mul) >> a.page_div.shift);
  };

  // A lane's key rows are tokens RI i + lane / CK (i < KI) in chunk lane % CK, its value
  // rows tokens 4 j + g (j < 8) in dims VC c (VC = 4 or 8, of each 128).
  const int krow = lane / CK, kchunk = lane % CK;
  const int kdim = D_FULL || kchunk * 8 < D ? kchunk * 8 : 0;
  constexpr int VC = VE < 8 ? VE : 8;
  v4u32_t kr[KI];
  uint32_t vt[8][VW];
  auto load_value = [&](int j, const T* r) {  // r: the token's row
    if constexpr (DT == 64) {
      const u32x2 x = __builtin_nontemporal_load(
          reinterpret_cast<const any2*>(r + (D_FULL || VC * c < D ? VC * c : 0)));
      vt[j][0] = x[0], vt[j][1] = x[1];
    } else {
#pragma unroll
      for (int s = 0; s < DT / 128; ++s) {
        const int d = 128 * s + VC * c;
        const v4u32_t x = __builtin_nontemporal_load(
            reinterpret_cast<const any4*>(r + (D_FULL || d < D ? d : 0)));
#pragma unroll
        for (int y = 0; y < 4; ++y) vt[j][4 * s + y] = x[y];
      }
    }
  };
  // Where a tile's rows lie: P8, the page of each group of 8 tokens and the
  // group's offset in it; otherwise nothing, rows are located one by one.  Tokens
  // outside [lo, n) are read from rows of the nearest group inside (or as the
  // nearest token), and masked below.
  struct Where {
    uint32_t page[P8 ? 4 : 1];
    int off[P8 ? 4 : 1];
    bool bad;
  };
  auto locate = [&](int base) {
    Where p{};
    if constexpr (P8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = min(max(base + 8 * i, lo & ~7), (n - 1) & ~7);
        const uint32_t k = page_of(t);
        p.page[i] = static_cast<uint32_t>(table[k]);
        p.off[i] = t - static_cast<int>(k * a.page_size);
      }
    }
    return p;
  };
  auto check = [&](Where& p) {  // page numbers out of range: row 0 is read, the tile poisoned
    if constexpr (P8) {
      p.bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool good = p.page[i] < a.pages;
        p.bad |= !good;
        p.page[i] = good ? p.page[i] : 0u;
      }
    }
  };
  auto row_of = [&](int tok, const T* base, int64_t ps, int64_t ts, bool* bad) {
    const int t = min(max(tok, lo), n - 1);
    const uint32_t k = page_of(t), id = static_cast<uint32_t>(table[k]);
    const bool good = id < a.pages;
    *bad |= !good;
    return base + static_cast<int64_t>(good ? id : 0u) * ps +
           static_cast<int64_t>(t - static_cast<int>(k * a.page_size)) * ts;
  };
  auto load_keys = [&](int base, Where& p) {
    if constexpr (P8) {
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int grp = i * RI / 8, in = i * RI % 8;  // the load's group, its first row there
        const T* r = kbase + static_cast<int64_t>(p.page[grp]) * a.kps +
                     static_cast<int64_t>(p.off[grp] + in) * a.kts;
        const int o = krow * static_cast<int>(a.kts) + kdim;
        kr[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(r + o));
      }
    } else {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const T* r = row_of(base + i * RI + krow, kbase, a.kps, a.kts, &bad);
        kr[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(r + kdim));
      }
      p.bad = __any(bad);
    }
    if (!D_FULL && kchunk * 8 >= D) {
#pragma unroll
      for (int i = 0; i < KI; ++i) kr[i] = v4u32_t(0u);
    }
  };
  auto load_values = [&](int base, const Where& p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (P8) {
        const T* r = vbase + static_cast<int64_t>(p.page[j / 2]) * a.vps +
                     static_cast<int64_t>(p.off[j / 2] + 4 * (j % 2)) * a.vts;
        load_value(j, r + g * static_cast<int>(a.vts));
      } else {
        bool bad = false;
        load_value(j, row_of(base + 4 * j + g, vbase, a.vps, a.vts, &bad));
      }
    }
  };

  uint8_t* keys = lds + wave * kWaveBytes;  // the wave's key tile
  auto key_at = [&](int t, int q) {         // chunk q of its row t
    const int x = DT == 64 ? (t >> 1) & 7 : t & 15;
    return reinterpret_cast<v4u32_t*>(keys + t * (DT * 2) + ((q ^ x) << 4));
  };

  float m = -__builtin_huge_valf(), l = 0.0f;
  v4f32 acc[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] = v4f32(0.0f);
  const float scale2 = a.scale * kLog2e;

  Where here, next;
  auto step = [&](int base, auto more) {
    constexpr bool MORE = decltype(more)::value;
    const int after = base + kUnit;
    const bool poisoned = here.bad;
#pragma unroll
    for (int i = 0; i < KI; ++i)
      *key_at(i * RI + krow, kchunk) = kr[i];
    if constexpr (MORE) {
      check(next);
      load_keys(after, next);
    }
    // Other lanes' keys: the wave's LDS operations are in order, and stay so.
    asm volatile("" ::: "memory");
    // S^T: row 4g + i of product u is token 16u + 4i + g.
    v4f32 d[2] = {v4f32(0.0f), v4f32(0.0f)};
#pragma unroll
    for (int k = 0; k < KK; ++k) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const v4u32_t x = *key_at(16 * u + 4 * (c & 3) + (c >> 2), 4 * k + g);
        d[u] = F::mfma(__builtin_bit_cast(V8, x), qf[k], d[u]);
      }
    }
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = d[j / 4][j % 4] * scale2;
    asm volatile("" ::: "memory");
    if (poisoned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = __builtin_nanf("");
    }
    if (base < lo || base + kTile > n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = base + 4 * j + g;
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
    V8 p, rest;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = __builtin_amdgcn_exp2f(s[j] - ref);
      l += e;
      p[j] = fromf<T>(e);
      rest[j] = fromf<T>(e - tof(p[j]));
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
      acc[e] = F::mfma(__builtin_bit_cast(V8, col), rest, acc[e]);
    }
    if constexpr (MORE) {
      load_values(after, next);
      here = next;
      next = locate(after + kUnit);
    }
  };
  int base = w.begin + wave * kTile;
  if (base < w.end) {
    here = locate(base);
    check(here);
    load_keys(base, here);
    load_values(base, here);
    next = locate(base + kUnit);
    for (; base + kUnit < w.end; base += kUnit) step(base, std::true_type{});
    step(base, std::false_type{});
  }

  // Joins the waves: outputs [wave][head][dim] with their maximum and sum.
  l += shfl_xor(l, 16);
  l += shfl_xor(l, 32);
  if (g == 0) sm[wave][c] = m, sl[wave][c] = l;
  auto out_at = [&](int v, int h, int d) {
    return reinterpret_cast<float*>(lds + v * kWaveBytes) + h * PITCH + d;
  };
  // acc[e][i] is dim VC (4g + i) + e of head c (of each 128 dims).
#pragma unroll
  for (int e = 0; e < VE; e += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f32 x;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = acc[e + y][i];
      *reinterpret_cast<v4f32*>(out_at(wave, c, (e / 8) * 128 + VC * (4 * g + i) + e % 8)) = x;
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
  const uint32_t slot0 = w.slot * a.heads + head * static_cast<uint32_t>(w.pieces);
  auto part_at = [&](int s, int word) {
    return ((slot0 + static_cast<uint32_t>(s)) * static_cast<uint32_t>(slot_floats) +
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
      const v4f32 y = *reinterpret_cast<const v4f32*>(out_at(v, h, 4 * d));
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
  // NG groups of threads take consecutive shares of the pieces, sixteen loads in flight
  // each, and are joined through LDS.
  constexpr int kThreads = kWaves * 64;
  int NG = 1;
  while (2 * NG * items <= kThreads && 2 * NG <= w.pieces) NG *= 2;
  const int width = min(items, kThreads);
  const int grp = static_cast<int>(threadIdx.x) / width;
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
  Joined* shared = reinterpret_cast<Joined*>(lds);
  static_assert(sizeof(Joined) == 32 && sizeof(lds) >= kThreads * sizeof(Joined), "LDS of a join");
  for (int x = static_cast<int>(threadIdx.x) % width; x < items && grp < NG; x += kThreads) {
    const int h = x / d4, d = x - h * d4;
    Joined j{v4f32(0.0f), -__builtin_huge_valf(), 0.0f};
    for (int s = s_begin; s < s_end; s += 16) {
      v4u32_t o[16];
      u32x2 ml[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int si = min(s + i, s_end - 1);
        o[i] = __builtin_amdgcn_raw_buffer_load_b128(
            parts, part_at(si, 2 * a.slot_rows + h * a.dim + 4 * d), 0, kSc1);
        ml[i] = __builtin_amdgcn_raw_buffer_load_b64(parts, part_at(si, 2 * h), 0, kSc1);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
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
hxm_status launch_attention(const AttnArgs& a, hipStream_t stream) {
  const int64_t groups = attn_grid(a.batch, a.heads, a.capacity);
  hxm_status st = check_grid("paged attention", groups, kWaves * 64);
  if (st != HXM_OK) return st;
  const unsigned n = static_cast<unsigned>(groups);
  const bool full = a.dim == DT;
  const bool p8 = a.page_size % 8 == 0 && std::max(a.kts, a.vts) <= (int64_t(1) << 24);
  if (full && p8) paged_attention_kernel<T, DT, true, true><<<n, kWaves * 64, 0, stream>>>(a);
  else if (full) paged_attention_kernel<T, DT, true, false><<<n, kWaves * 64, 0, stream>>>(a);
  else if (p8) paged_attention_kernel<T, DT, false, true><<<n, kWaves * 64, 0, stream>>>(a);
  else paged_attention_kernel<T, DT, false, false><<<n, kWaves * 64, 0, stream>>>(a);
  return check_launch("paged attention");
}

template <typename T>
hxm_status launch_attention_dim(const AttnArgs& a, hipStream_t stream) {
  if (a.dim <= 64) return launch_attention<T, 64>(a, stream);
  if (a.dim <= 128) return launch_attention<T, 128>(a, stream);
  return launch_attention<T, 256>(a, stream);
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
  // 2^24 sequences times heads keep every count of pieces in 32 bits.  A launch holds one
  // workgroup fewer, the pieces of sequences that are cut among them (attn_grid).
  constexpr int64_t kMaxBatchHeads = int64_t(1) << 24;
  constexpr int64_t kMaxGroups = 0xffffffffLL / (kWaves * 64);
  if (q_heads > 65535 || batch > kMaxBatchHeads || batch * q_heads > kMaxBatchHeads ||
      batch * cache->heads * ceil_div(q_heads / cache->heads, kHeads) >
          kMaxGroups - (batch > kAttnCutBatch ? 0 : kAttnFine * kAttnGroups))
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
  a.ld_table = ld_table;
  a.capacity = std::min(table_pages * cache->page_size, kAttnMaxTokens);
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
  // Partial results of the sequences cut in pieces, and a counter for each
  // sequence and head, zero between launches.
  a.slot_rows = std::min(a.group, kHeads);
  const int64_t parts = int64_t(2 * kAttnFine * kAttnGroups) * a.slot_rows * (a.dim + 2) * 4;
  const int64_t counts = batch * a.heads * 4;
  void* ws = nullptr;
  hipStream_t s = as_stream(stream);
  if ((st = stream_workspace(s, static_cast<size_t>(counts), &ws, kWsCount)) != HXM_OK) return st;
  a.counts = static_cast<uint32_t*>(ws);
  if ((st = stream_workspace(s, static_cast<size_t>(parts), &ws, kWsLayer)) != HXM_OK) return st;
  a.parts = static_cast<float*>(ws);
  a.parts_bytes = static_cast<int>(parts);
  return dtype == HXM_F16 ? launch_attention_dim<_Float16>(a, s)
                          : launch_attention_dim<__bf16>(a, s);
}
