// Attention of a tree of drafted tokens per sequence over the paged key-value cache.
//
// The rows that share a key head, nodes x group of them, are the 32-wide side of the
// MFMAs, so that one read of the keys and values serves up to 128 rows: 4 * dim bytes a
// token against 4 * dim * rows operations.  Few rows are bound by memory, many by the matrix
// cores and the exponentials beside them: 4 sequences to 32768 tokens, 64 nodes, 8 x 4 heads of
// 128, 109 GFLOP in 202 to 207 us (538 TFLOP/s at 203; with the second half of the
// probabilities, below, 807 on the matrix cores, 44% of their cycles); 16 sequences to 4096, 16
// nodes, 44.5 us, 3.0 TB/s, of which the join takes 6 and a workgroup's start and end 9.  Heads
// of 256 keep one wave a SIMD, and up to 32 rows spill 47 registers: 16 x 16 to 4096, 4 x 2 heads
// 66 us, 4 x 4 (64 rows) 56; 4 x 64 to 32768, 4 x 4 heads 188.
//
// A workgroup has four waves of 32 rows.  Up to 32 rows, its waves take tokens in turn, each
// with tiles of its own; up to 64 rows two by two; more, all four share a tile of 64 tokens,
// and rows past 128 take further workgroups, eight blocks on, so that they run on the same XCD
// and read the tile from its L2 (210 MB of 424 come from beyond it at 4 x 64 x 32768).
//
// S^T = K Q^T leaves lane (h, c) = (lane / 32, lane % 32) 16 scores of row c of 32 tokens,
// of tokens 8 j + 4 h + 0 .. 3.  O^T = V^T P^T wants 8 tokens of P^T in each lane's right
// operand; taking exactly those 16 scores as two of them fixes which tokens of V^T the left
// operand has, and the transposing LDS read delivers those.  So the probabilities stay in the
// lane they are in, and a row's maximum, sum and output in one column of lanes.
//
// Keys and values come in whole rows through registers into LDS, the next tile's on their way
// while this one is multiplied.  Row t of keys has its 16-byte chunk q at q ^ t % 16 (of 8
// chunks q ^ t / 2 % 8), row t of values its 64-byte chunk e at e ^ t % 4 (of 2: e ^ t / 2 %
// 2): no read or write meets a bank twice.
//
// A tile that some row does not see the whole of (drafted tokens, the window's edge, the ends)
// takes a mask of 32 bits a row.  Values there that are no numbers would pass into every row
// (0 * NaN), so they go into LDS as zeros and join those rows that see them at the very end;
// inside the loop that branch cost every tile its registers (4 x 64 over 32768: 677 us spilled,
// 361 without).
//
// The running maximum moves only when a score passes it by more than 2^8, and the
// probabilities enter the second product as two 16-bit halves, each rounded (22 bits in f16, 16
// in bf16; the first cut off instead leaves one fewer in the same time, 203 us at 4 x 64 over
// 32768), both as in the attention of one token.  One half alone took 170 us there and added as
// much to the error as the output's own rounding; elsewhere its time does not show.
#include <algorithm>
#include <type_traits>

#include "attention_cut.h"
#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;  // of the running maximum, in powers of two
constexpr int kMaxNodes = 64;
constexpr int kWaves = 4;

struct TreeArgs {
  const void* q;
  void* out;
  const void* kc;
  const void* vc;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* parents;
  float* lse;
  int64_t q_ts, q_hs, o_ts, o_hs;
  int64_t kps, khs, kts, vps, vhs, vts;
  int64_t ld_table, capacity;  // tokens a table row holds
  int64_t span;                // and those of them that a sequence can have read
  int2* cuts;  // [batch]: pieces of a sequence and the partial slots before them
  float* parts;
  uint32_t pages, page_size;
  FastDiv page_div;
  int batch, nodes, hkv, group, tiles, heads, dim;  // heads: hkv * tiles
  int window;  // tokens that some node of a sequence sees (the last ones, 0: all)
  int reach;   // and that one node sees
  float scale;
  bool whole;  // no sequence is cut
};

typedef float v8f32 __attribute__((ext_vector_type(8)));

template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef v8f16 V;
  static constexpr float kShift = 7.0f;
  static constexpr uint32_t kNan = 0x7e007e00u, kExp = 0x7c00u;
  static __device__ __forceinline__ v16f32 mfma(V a, V b, v16f32 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // x rounded; x keeps what that leaves.
  static __device__ __forceinline__ V split(v8f32& x) {
    const V r = __builtin_convertvector(x, V);
    x -= __builtin_convertvector(r, v8f32);
    return r;
  }
};
template <>
struct Frag<__bf16> {
  typedef v8bf16 V;
  static constexpr float kShift = 0.0f;
  static constexpr uint32_t kNan = 0x7fc07fc0u, kExp = 0x7f80u;
  static __device__ __forceinline__ v16f32 mfma(V a, V b, v16f32 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V split(v8f32& x) {
    const V r = __builtin_convertvector(x, V);
    const v4u32_t b = __builtin_bit_cast(v4u32_t, r);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      x[i] -= __builtin_bit_cast(float, b[i / 2] << 16);
      x[i + 1] -= __builtin_bit_cast(float, b[i / 2] & 0xffff0000u);
    }
    return r;
  }
};

typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short v4i16 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float shfl_xor(float v, int m) { return __shfl_xor(v, m, 64); }
__device__ __forceinline__ float finite(float M) { return M == -__builtin_huge_valf() ? 0.0f : M; }

// What node `lane` of sequence b sees of the drafted tokens, and where it stands.
struct Node {
  uint64_t sees;  // drafted tokens, a bit each
  int first;      // first token of the context that it sees, ctx and more: none
  bool bad;       // of a parent that is none
};
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(v), lane, 64);
  const uint32_t hi = __shfl(static_cast<uint32_t>(v >> 32), lane, 64);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ Node node_of(const TreeArgs& a, int b, int ctx, int lane) {
  Node r;
  int p = lane - 1;
  if (a.parents) p = lane < a.nodes ? a.parents[static_cast<int64_t>(b) * a.nodes + lane] : -2;
  const bool pad = p < -1;
  const uint64_t pads = __ballot(pad), wrong = __ballot(p >= lane);
  if (p >= lane) p = -1;
  // Ancestors by doubling: those up to 2 k - 1 above.
  uint64_t up = uint64_t(1) << lane;
  int to = p;
  for (int k = 1; k < a.nodes; k *= 2) {
    const int at = max(to, 0);
    const uint64_t more = shfl64(up, at);
    const int next = __shfl(to, at, 64);
    if (to >= 0) up |= more, to = next;
  }
  r.bad = !pad && (up & (pads | wrong)) != 0;
  const int depth = __builtin_popcountll(up) - 1;
  r.first = 0;
  r.sees = up;
  if (a.reach > 0) {
    r.first = max(0, ctx + depth - a.reach + 1);
    if (a.reach < a.nodes) {  // the nearest ancestors only
      uint64_t near = 0;
      int at = lane;
      for (int k = 0; k < a.reach; ++k) {
        if (at >= 0) near |= uint64_t(1) << at;
        const int next = __shfl(p, max(at, 0), 64);
        at = at >= 0 ? next : -1;
      }
      r.sees = near;
    }
  }
  if (pad) r.sees = 0, r.first = INT32_MAX;
  return r;
}

constexpr int tree_waves(int dt) { return dt <= 128 ? 2 : 1; }

// Pieces of a batch: as many as run at once, two workgroups a CU where registers and LDS hold
// them (one a CU: 4 x 64 over 32768 361 us for 242, 16 x 16 over 4096 72 for 51).
constexpr uint32_t tree_groups(int dt) { return (dt <= 128 ? 2 : 1) * kAttnGroups; }

// WR of the four waves side by side over the rows, 32 each, the others over tokens.
template <typename T, int DT, int WR, bool P>
__global__ __launch_bounds__(kWaves * 64)
    __attribute__((amdgpu_waves_per_eu(tree_waves(DT)))) void tree_attention_kernel(TreeArgs a) {
  using F = Frag<T>;
  using V8 = typename F::V;
  constexpr int WT = kWaves / WR;
  constexpr int TK = WR == 4 ? 64 : 32;  // tokens of a tile
  constexpr int NB = WR == 1 ? 1 : 2;    // buffers
  constexpr int CK = DT / 8;             // 16-byte chunks of a row
  constexpr int GT = WR * 64;            // threads that share a tile
  constexpr int RP = GT / CK;            // rows of a load
  constexpr int NP = TK / RP;            // loads of a tile's keys
  constexpr int TB = TK / 32;
  constexpr int KS = DT / 16, DB = DT / 32;
  constexpr int PITCH = DT + 4;          // floats of a row of the join
  constexpr int kTileBytes = TK * DT * 2;
  constexpr int kLoopBytes = WT * NB * 2 * kTileBytes, kOutBytes = kWaves * 32 * PITCH * 4;
  __shared__ __align__(16) uint8_t lds[kLoopBytes > kOutBytes ? kLoopBytes : kOutBytes];
  __shared__ float sm[kWaves][32], sl[kWaves][32];
  __shared__ uint64_t row_sees[32 * WR];
  __shared__ int row_first[32 * WR], odd;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wr = wave % WR, tg = wave / WR;
  const int gt = static_cast<int>(threadIdx.x) % GT;
  const int h = lane >> 5, c = lane & 31;

  // Eight (piece, key head) pairs run on the eight XCDs, the row tiles of one on its own.
  const uint32_t pair = blockIdx.x / (8u * a.tiles) * 8u + blockIdx.x % 8u;
  const int tile = static_cast<int>(blockIdx.x / 8u % static_cast<uint32_t>(a.tiles));
  const int hk = static_cast<int>(pair % static_cast<uint32_t>(a.hkv));
  const Piece w = find_piece<tree_groups(DT), true>(a, pair / static_cast<uint32_t>(a.hkv), lane);
  if (w.b < 0) return;
  const int D = a.dim;
  const int b = w.b, n = w.n, lo = w.lo;
  const int ctx = n - a.nodes;
  const bool broken = w.over || (n > 0 && ctx < 0);
  const int total = a.nodes * a.group;
  const int row0 = tile * 32 * WR + wr * 32;  // of this wave
  const int row = row0 + c;
  const bool live = row < total;
  const int node = live ? row / a.group : 0;
  const int head = hk * a.group + (live ? row - node * a.group : 0);

  const T* kbase = static_cast<const T*>(a.kc) + hk * a.khs;
  const T* vbase = static_cast<const T*>(a.vc) + hk * a.vhs;
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
  auto page_of = [&](int tok) {
    return static_cast<uint32_t>((static_cast<uint64_t>(static_cast<uint32_t>(tok)) *
                                  a.page_div.mul) >> a.page_div.shift);
  };

  // A thread's rows of a tile are tokens RP j + gt / CK (j < NP), in chunk gt % CK.
  const int trow = gt / CK, chunk = gt % CK;
  const bool in_dim = chunk * 8 < D;
  const int dim0 = in_dim ? chunk * 8 : 0;
  // Where the rows lie.  P: a wave's rows of a load are of one page, whose number and
  // address the scalar unit works out; otherwise every thread its own.
  constexpr int RW = 64 / CK;  // rows of a wave's load
  struct Ids {
    uint32_t page[NP];
    int off[NP];  // of the first row in its page
  };
  typedef const int32_t __attribute__((address_space(4))) * ConstInts;
  const ConstInts ctable = (ConstInts)(reinterpret_cast<uintptr_t>(table));
  auto locate = [&](int base) {
    Ids r;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int t = P ? min(max(base + j * RP + wr * RW, lo & -RW), (n - 1) & -RW)
                      : min(max(base + j * RP + trow, lo), n - 1);
      // (P: page_size is 2 or more, and the shift 32 or more.)
      const uint32_t k = P ? __umulhi(static_cast<uint32_t>(t), a.page_div.mul) >>
                                 (a.page_div.shift - 32)
                           : page_of(t);
      r.page[j] = static_cast<uint32_t>(P ? ctable[k] : table[k]);
      r.off[j] = t - static_cast<int>(k * a.page_size);
    }
    return r;
  };
  const uint32_t klane = (P ? lane / CK * static_cast<uint32_t>(a.kts) : 0u) + dim0;
  const uint32_t vlane = (P ? lane / CK * static_cast<uint32_t>(a.vts) : 0u) + dim0;
  v4u32_t kr[NP], vr[NP];
  auto load = [&](const Ids& ids) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const uint32_t id = ids.page[j] < a.pages ? ids.page[j] : 0u;
      const T *k = kbase, *v = vbase;
      if constexpr (P) {
        const uint32_t off = static_cast<uint32_t>(ids.off[j]);
        k += static_cast<uint64_t>(id) * static_cast<uint32_t>(a.kps) +
             off * static_cast<uint32_t>(a.kts);
        v += static_cast<uint64_t>(id) * static_cast<uint32_t>(a.vps) +
             off * static_cast<uint32_t>(a.vts);
      } else {
        k += id * a.kps + ids.off[j] * a.kts;
        v += id * a.vps + ids.off[j] * a.vts;
      }
      kr[j] = *reinterpret_cast<const any4*>(k + klane);
      vr[j] = *reinterpret_cast<const any4*>(v + vlane);
    }
  };
  // The first tile on its way before anything else.
  constexpr int STEP = WT * TK;
  const bool any_tokens = !broken && w.begin < w.end;
  int base = w.begin + tg * TK;
  Ids ids{}, next{};
  if (any_tokens) {
    ids = locate(base);
    load(ids);
    next = locate(base + STEP);
  }

  // Q^T: dims 16k + 8h .. of row c, zeros past the last row and past D.  A negative scale
  // is Q's sign.
  V8 qf[KS];
  {
    const T* q = static_cast<const T*>(a.q) +
                 (static_cast<int64_t>(b) * a.nodes + node) * a.q_ts + head * a.q_hs;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = k * 16 + h * 8;
      const v4u32_t x = *reinterpret_cast<const any4*>(q + (d < D ? d : 0));
      qf[k] = __builtin_bit_cast(V8, live && d < D ? x ^ flip : v4u32_t(0u));
    }
  }

  const Node mine = node_of(a, b, ctx, lane);
  const uint64_t sees = shfl64(mine.sees, node);
  const int first = __shfl(mine.first, node, 64);
  const bool bad = __shfl(static_cast<int>(mine.bad), node, 64) != 0;

  auto vswz = [](int t) { return DT == 64 ? (t >> 1) & 1 : t & 3; };
  auto kswz = [](int t) { return DT == 64 ? (t >> 1) & 7 : t & 15; };
  auto buffer = [&](int i) { return lds + (tg * NB + i % NB) * (2 * kTileBytes); };
  // A tile that some row does not see the whole of.
  auto at_edge = [&](int base) {
    return base + TK > ctx || base < lo || (a.reach > 0 && base < n - a.reach);
  };
  // Into LDS: keys of a page that is none as NaN, values of tokens outside [lo, n) as zeros
  // (0 * V must be 0 for what lies in the cache there), and so at an edge those that are no
  // numbers, which join at the end (`odd`).
  auto store = [&](int base, const Ids& ids, int i) {
    uint8_t* to = buffer(i);
    bool bad_page = false;
#pragma unroll
    for (int j = 0; j < NP; ++j) bad_page |= ids.page[j] >= a.pages;
    if (at_edge(base) || (P ? bad_page : __any(bad_page))) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int t = base + j * RP + trow;
        const bool good = ids.page[j] < a.pages, in = t >= lo && t < n && good;
        if (!good) kr[j] = v4u32_t(F::kNan);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t x = in ? vr[j][y] : 0u;
          const uint32_t bad = ((x & F::kExp) == F::kExp ? 0xffffu : 0u) |
                               ((x & (F::kExp << 16)) == (F::kExp << 16) ? 0xffff0000u : 0u);
          any |= bad != 0;
          vr[j][y] = x & ~bad;
        }
      }
      if (any && in_dim) odd = 1;
    }
    if (D < DT) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        kr[j] = in_dim ? kr[j] : v4u32_t(0u);
        vr[j] = in_dim ? vr[j] : v4u32_t(0u);
      }
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int r = j * RP + trow;
      *reinterpret_cast<v4u32_t*>(to + r * (DT * 2) + ((chunk ^ kswz(r)) << 4)) = kr[j];
      *reinterpret_cast<v4u32_t*>(to + kTileBytes + r * (DT * 2) +
                                  ((((chunk >> 2) ^ vswz(r)) << 6) | ((chunk & 3) << 4))) = vr[j];
    }
  };

  float m = -__builtin_huge_valf(), l = 0.0f;
  v16f32 acc[DB];
#pragma unroll
  for (int e = 0; e < DB; ++e) acc[e] = v16f32(0.0f);
  const float scale2 = fabsf(a.scale) * kLog2e;

  auto compute = [&](int base, const uint8_t* from) {
    const bool edge = at_edge(base);
    const uint8_t* keys = from;
    const uint8_t* values = from + kTileBytes;
    // S^T: register i of lane (h, c) is row c's score of token 8 (i / 4) + 4 h + i % 4.
    v16f32 s[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) s[t] = v16f32(0.0f);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        const v4u32_t x = *reinterpret_cast<const v4u32_t*>(
            keys + (32 * t + c) * (DT * 2) + (((2 * k + h) ^ kswz(c)) << 4));
        s[t] = F::mfma(__builtin_bit_cast(V8, x), qf[k], s[t]);
      }
    float by = scale2;
    if (edge) {
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        const int at = base + 32 * t, from_ctx = at - ctx;
        auto ones = [](int k) {  // the first k bits
          return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
        };
        const uint32_t drafted =
            from_ctx >= 0 ? (from_ctx < 64 ? static_cast<uint32_t>(sees >> from_ctx) : 0u)
                          : (from_ctx > -32 ? static_cast<uint32_t>(sees) << -from_ctx : 0u);
        // (first is INT32_MAX for padding; at - first then stays in range.)
        const uint32_t seen = (ones(-from_ctx) & ~ones(first - at)) | drafted;  // a bit a token
        const uint32_t mine = seen >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[t][i] = (mine >> (8 * (i / 4) + i % 4)) & 1 ? s[t][i] * scale2 : -__builtin_huge_valf();
      }
      by = 1.0f;
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < TB; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    top *= by;
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, shfl_xor(top, 32));
      const float mn = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(m - finite(mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[e] *= alpha;
    }
    const float ref = finite(m) - F::kShift;
    // O^T: dims 32 e of the 16 tokens of step t, transposed on the way out of LDS: four
    // tokens of 16 dims for each 16 lanes.
    const int v16 = lane & 15, vdim = 16 * ((lane >> 4) & 1) + 4 * (v16 & 3);
    const int vtok = 4 * h + (v16 >> 2);
    V8 p[2], rest[2], vt[2][DB];
    auto weights = [&](int t) {  // of step t's tokens
      v8f32 x;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(s[t / 2][8 * (t % 2) + i], by, -ref));
        l += x[i];
      }
      p[t % 2] = F::split(x);
      rest[t % 2] = __builtin_convertvector(x, V8);
    };
    auto read_values = [&](int t) {
#pragma unroll
      for (int e = 0; e < DB; ++e) {
        v4u32_t x;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = 16 * t + 8 * y + vtok;
          const uint8_t* at = values + r * (DT * 2) + ((e ^ vswz(vtok)) << 6) + vdim * 2;
          const u32x2 z = __builtin_bit_cast(
              u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                         (__attribute__((address_space(3))) v4i16*)(at)));
          x[2 * y] = z[0], x[2 * y + 1] = z[1];
        }
        vt[t % 2][e] = __builtin_bit_cast(V8, x);
      }
    };
    // The next step's weights are made and its values read under this one's products (both
    // halves of one dim apart: the second waits for the first).
    read_values(0);
    weights(0);
#pragma unroll
    for (int t = 0; t < 2 * TB; ++t) {
      if (t + 1 < 2 * TB) read_values(t + 1), weights(t + 1);
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[e] = F::mfma(vt[t % 2][e], p[t % 2], acc[e]);
#pragma unroll
      for (int e = 0; e < DB; ++e) acc[e] = F::mfma(vt[t % 2][e], rest[t % 2], acc[e]);
    }
  };

  if (threadIdx.x == 0) odd = 0;
  __syncthreads();
  if (any_tokens) {
    const int count = (w.end - w.begin + STEP - 1) / STEP;
    store(base, ids, 0);
    if (NB > 1) __syncthreads();
    for (int i = 0; i < count; ++i, base += STEP) {
      if (NB == 1) asm volatile("" ::: "memory");
      const bool more = i + 1 < count;
      if (more) {
        ids = next;
        load(ids);
        next = locate(base + 2 * STEP);
      }
      if (base < w.end) compute(base, buffer(i));
      if (NB == 1) asm volatile("" ::: "memory");
      if (more) store(base + STEP, ids, i + 1);
      if (NB > 1) __syncthreads();
    }
  }
  __syncthreads();

  // Joins the waves that share rows: outputs [wave][row][dim] with their maximum and sum.
  l += shfl_xor(l, 32);
  // (A sequence without tokens sees nothing whatever its parents, nor does padding.  Asking
  // for it behind the NaN took 0.6 us more of 17 with windows.)
  if (broken || (bad && n > 0)) l = __builtin_nanf("");
  if (first == INT32_MAX) m = -__builtin_huge_valf(), l = 0.0f;
  if (h == 0) sm[wave][c] = m, sl[wave][c] = l;
  if (h == 0 && tg == 0) row_sees[32 * wr + c] = sees, row_first[32 * wr + c] = first;
  auto out_at = [&](int v, int r, int d) {
    return reinterpret_cast<float*>(lds) + (v * 32 + r) * PITCH + d;
  };
#pragma unroll
  for (int e = 0; e < DB; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f32 x;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = acc[e][4 * i + y];
      *reinterpret_cast<v4f32*>(out_at(wave, c, 32 * e + 8 * i + 4 * h)) = x;
    }
  __syncthreads();

  if (!a.whole && w.index == 0 && hk == 0 && tile == 0 && threadIdx.x == 0)
    a.cuts[b] = make_int2(w.pieces, static_cast<int>(w.slot));
  const int tile0 = tile * 32 * WR, rows = min(32 * WR, total - tile0);
  const int d4 = D / 4, items = rows * d4;
  const int64_t slot_floats = static_cast<int64_t>(32 * WR) * (D + 2);
  float* part = a.parts + ((static_cast<int64_t>(w.slot) * a.heads +
                            (hk * a.tiles + tile) * static_cast<int64_t>(w.pieces)) + w.index) *
                              slot_floats;
  // The values that are no numbers in the tiles at an edge, of the tokens that row r sees:
  // their weights are above zero, whatever they are.
  auto stray = [&](int r, int d) {
    v4f32 x = v4f32(0.0f);
    for (int base = w.begin; base < w.end; base += TK) {
      if (!at_edge(base)) continue;
      for (int t = max(base, lo); t < min(base + TK, w.end); ++t) {
        const bool seen =
            t < ctx ? t >= row_first[r] : ((row_sees[r] >> (t - ctx)) & 1) != 0;
        const uint32_t id = static_cast<uint32_t>(table[page_of(t)]);
        if (!seen || id >= a.pages) continue;
        const T* v = vbase + id * a.vps +
                     static_cast<int64_t>(t - static_cast<int>(page_of(t) * a.page_size)) * a.vts;
        for (int e = 0; e < 4; ++e)
          if ((__builtin_bit_cast(uint16_t, v[4 * d + e]) & F::kExp) == F::kExp)
            x[e] += tof(v[4 * d + e]);
      }
    }
    return x;
  };
  for (int x = threadIdx.x; x < items; x += kWaves * 64) {
    const int r = x / d4, d = x - r * d4, wv = r >> 5, rr = r & 31;
    float M = sm[wv][rr];
#pragma unroll
    for (int v = 1; v < WT; ++v) M = fmaxf(M, sm[wv + v * WR][rr]);
    v4f32 o = v4f32(0.0f);
    float L = 0.0f;
#pragma unroll
    for (int v = 0; v < WT; ++v) {
      const float f = __builtin_amdgcn_exp2f(sm[wv + v * WR][rr] - finite(M));
      const v4f32 y = *reinterpret_cast<const v4f32*>(out_at(wv + v * WR, rr, 4 * d));
      L = fmaf(f, sl[wv + v * WR][rr], L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, y[e], o[e]);
    }
    if (odd) o += stray(r, d);
    if (w.pieces == 1) {
      const int nd = (tile0 + r) / a.group, hd = hk * a.group + (tile0 + r - nd * a.group);
      const int64_t tok = static_cast<int64_t>(b) * a.nodes + nd;
      T* out = static_cast<T*>(a.out) + tok * a.o_ts + hd * a.o_hs + 4 * d;
      const float inv = 1.0f / L;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = fromf<T>(L == 0.0f ? 0.0f : o[e] * inv);
      if (d == 0 && a.lse)
        a.lse[tok * a.hkv * a.group + hd] =
            L == 0.0f ? -__builtin_huge_valf()
                      : (M + (__builtin_amdgcn_logf(L) - F::kShift)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<v4f32*>(part + 2 * (32 * WR) + r * D + 4 * d) = o;
      if (d == 0) part[2 * r] = M, part[2 * r + 1] = L;
    }
  }
}

// Joins the pieces of the sequences that were cut, in their order: a thread a row's four
// dims.  How a sequence was cut its first workgroup has written down (worked out again from the
// lengths, 16 x 16 over 4096 took 45.9 us for 44.7).
template <typename T>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int tile_rows, int slices) {
  const uint32_t x = blockIdx.x / static_cast<uint32_t>(slices);
  const int slice = static_cast<int>(blockIdx.x % static_cast<uint32_t>(slices));
  const int b = static_cast<int>(x / static_cast<uint32_t>(a.heads));
  const int ht = static_cast<int>(x % static_cast<uint32_t>(a.heads));
  const int pieces = a.cuts[b].x, slot = a.cuts[b].y;
  if (pieces < 2) return;
  const int D = a.dim, d4 = D / 4, per = 256 / d4;
  const int hk = ht / a.tiles, tile = ht % a.tiles;
  const int r = slice * per + static_cast<int>(threadIdx.x) / d4;
  const int d = static_cast<int>(threadIdx.x) % d4;
  const int total = a.nodes * a.group;
  if (static_cast<int>(threadIdx.x) >= per * d4 || r >= tile_rows || tile * tile_rows + r >= total)
    return;
  const int64_t slot_floats = static_cast<int64_t>(tile_rows) * (D + 2);
  const float* part =
      a.parts + (static_cast<int64_t>(slot) * a.heads + ht * static_cast<int64_t>(pieces)) *
                    slot_floats;
  float M = -__builtin_huge_valf(), L = 0.0f;
  v4f32 o = v4f32(0.0f);
  for (int s = 0; s < pieces; s += 8) {
    v4f32 y[8];
    float mm[8], ll[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* at = part + min(s + i, pieces - 1) * slot_floats;
      mm[i] = at[2 * r], ll[i] = at[2 * r + 1];
      y[i] = *reinterpret_cast<const v4f32*>(at + 2 * tile_rows + r * D + 4 * d);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s + i >= pieces) break;
      const float mn = fmaxf(M, mm[i]);
      const float fa = __builtin_amdgcn_exp2f(M - finite(mn));
      const float fb = __builtin_amdgcn_exp2f(mm[i] - finite(mn));
      M = mn;
      L = fmaf(fb, ll[i], fa * L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(fb, y[i][e], fa * o[e]);
    }
  }
  const int row = tile * tile_rows + r;
  const int nd = row / a.group, hd = hk * a.group + (row - nd * a.group);
  const int64_t tok = static_cast<int64_t>(b) * a.nodes + nd;
  T* out = static_cast<T*>(a.out) + tok * a.o_ts + hd * a.o_hs + 4 * d;
  const float inv = 1.0f / L;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = fromf<T>(L == 0.0f ? 0.0f : o[e] * inv);
  if (d == 0 && a.lse)
    a.lse[tok * a.hkv * a.group + hd] =
        L == 0.0f
            ? -__builtin_huge_valf()
            : (M + (__builtin_amdgcn_logf(L) - Frag<T>::kShift)) * 0.6931471805599453f;
}

int tile_rows(int64_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

template <typename T, int DT>
hxm_status launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int rows = tile_rows(int64_t(a.nodes) * a.group);
  const int64_t pairs =
      a.whole ? int64_t(a.batch) * a.hkv
              : ceil_div(attn_step_grid(a.batch, a.heads, a.span, tree_groups(DT)), a.tiles);
  const int64_t groups = ceil_div(pairs, 8) * 8 * a.tiles;
  const int per = 256 / (a.dim / 4), slices = static_cast<int>(ceil_div(rows, per));
  const int64_t joins = a.whole ? 0 : int64_t(a.batch) * a.heads * slices;
  hxm_status st = check_grid("tree attention", std::max(groups, joins), 256);
  if (st != HXM_OK) return st;
  const unsigned n = static_cast<unsigned>(groups);
  // A wave loads 512 / DT rows at a time; a page and its stride within 32 bits.
  const bool paged = a.page_size % (512 / DT) == 0 &&
                     std::max(a.kts, a.vts) <= (int64_t(1) << 30) / a.page_size &&
                     std::max(a.kps, a.vps) <= UINT32_MAX;
  auto launch = [&](auto wr) {
    constexpr int WR = decltype(wr)::value;
    if (paged) tree_attention_kernel<T, DT, WR, true><<<n, 256, 0, stream>>>(a);
    else tree_attention_kernel<T, DT, WR, false><<<n, 256, 0, stream>>>(a);
  };
  if (rows == 32) launch(std::integral_constant<int, 1>{});
  else if (rows == 64) launch(std::integral_constant<int, 2>{});
  else launch(std::integral_constant<int, 4>{});
  if ((st = check_launch("tree attention")) != HXM_OK) return st;
  if (a.whole) return ok();
  tree_join_kernel<T><<<static_cast<unsigned>(joins), 256, 0, stream>>>(a, rows, slices);
  return check_launch("tree attention join");
}

template <typename T>
hxm_status launch_tree_dim(const TreeArgs& a, hipStream_t stream) {
  if (a.dim <= 64) return launch_tree<T, 64>(a, stream);
  if (a.dim <= 128) return launch_tree<T, 128>(a, stream);
  return launch_tree<T, 256>(a, stream);
}

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_tree_attention(const hxm_heads* q, const hxm_heads* out, int64_t q_heads,
                                         const hxm_kv_cache* cache, const int32_t* block_table,
                                         int64_t ld_table, int64_t table_pages,
                                         const int32_t* seq_lens, const int32_t* parents,
                                         int64_t batch, int64_t nodes, float scale, int64_t window,
                                         float* lse, int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE,
                "unsupported-dtype: tree_attention takes f16 or bf16 (got %d)", dtype);
  hxm_status st = check_kv_cache("tree_attention", cache, false);
  if (st != HXM_OK) return st;
  if (batch < 0 || nodes < 1 || q_heads < 1 || q_heads % cache->heads != 0 || window < 0)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: tree_attention batch=%lld, nodes=%lld, %lld query heads over "
                "%lld, window=%lld",
                (long long)batch, (long long)nodes, (long long)q_heads, (long long)cache->heads,
                (long long)window);
  // 2^18 sequences times heads times tiles of rows: neither launch then holds more than 2^23
  // workgroups of 256.
  constexpr int64_t kMaxHeads = int64_t(1) << 18;
  const int64_t of_head = std::min(nodes, int64_t(kMaxNodes)) * (q_heads / cache->heads);
  if (nodes > kMaxNodes || q_heads > 65535 || batch > kMaxHeads ||
      batch * cache->heads * ceil_div(of_head, tile_rows(of_head)) > kMaxHeads)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: tree_attention batch=%lld, nodes=%lld, %lld heads",
                (long long)batch, (long long)nodes, (long long)q_heads);
  const int64_t tokens = batch * nodes;
  if ((st = check_heads("tree_attention", "q", q, tokens, q_heads, cache->dim, false)) != HXM_OK ||
      (st = check_heads("tree_attention", "out", out, tokens, q_heads, cache->dim, true)) != HXM_OK)
    return st;
  if (batch > 0 && !heads_apart(out, q_heads, q, q_heads, tokens, cache->dim))
    return fail(HXM_INVALID_ARG, "invalid-argument: tree_attention out overlaps q");
  if (table_pages < 0 || table_pages > INT32_MAX || !stride_ok(ld_table) ||
      (batch > 1 && ld_table < table_pages) ||
      (batch > 0 && (!seq_lens || (table_pages > 0 && !block_table))))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: tree_attention table of %lld pages, ld %lld, or null lengths",
                (long long)table_pages, (long long)ld_table);
  if (!(scale == scale))
    return fail(HXM_INVALID_ARG, "invalid-argument: tree_attention scale is NaN");
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (batch == 0) return ok();
  TreeArgs a{};
  a.q = q->data, a.q_ts = q->token_stride, a.q_hs = q->head_stride;
  a.out = out->data, a.o_ts = out->token_stride, a.o_hs = out->head_stride;
  a.kc = cache->k, a.vc = cache->v;
  a.kps = cache->k_page_stride, a.khs = cache->k_head_stride, a.kts = cache->k_token_stride;
  a.vps = cache->v_page_stride, a.vhs = cache->v_head_stride, a.vts = cache->v_token_stride;
  a.table = block_table, a.lens = seq_lens, a.parents = parents, a.lse = lse;
  a.ld_table = ld_table;
  a.capacity = std::min(table_pages * cache->page_size, kAttnMaxTokens);
  a.pages = static_cast<uint32_t>(cache->pages);
  a.page_size = static_cast<uint32_t>(cache->page_size);
  a.page_div = fast_div(a.page_size);
  a.batch = static_cast<int>(batch);
  a.nodes = static_cast<int>(nodes);
  a.hkv = static_cast<int>(cache->heads);
  a.group = static_cast<int>(q_heads / cache->heads);
  const int rows = tile_rows(nodes * a.group);
  a.tiles = static_cast<int>(ceil_div(nodes * a.group, rows));
  a.heads = a.hkv * a.tiles;
  a.dim = static_cast<int>(cache->dim);
  a.reach = window >= kAttnMaxTokens ? 0 : static_cast<int>(window);
  a.window = a.reach > 0 ? a.reach + a.nodes - 1 : 0;
  a.scale = scale;
  // How the sequences were cut, and the partial results of those in pieces.
  hipStream_t s = as_stream(stream);
  // Sequences of up to kAttnWhole units are one piece each.
  a.span = attn_span(a.capacity, a.window);
  a.whole = batch > kAttnCutBatch || a.span <= kAttnWhole * kAttnUnit;
  if (!a.whole) {
    const int64_t slots = attn_step_slots(batch, a.heads, a.span, tree_groups(a.dim));
    void* ws = nullptr;
    const int64_t cuts = ceil_div(batch * static_cast<int64_t>(sizeof(int2)), 256) * 256;
    st = stream_workspace(s, static_cast<size_t>(cuts + slots * rows * (a.dim + 2) * 4), &ws,
                          kWsLayer);
    if (st != HXM_OK) return st;
    a.cuts = static_cast<int2*>(ws);
    a.parts = reinterpret_cast<float*>(static_cast<char*>(ws) + cuts);
  }
  return dtype == HXM_F16 ? launch_tree_dim<_Float16>(a, s) : launch_tree_dim<__bf16>(a, s);
}
