// How the attention kernels over a paged cache cut a batch into pieces, one for a
// workgroup, on the device (the arithmetic is host_logic.h's).  Args has batch, heads
// (workgroups that read a piece), lens, capacity (tokens a table row holds) and window
// (of the last tokens, 0: all); with STEPS whole, which says that no sequence is cut.
#pragma once

#include "device_util.h"
#include "host_logic.h"

namespace hxm {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
// Sum of v over lanes 0 .. lane: within the 16-lane rows by row_shr 1, 2, 4, 8
// (zeros come in), then the totals of the rows before.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {
  v += dpp_u32<0x111>(v);
  v += dpp_u32<0x112>(v);
  v += dpp_u32<0x114>(v);
  v += dpp_u32<0x118>(v);
  return v + (lane >= 16 ? lane_u32(v, 15) : 0u) + (lane >= 32 ? lane_u32(v, 31) : 0u) +
         (lane >= 48 ? lane_u32(v, 47) : 0u);
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  v += dpp_u32<kDppQuadXor1>(v);
  v += dpp_u32<kDppQuadXor2>(v);
  v += dpp_u32<kDppRowHalfMirror>(v);
  v += dpp_u32<kDppRowMirror>(v);
  return lane_u32(v, 0) + lane_u32(v, 16) + lane_u32(v, 32) + lane_u32(v, 48);
}

// A workgroup's piece of the batch.
struct Piece {
  int b;              // sequence, -1: none
  int n, lo;          // its tokens [lo, n)
  int begin, end;     // the piece's, begin a multiple of kAttnTile
  int pieces, index;  // of the sequence's head, and this one
  uint32_t slot;      // partial slots (of one head) of the sequences before
  bool over;          // longer than its table row
};

// Piece u of the batch, its sequences in order, cut as host_logic.h says.  Every wave
// works it out from the lengths, 64 sequences at a time, all loaded at once: they are on
// the device, so the host cannot.  Batches of more than 64 take the fine pieces without
// trying the others, which took 13 us instead of 15.4 for 256 x 600 tokens, one head, 12.3 for
// 13.7 (128 x 600, two) and 149 for 152 (256 x 2048, eight), and 15 for 11.6 where few tokens
// are many sequences' (65 x 1024, one head) and 30 for 25 (200 x 2048, one).  Trees of 8, heads
// of 128, in small steps past 64 sequences too: 65 x 2048 39.5 us for 32.0 with the steps (one
// head of 8), 38.1 for 36.6 (two of 4), 132 for 137 (eight of 4); 256 x 2048 67 for 64, 118 for
// 111, 397 for 411; one of 16384 among 65 of 200 tokens 39.9 for 40.3, 31.5 for 39.9, 42 for 48.
template <uint32_t GROUPS = kAttnGroups, bool STEPS = false, typename Args>
__device__ __forceinline__ Piece find_piece(const Args& a, uint32_t u, int lane) {
  auto tokens = [&](int32_t len, int* lo) {
    const int n = len > a.capacity ? 0 : max(len, 0);
    *lo = a.window > 0 ? max(0, n - a.window) : 0;
    return n;
  };
  auto units = [&](int b, int32_t len) {  // zero past the last sequence
    int lo;
    const int n = tokens(len, &lo);
    return b < a.batch ? attn_units(n, lo) : 0u;
  };
  auto length = [&](int b) { return b < a.batch ? a.lens[b] : 0; };
  Piece r{};
  r.b = -1;
  bool whole = a.batch > kAttnCutBatch;
  if constexpr (STEPS) whole = a.whole;
  if (whole) {  // a sequence each
    if (u >= static_cast<uint32_t>(a.batch)) return r;
    const int32_t len = a.lens[u];
    r.b = static_cast<int>(u), r.n = tokens(len, &r.lo), r.over = len > a.capacity;
    r.pieces = 1, r.begin = r.lo & ~static_cast<int>(kAttnTile - 1), r.end = r.n;
    return r;
  }
  constexpr int CHUNKS = kAttnCutBatch / 64;
  int32_t len[CHUNKS];
  uint32_t w[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) len[i] = 64 * i < a.batch ? length(64 * i + lane) : 0;
  uint64_t total = 0;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    w[i] = units(64 * i + lane, len[i]);
    if (64 * i < a.batch) total += wave_sum(w[i]);
  }
  const uint32_t share = attn_share(total, a.heads, GROUPS);
  uint32_t size = 0;
  bool fits = false;
  if (a.batch <= 64)
    for (uint32_t k = 0; k < (STEPS ? kAttnSteps : 4) && !fits; ++k) {
      size = STEPS ? attn_step_size(share, k) : attn_size(share, k);
      fits = wave_sum(attn_cut(w[0], size)) * a.heads <= GROUPS;
    }
  if (!fits) size = attn_fine_size(share);
  uint32_t first = 0, slots = 0;  // pieces, and partial slots, of the sequences before
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    if (64 * i >= a.batch) break;
    const uint32_t c = attn_cut(w[i], size), cs = c > 1 ? c : 0u;
    const uint32_t upto = wave_scan(c, lane), upto_s = wave_scan(cs, lane);
    const uint64_t hit = __ballot(u < first + upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int32_t len_l = static_cast<int32_t>(lane_u32(static_cast<uint32_t>(len[i]), l));
      const uint32_t pieces = lane_u32(c, l);
      const int step = static_cast<int>((lane_u32(w[i], l) + pieces - 1) / pieces) *
                       static_cast<int>(kAttnUnit);
      r.b = 64 * i + l;
      r.n = tokens(len_l, &r.lo);
      r.over = len_l > a.capacity;
      r.pieces = static_cast<int>(pieces);
      r.index = static_cast<int>(u - (first + lane_u32(upto, l) - pieces));
      r.slot = slots + lane_u32(upto_s, l) - lane_u32(cs, l);
      r.begin = (r.lo & ~static_cast<int>(kAttnTile - 1)) + r.index * step;
      r.end = r.index + 1 < r.pieces ? min(r.n, r.begin + step) : r.n;
      return r;
    }
    first += lane_u32(upto, 63);
    slots += lane_u32(upto_s, 63);
  }
  return r;
}

}  // namespace hxm
