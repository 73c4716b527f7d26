// Rows and pages of the paged key-value cache moved in every layer by one launch: the rows
// of the drafted tokens that were kept to the end of the context, and whole pages for
// sequences that fork.
//
// Bound by memory: every moved element is read once and written once (300 pages of 64 x 8 x 128
// in 16 layers, 2.2 GB in 439 us, 5.0 TB/s, a copy's rate; one page of 16 x 8 x 128 in 32 layers
// 3.8 us on the GPU, the kept rows of 8 trees of 32 in 32 layers 3.2).
#include <algorithm>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kMaxNodes = 64;
constexpr int kThreads = 256;
constexpr int kBatch = 8;  // vectors a thread has in flight (copies with 2: one page 7.1 us for 6.5)

struct LayersArg {
  char *k, *v;
  int64_t kls, kps, khs, kts, vls, vps, vhs, vts;
  int64_t pages;
  uint32_t page_size;
  int layers, heads, dim;
};

struct CompactArgs {
  LayersArg c;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* path;
  const int32_t* counts;
  int32_t* lens_out;
  int64_t ld_table, capacity;
  int nodes, groups;  // workgroups of a sequence
  int items;          // 16-byte columns of a token over all layers, keys and values
};

// A thread has one 16-byte column of a token's keys or values in one layer and moves it
// through all rows: eight loads, then eight stores, in the rows' order.  A row goes to a
// place before its own or its own, and the places are in order too, so that no load comes
// after a store to where it reads.
__global__ __launch_bounds__(kThreads) void compact_cache_kernel(CompactArgs a) {
  const int b = blockIdx.x / a.groups, group = blockIdx.x - b * a.groups;
  const int lane = threadIdx.x & 63;
  __shared__ int64_t from[2][kMaxNodes], to[2][kMaxNodes];
  __shared__ int moves;
  if (threadIdx.x < 64) {
    const int n = a.lens[b], count = a.counts[b];
    const int ctx = n - a.nodes;
    const bool in = lane < a.nodes && lane < count;
    const int node = in ? a.path[static_cast<int64_t>(b) * a.nodes + lane] : 0;
    const int before = __shfl_up(node, 1, 64);
    const bool wrong = in && (node >= a.nodes || node < (lane ? before + 1 : 0));
    // Left as it is: of too few or too many tokens, or no path.
    const bool valid =
        n >= a.nodes && n <= a.capacity && count >= 0 && count <= a.nodes && !__any(wrong);
    int64_t page[2] = {0, 0}, off[2] = {0, 0};
    bool move = valid && in && node != lane;
    if (move) {
      for (int i = 0; i < 2; ++i) {
        const uint32_t t = static_cast<uint32_t>(ctx + (i ? lane : node));
        page[i] = a.table[b * a.ld_table + t / a.c.page_size];
        off[i] = t % a.c.page_size;
        move &= page[i] >= 0 && page[i] < a.c.pages;
      }
    }
    const uint64_t all = __ballot(move);
    if (move) {
      const int at = __builtin_popcountll(all & ((uint64_t(1) << lane) - 1));
      from[0][at] = page[0] * a.c.kps + off[0] * a.c.kts;
      to[0][at] = page[1] * a.c.kps + off[1] * a.c.kts;
      from[1][at] = page[0] * a.c.vps + off[0] * a.c.vts;
      to[1][at] = page[1] * a.c.vps + off[1] * a.c.vts;
    }
    if (lane == 0) {
      moves = __builtin_popcountll(all);
      if (group == 0 && a.lens_out) a.lens_out[b] = valid ? ctx + count : n;
    }
  }
  __syncthreads();
  const int item = group * kThreads + static_cast<int>(threadIdx.x);
  if (item >= a.items) return;
  const int chunks = a.c.dim / 8;
  const int chunk = item % chunks, head = item / chunks % a.c.heads;
  const int rest = item / chunks / a.c.heads, kv = rest & 1;
  const int64_t layer = rest >> 1;
  typedef AnyVec<_Float16> Vec;
  _Float16* base = reinterpret_cast<_Float16*>(kv ? a.c.v : a.c.k) +
                   layer * (kv ? a.c.vls : a.c.kls) + head * (kv ? a.c.vhs : a.c.khs) + chunk * 8;
  const int n = moves;
  for (int i = 0; i < n; i += kBatch) {
    Vec x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (i + j < n) x[j] = *reinterpret_cast<const Vec*>(base + from[kv][i + j]);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (i + j < n) *reinterpret_cast<Vec*>(base + to[kv][i + j]) = x[j];
  }
}

struct CopyArgs {
  LayersArg c;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* rows;
  FastDiv chunk_div, inner_div;
  int inner;          // heads or tokens, whichever lie nearer
  bool tokens_outer;
  int items, parts;   // 16-byte vectors of a page of one layer's keys, workgroups for them
};

__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a) {
  uint32_t x = blockIdx.x;
  const int part = static_cast<int>(x % static_cast<uint32_t>(a.parts));
  x /= static_cast<uint32_t>(a.parts);
  const int kv = static_cast<int>(x & 1u);
  x >>= 1;
  const int64_t layer = x % static_cast<uint32_t>(a.c.layers);
  const int64_t i = x / static_cast<uint32_t>(a.c.layers);
  const int64_t src = a.src[i], dst = a.dst[i];
  if (src < 0 || src >= a.c.pages || dst < 0 || dst >= a.c.pages) return;
  const int rows = a.rows ? a.rows[i] : static_cast<int>(a.c.page_size);
  _Float16* base = reinterpret_cast<_Float16*>(kv ? a.c.v : a.c.k) +
                   layer * (kv ? a.c.vls : a.c.kls);
  const int64_t ps = kv ? a.c.vps : a.c.kps, hs = kv ? a.c.vhs : a.c.khs,
                ts = kv ? a.c.vts : a.c.kts;
  const int chunks = a.c.dim / 8;
  typedef AnyVec<_Float16> Vec;
  Vec v[kBatch];
  int64_t at[kBatch];
  auto div = [](uint32_t n, FastDiv d) {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * d.mul) >> d.shift);
  };
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int64_t item = static_cast<int64_t>(part) * (kThreads * kBatch) + j * kThreads +
                         static_cast<int>(threadIdx.x);
    at[j] = -1;
    if (item < a.items) {
      const uint32_t row = div(static_cast<uint32_t>(item), a.chunk_div);
      const uint32_t chunk = static_cast<uint32_t>(item) - row * chunks;
      const uint32_t outer = div(row, a.inner_div), inner = row - outer * a.inner;
      const uint32_t tok = a.tokens_outer ? outer : inner, head = a.tokens_outer ? inner : outer;
      if (static_cast<int64_t>(tok) < rows)
        at[j] = static_cast<int64_t>(tok) * ts + static_cast<int64_t>(head) * hs + chunk * 8;
    }
    if (at[j] >= 0) v[j] = load_any(base + src * ps + at[j]);
  }
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (at[j] >= 0) store_any(base + dst * ps + at[j], v[j]);
}

// The cache of every layer, checked.
hxm_status layers_arg(const char* op, const hxm_kv_cache* c, int64_t layers, int64_t kls,
                      int64_t vls, LayersArg* out) {
  hxm_status st = check_kv_cache(op, c, true);
  if (st != HXM_OK) return st;
  if (layers < 1 || layers > 65535 || !stride_ok(kls) || !stride_ok(vls))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s %lld layers, strides %lld, %lld", op,
                (long long)layers, (long long)kls, (long long)vls);
  if (layers > 1 && !layers_apart(c, layers, kls, vls))
    return fail(HXM_INVALID_ARG, "invalid-argument: %s layers share elements", op);
  *out = LayersArg{static_cast<char*>(c->k), static_cast<char*>(c->v), kls, c->k_page_stride,
                   c->k_head_stride, c->k_token_stride, vls, c->v_page_stride, c->v_head_stride,
                   c->v_token_stride, c->pages, static_cast<uint32_t>(c->page_size),
                   static_cast<int>(layers), static_cast<int>(c->heads),
                   static_cast<int>(c->dim)};
  return HXM_OK;
}

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_compact_cache(const hxm_kv_cache* cache, int64_t layers,
                                        int64_t k_layer_stride, int64_t v_layer_stride,
                                        const int32_t* block_table, int64_t ld_table,
                                        int64_t table_pages, const int32_t* seq_lens,
                                        const int32_t* path, const int32_t* counts,
                                        int32_t* lens_out, int64_t batch, int64_t nodes,
                                        int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: compact_cache takes f16 or bf16 (got %d)",
                dtype);
  CompactArgs a{};
  hxm_status st = layers_arg("compact_cache", cache, layers, k_layer_stride, v_layer_stride, &a.c);
  if (st != HXM_OK) return st;
  if (batch < 0 || nodes < 1)
    return fail(HXM_INVALID_ARG, "invalid-argument: compact_cache batch=%lld, nodes=%lld",
                (long long)batch, (long long)nodes);
  const int64_t items = layers * 2 * cache->heads * (cache->dim / 8);
  if (nodes > kMaxNodes || batch > INT32_MAX || items > INT32_MAX / 2)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: compact_cache batch=%lld, nodes=%lld, %lld layers",
                (long long)batch, (long long)nodes, (long long)layers);
  if (table_pages < 0 || table_pages > INT32_MAX || !stride_ok(ld_table) ||
      (batch > 1 && ld_table < table_pages) ||
      (batch > 0 && (!seq_lens || !path || !counts || (table_pages > 0 && !block_table))))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: compact_cache table of %lld pages, ld %lld, or null operand",
                (long long)table_pages, (long long)ld_table);
  for (const int32_t* p : {seq_lens, counts})
    if (lens_out && !matrices_disjoint(reinterpret_cast<uintptr_t>(lens_out), batch,
                                       reinterpret_cast<uintptr_t>(p), batch, 1, batch, batch, 4))
      return fail(HXM_INVALID_ARG,
                  "invalid-argument: compact_cache lens_out overlaps seq_lens or counts");
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (batch == 0) return ok();
  a.table = block_table, a.lens = seq_lens, a.path = path, a.counts = counts;
  a.lens_out = lens_out, a.ld_table = ld_table;
  a.capacity = std::min(table_pages * cache->page_size, int64_t(INT32_MAX));
  a.nodes = static_cast<int>(nodes), a.items = static_cast<int>(items);
  a.groups = static_cast<int>(ceil_div(items, kThreads));
  const int64_t groups = batch * a.groups;
  if ((st = check_grid("compact cache", groups, kThreads)) != HXM_OK) return st;
  compact_cache_kernel<<<static_cast<unsigned>(groups), kThreads, 0, as_stream(stream)>>>(a);
  return check_launch("compact cache");
}

extern "C" hxm_status hxm_copy_pages(const hxm_kv_cache* cache, int64_t layers,
                                     int64_t k_layer_stride, int64_t v_layer_stride,
                                     const int32_t* src, const int32_t* dst, const int32_t* rows,
                                     int64_t count, int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: copy_pages takes f16 or bf16 (got %d)",
                dtype);
  CopyArgs a{};
  hxm_status st = layers_arg("copy_pages", cache, layers, k_layer_stride, v_layer_stride, &a.c);
  if (st != HXM_OK) return st;
  if (count < 0 || (count > 0 && (!src || !dst)))
    return fail(HXM_INVALID_ARG, "invalid-argument: copy_pages of %lld, or null pages",
                (long long)count);
  const int64_t chunks = cache->dim / 8;
  // (page_size * heads stays under 2^47.)
  if (cache->page_size * cache->heads > INT32_MAX / 2 / chunks || count > (int64_t(1) << 24))
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: copy_pages of %lld, of %lld tokens, %lld heads", (long long)count,
                (long long)cache->page_size, (long long)cache->heads);
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (count == 0) return ok();
  a.src = src, a.dst = dst, a.rows = rows;
  a.items = static_cast<int>(cache->page_size * cache->heads * chunks);
  a.parts = static_cast<int>(ceil_div(a.items, kThreads * kBatch));
  a.tokens_outer = cache->k_token_stride > cache->k_head_stride;
  a.inner = static_cast<int>(a.tokens_outer ? cache->heads : cache->page_size);
  a.chunk_div = fast_div(static_cast<uint32_t>(chunks));
  a.inner_div = fast_div(static_cast<uint32_t>(a.inner));
  const int64_t groups = count * layers * 2 * a.parts;
  if ((st = check_grid("copy pages", groups, kThreads)) != HXM_OK) return st;
  copy_pages_kernel<<<static_cast<unsigned>(groups), kThreads, 0, as_stream(stream)>>>(a);
  return check_launch("copy pages");
}
