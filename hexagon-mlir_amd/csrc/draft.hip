// Which of a sequence's drafted tokens the target's probabilities keep, and the token that
// follows them.
//
// Bound by the read of one row of the vocabulary per sequence (two with the draft's
// probabilities): the tests themselves need one probability per drafted token.  64 chains of
// five over 128000, both tables fp32, 62 MB in 27 us; one tree of 26 over 32000 in 12.9, a chain
// of dependent reads: the tree, its probabilities, the row, the sums, the token's block.
//
// A sequence's row is cut into chunks, a workgroup each.  Every one of them walks the tree by
// itself (a lane a node; the probabilities of all nodes are read at once, the walk then
// takes one child after the other), sums its chunk of what is left in the row where the walk
// ends, and the last to arrive looks for the chunk that holds the drawn point, and for the
// token in it.  Nobody waits.  (Arrivals with release and acquire, which maintain the caches,
// and chunks that end inside a block of loads: 51 us for 27.)
//
// Sums and products are in 64 bits: probabilities have 24, a product of two is exact, and
// the sum of a row is off by about 2^-53 of itself per term, so that the drawn token is
// that of exact arithmetic but for a point within that of a border between two tokens.
#include <algorithm>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kMaxNodes = 64;
constexpr int kThreads = 256;
// A chunk is whole blocks of elements, 16 a thread; as many chunks as give this many workgroups
// (64 x 5 x 128000: 512 31.5 us, 1024 26.8, 2048 30.1; 128 x 5 x 32000 20.3, 18.4, 18.4).
constexpr int64_t kBlock = 16 * kThreads, kGroups = 1024;

struct VerifyArgs {
  const int32_t* tokens;
  const int32_t* parents;
  const void* target;
  const void* draft;
  const float* uniform;
  int64_t ldt, ldd, vocab;
  int32_t *path, *counts, *next;
  double* sums;       // [batch][chunks]
  uint32_t* arrived;  // [batch], zero between launches
  int batch, nodes, chunks;
  int64_t chunk;      // elements
};

// Probabilities below zero, and those that are no numbers, count as zero.
template <typename T>
__device__ __forceinline__ double prob(T v) {
  return static_cast<double>(fmaxf(tof(v), 0.0f));
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Where the walk of a sequence ends.
struct End {
  int node;        // the last one kept, -1: no sequence
  int count;       // kept ones
  uint64_t kept;   // a bit each
  uint64_t tried;  // its children that were tried, none kept
  int token;       // lane i: node i's token
  double first;    // node 0's random number
};
template <typename T, bool DRAFT>
__device__ __forceinline__ End walk(const VerifyArgs& a, int b, int lane) {
  const bool in = lane < a.nodes;
  const int64_t at = static_cast<int64_t>(b) * a.nodes + (in ? lane : 0);
  const int token = a.tokens[at];
  int parent = a.parents ? a.parents[at] : lane - 1;
  const double u = a.uniform[at];
  // No child: past the nodes, of no earlier node, or of a token that is none.
  const bool child = in && parent >= 0 && parent < lane && token >= 0 && token < a.vocab;
  End r{-1, 0, 0, 0, token, lane_f64(u, 0)};
  if (__builtin_amdgcn_readfirstlane(parent) != -1) return r;
  double p = 0.0, q = 1.0;
  if (child) {
    const int64_t row = static_cast<int64_t>(b) * a.nodes + parent;
    p = prob(static_cast<const T*>(a.target)[row * a.ldt + token]);
    if (DRAFT) q = prob(static_cast<const T*>(a.draft)[row * a.ldd + token]);
  }
  if (!child) parent = -1;
  // From node to node; a node's children in their order.
  const double bound = u * q;
  r.node = 0, r.kept = 1, r.count = 1;
  double left = 1.0;
  for (uint64_t children = __ballot(parent == 0); children;) {
    const int c = __builtin_ctzll(children);
    const uint64_t bit = children & (0 - children);
    children ^= bit;
    if (!DRAFT) {
      const int tc = __builtin_amdgcn_readlane(token, c);
      const uint64_t same = __ballot(token == tc) & r.tried;
      r.tried |= bit;
      if (same) continue;
    }
    const double pc = lane_f64(p, c);
    if (lane_f64(bound, c) * left < pc) {
      r.node = c, r.kept |= bit, ++r.count;
      r.tried = 0, left = 1.0;
      children = __ballot(parent == c);
    } else if (DRAFT) {
      r.tried = bit;
      break;
    } else {
      left -= pc;
    }
  }
  return r;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m, 64);
  return v;
}

template <typename T, bool DRAFT>
__global__ __launch_bounds__(kThreads) void verify_draft_kernel(VerifyArgs a) {
  constexpr int E = RowVec<T>::N;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x;
  __shared__ double totals[kThreads / 64];
  __shared__ int32_t gone[kMaxNodes];
  __shared__ int furthest, last;
  __shared__ double found_before;
  __shared__ int found;

  const End end = walk<T, DRAFT>(a, b, lane);
  if (chunk == 0 && wave == 0) {
    if (lane < a.nodes) {
      // The kept nodes in front, in their order, then -1.
      const bool kept = (end.kept >> lane) & 1;
      const uint64_t below = (uint64_t(1) << lane) - 1;
      const int at = kept ? __builtin_popcountll(end.kept & below)
                          : end.count + __builtin_popcountll(~end.kept & below);
      a.path[static_cast<int64_t>(b) * a.nodes + at] = kept ? lane : -1;
    }
    if (lane == 0) a.counts[b] = end.count;
    if (lane == 0 && end.node < 0) a.next[b] = -1;
  }
  if (end.node < 0) return;
  // The tokens in [from, to) that are gone from the row (a one-hot draft's).
  auto list_gone = [&](int64_t from, int64_t to) {
    if (DRAFT) return 0;
    __syncthreads();
    const uint64_t in =
        __ballot(((end.tried >> lane) & 1) != 0 && end.token >= from && end.token < to);
    if (wave == 0 && ((in >> lane) & 1))
      gone[__builtin_popcountll(in & ((uint64_t(1) << lane) - 1))] = end.token;
    __syncthreads();
    return static_cast<int>(__builtin_popcountll(in));
  };
  const int64_t row = static_cast<int64_t>(b) * a.nodes + end.node;
  const T* p = static_cast<const T*>(a.target) + row * a.ldt;
  const T* q = DRAFT && end.tried ? static_cast<const T*>(a.draft) + row * a.ldd : nullptr;
  // What the row leaves of element v, `ngone` of the tokens listed (whole: of all of them).
  auto weigh = [&](T pv, T qv, int64_t v, int ngone, bool whole) {
    double w = prob(pv);
    if (DRAFT && q && !whole) w = fmax(w - prob(qv), 0.0);
    if (!DRAFT)
      for (int i = 0; i < ngone; ++i) w = gone[i] == v ? 0.0 : w;
    return w;
  };
  // Vectors of a thread, at a distance of `step` elements, from v on, as far as `to` (inside:
  // all of them of every thread, which are loaded at once).
  auto weights = [&](auto& w, int64_t v, int64_t step, int64_t to, bool inside, int ngone,
                     bool whole) {
    constexpr int N = sizeof(w) / sizeof(w[0]) / E;
    RawVec<T> pv[N], qv[N];
    if (inside) {
#pragma unroll
      for (int i = 0; i < N; ++i) pv[i] = load_any(p + v + i * step);
      if (DRAFT && q) {
#pragma unroll
        for (int i = 0; i < N; ++i) qv[i] = load_any(q + v + i * step);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t x = v + i * step;
        pv[i] = qv[i] = RawVec<T>(T(0));
        if (x + E <= to) {
          pv[i] = load_any(p + x);
          if (DRAFT && q) qv[i] = load_any(q + x);
        } else if (x < to) {
          pv[i] = load_tail(p, x, to, T(0));
          if (DRAFT && q) qv[i] = load_tail(q, x, to, T(0));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e)
        w[i * E + e] = weigh(pv[i][e], qv[i][e], v + i * step + e, ngone, whole);
  };
  const int64_t lo = chunk * a.chunk, hi = min(a.vocab, lo + a.chunk);
  auto block_sum = [&](double s) {
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) totals[wave] = s;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) t += totals[i];
    return t;
  };
  auto sum_of = [&](int64_t from, int64_t to, bool whole) {
    constexpr int N = 16 / E;
    const int ngone = whole ? 0 : list_gone(from, to);
    double s = 0.0;
    for (int64_t v = from; v < to; v += kThreads * N * E) {
      double w[N * E];
      weights(w, v + tid * E, kThreads * E, to, v + kThreads * N * E <= to, ngone, whole);
#pragma unroll
      for (int e = 0; e < N * E; ++e) s += w[e];
    }
    return block_sum(s);
  };
  const double mine = sum_of(lo, hi, false);
  double* sums = a.sums + static_cast<int64_t>(b) * a.chunks;
  if (tid == 0) {
    // Written through to the coherence point, and there before the arrival is.
    __hip_atomic_store(sums + chunk, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t before =
        __hip_atomic_fetch_add(a.arrived + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = before == static_cast<uint32_t>(a.chunks - 1);
    if (last) __hip_atomic_store(a.arrived + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;

  // The chunk where the sum of those up to it passes the drawn point: lanes of the first
  // wave, 64 chunks at a time.
  auto load_sum = [&](int i) {
    return i < a.chunks
               ? __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
               : 0.0;
  };
  auto scan = [&](double v) {  // over lanes 0 .. lane
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const double o = __shfl_up(v, m, 64);
      if (lane >= m) v += o;
    }
    return v;
  };
  double total = 0.0;
  for (int i = 0; i < a.chunks; i += 64) total += wave_sum(load_sum(i + lane));
  bool whole = false;
  if (!(total > 0.0)) {
    // Nothing is left (the target's probabilities lie below the draft's everywhere, by
    // their rounding): the whole row.
    whole = true;
    total = sum_of(0, a.vocab, true);
  }
  if (!(total > 0.0) || !(total < __builtin_huge_val())) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  const double point = end.first * total;
  int64_t from = 0, to = a.vocab;
  double before = 0.0;
  if (!whole) {
    if (wave == 0) {
      double run = 0.0, start = 0.0;
      int at = -1, some = 0;
      double some_before = 0.0;
      for (int i = 0; i < a.chunks && at < 0; i += 64) {
        const double v = load_sum(i + lane), upto = run + scan(v);
        const uint64_t past = __ballot(i + lane < a.chunks && v > 0.0 && upto > point);
        const uint64_t any = __ballot(v > 0.0);
        if (past) {
          const int k = __builtin_ctzll(past);
          at = i + k, start = lane_f64(upto - v, k);
        }
        if (any) {
          const int k = 63 - __builtin_clzll(any);
          some = i + k, some_before = lane_f64(upto - v, k);
        }
        run = lane_f64(upto, 63);
      }
      // (The sums round: the last chunk that has any where none passes the point.)
      if (lane == 0) found = at >= 0 ? at : some, found_before = at >= 0 ? start : some_before;
    }
    __syncthreads();
    from = found * a.chunk, to = min(a.vocab, from + a.chunk), before = found_before;
    __syncthreads();
  }
  // The token: blocks of consecutive elements, a thread 16 of them.
  constexpr int P = 16;
  const int ngone = whole ? 0 : list_gone(from, to);
  if (tid == 0) found = INT32_MAX, furthest = -1;
  for (int64_t v0 = from; v0 < to; v0 += kThreads * P) {
    const int64_t v = v0 + tid * P;
    double w[P];
    weights(w, v, E, to, v0 + kThreads * P <= to, ngone, whole);
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < P; ++e) s += w[e];
    const double upto = scan(s);
    __syncthreads();
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    double run = before + (upto - s);
    for (int i = 0; i < wave; ++i) run += totals[i];
    int first = INT32_MAX, end_of = -1;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      run += w[e];
      if (w[e] > 0.0) {
        end_of = static_cast<int>(v + e);
        if (run > point && first == INT32_MAX) first = end_of;
      }
    }
    if (first != INT32_MAX) atomicMin(&found, first);
    if (end_of >= 0) atomicMax(&furthest, end_of);
    __syncthreads();
    if (found != INT32_MAX) break;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) before += totals[i];
  }
  // (The sums round: the last that has any where none passes the point.)
  if (tid == 0) a.next[b] = found != INT32_MAX ? found : furthest;
}

template <typename T>
hxm_status launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int64_t groups = int64_t(a.batch) * a.chunks;
  hxm_status st = check_grid("verify draft", groups, kThreads);
  if (st != HXM_OK) return st;
  const unsigned n = static_cast<unsigned>(groups);
  if (a.draft) verify_draft_kernel<T, true><<<n, kThreads, 0, s>>>(a);
  else verify_draft_kernel<T, false><<<n, kThreads, 0, s>>>(a);
  return check_launch("verify draft");
}

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_verify_draft(const int32_t* tokens, const int32_t* parents,
                                       const void* target, int64_t ld_target, const void* draft,
                                       int64_t ld_draft, const float* uniform, int32_t* path,
                                       int32_t* counts, int32_t* next_tokens, int64_t batch,
                                       int64_t nodes, int64_t vocab, int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16 && dtype != HXM_F32)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: verify_draft takes f16, bf16 or f32 "
                "(got %d)", dtype);
  if (batch < 0 || nodes < 1 || vocab < 1)
    return fail(HXM_INVALID_ARG, "invalid-argument: verify_draft batch=%lld, nodes=%lld, vocab=%lld",
                (long long)batch, (long long)nodes, (long long)vocab);
  if (nodes > kMaxNodes || batch > (int64_t(1) << 20) || vocab > INT32_MAX / 2)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: verify_draft batch=%lld, nodes=%lld, vocab=%lld",
                (long long)batch, (long long)nodes, (long long)vocab);
  if (batch > 0 && (!tokens || !target || !uniform || !path || !counts || !next_tokens))
    return fail(HXM_INVALID_ARG, "invalid-argument: verify_draft null operand");
  for (const int64_t ld : {ld_target, draft ? ld_draft : vocab})
    if (!stride_ok(ld) || (batch * nodes > 1 && ld < vocab))
      return fail(HXM_INVALID_ARG, "invalid-argument: verify_draft ld=%lld of %lld",
                  (long long)ld, (long long)vocab);
  hxm_status st = require_device(nullptr);
  if (st != HXM_OK) return st;
  if (batch == 0) return ok();
  VerifyArgs a{};
  a.tokens = tokens, a.parents = parents, a.target = target, a.draft = draft;
  a.uniform = uniform, a.ldt = ld_target, a.ldd = ld_draft, a.vocab = vocab;
  a.path = path, a.counts = counts, a.next = next_tokens;
  a.batch = static_cast<int>(batch), a.nodes = static_cast<int>(nodes);
  const int64_t want = std::max(int64_t(1), kGroups / batch);
  a.chunk = ceil_div(ceil_div(vocab, want), kBlock) * kBlock;
  a.chunks = static_cast<int>(ceil_div(vocab, a.chunk));
  hipStream_t s = as_stream(stream);
  void* ws = nullptr;
  if ((st = stream_workspace(s, static_cast<size_t>(batch) * 4, &ws, kWsCount)) != HXM_OK) return st;
  a.arrived = static_cast<uint32_t*>(ws);
  st = stream_workspace(s, static_cast<size_t>(batch) * a.chunks * 8, &ws, kWsLayer);
  if (st != HXM_OK) return st;
  a.sums = static_cast<double*>(ws);
  if (dtype == HXM_F16) return launch_verify<_Float16>(a, s);
  if (dtype == HXM_BF16) return launch_verify<__bf16>(a, s);
  return launch_verify<float>(a, s);
}
