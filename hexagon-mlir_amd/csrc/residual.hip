// The norms on both sides of a block, its gate and the residual add, in one
// pass over the rows:
//   p = post(h);  y = residual_scale * x + block_scale * gate * p;  z = pre(y).
//
// Bound by memory: h and x are read once, y and z written once, 4 * rows * cols
// elements against about ten operations each (8192 x 4096 f16: 268 MB in 48 us, 5.6
// TB/s; a copy of as much runs at 5.4).  Done apart (norm, add, norm) the same
// takes 8 * rows * cols.  As in the row kernels a row is held in
// registers by S waves: h and x in their storage type, y in fp32, so that z is
// the norm of the y before its rounding; the norms' sums cross the waves
// through LDS.  The kinds of the two norms are uniform branches, not template
// arguments: nine pairs of kinds would be nine copies of every row width.
#include <type_traits>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

struct NormArgs {
  int kind;
  float eps;
  const void* gamma;
  const void* beta;
};

struct ResidualArgs {
  const void* h;
  const void* x;
  void* y;
  void* z;
  const void* gate;
  int64_t ldh, ldx, ldy, ldz, ldg;
  int64_t cols;
  NormArgs post, pre;
  float block_scale, residual_scale;
  uint32_t rows, rows_per_gate;  // rows_per_gate 0: one gate row for all
};

// Scale and shift of a norm's row: v -> (v - mean) * rstd.
struct RowStats {
  float mean, rstd;
};

// Registers: h, x and the fp32 y of VPL vectors a lane.
//
// EARLY: weights, biases and gate are loaded with h and x, not where they are used. For
// calls of one workgroup a CU or fewer, whose time is their chain of loads (1 x 8192 bf16,
// LayerNorms and gate: 7.6 -> 6.6 us; 300 x 1000 f32: 6.1 -> 5.3); the registers it takes
// cost larger ones more (2048 x 4096 bf16 14.4 -> 16.6), and 16 waves a row have none left.
template <typename T, int VPL, int S, bool EARLY>
__global__ __launch_bounds__(row_waves(S) * 64) void residual_norm_kernel(ResidualArgs a) {
  constexpr int N = RowVec<T>::N;
  constexpr int WAVES = row_waves(S);
  constexpr int TAIL0 = VPL <= 4 ? VPL - 1 : VPL / 2;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, part = wv % S;
  const uint32_t r = blockIdx.x * (WAVES / S) + wv / S;
  // Waves past the last row stay for the barriers, read row 0, store nothing.
  const bool valid = r < a.rows;
  const int64_t rv = valid ? r : 0;
  const T* hr = static_cast<const T*>(a.h) + rv * a.ldh;
  const T* xr = static_cast<const T*>(a.x) + rv * a.ldx;
  const int64_t cols = a.cols;
  __shared__ float red[4][WAVES];
  auto row_sum = [&](float v, int slot) {
    v = wave_reduce(v, OpSum());
    if constexpr (S > 1) {
      if (lane == 0) red[slot][wv] = v;
      __syncthreads();
      v = wave_totals<S>(red[slot] + (wv / S) * S, OpSum());
    }
    return v;
  };
  auto col0 = [&](int i) { return ((static_cast<int64_t>(i) * S + part) * 64 + lane) * N; };
  // Slot i holds row elements only (uniform; every slot before TAIL0 does).
  auto whole = [&](int i) { return i < TAIL0 || (i + 1) * (S * 64 * N) <= cols; };
  auto load_at = [&](const T* p, int i, T fill) -> RawVec<T> {
    const int64_t c = col0(i);
    if (i < TAIL0) return load_any(p + c);
    RawVec<T> v = RawVec<T>(fill);
    if (cols >= N) {  // a lane past the row loads column 0: no branch splits the loads
      const bool in = c + N <= cols;
      const RawVec<T> t = load_any(p + (in ? c : 0));
      v = in ? t : v;
    }
    if (c < cols && c + N > cols) v = load_tail(p, c, cols, fill);
    return v;
  };
  auto store_at = [&](T* p, int i, RawVec<T> v) {
    const int64_t c = col0(i);
    if (i < TAIL0 || c + N <= cols) store_any(p + c, v);
    else if (c < cols) store_tail(p, c, cols, v);
  };
  auto param = [&](const void* p, int i, T none) {
    return p ? load_at(static_cast<const T*>(p), i, T(0)) : RawVec<T>(none);
  };
  // Mean and 1 / sqrt(var + eps) of a row given by f(i, j); the centred second
  // pass keeps the cancellation out of the variance.
  auto stats = [&](const NormArgs& n, int slot, auto f) {
    RowStats s{0.0f, 1.0f};
    if (n.kind == HXM_NORM_LAYER) {
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) t += f(i, j);
      s.mean = row_sum(t, slot) / static_cast<float>(cols);
    }
    if (n.kind != HXM_NORM_NONE) {
      float q = 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const bool all = whole(i);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float d = f(i, j) - s.mean;
          q = (all || col0(i) + j < cols) ? fmaf(d, d, q) : q;
        }
      }
      s.rstd = 1.0f / sqrtf(row_sum(q, slot + 1) / static_cast<float>(cols) + n.eps);
    }
    return s;
  };

  RawVec<T> h[VPL], x[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) h[i] = load_at(hr, i, T(0));
#pragma unroll
  for (int i = 0; i < VPL; ++i) x[i] = load_at(xr, i, T(0));
  const T* gate = static_cast<const T*>(a.gate);
  if (gate && a.rows_per_gate)
    gate += static_cast<int64_t>(static_cast<uint32_t>(rv) / a.rows_per_gate) * a.ldg;

  struct Params {
    RawVec<T> post_w, post_b, gate, pre_w, pre_b;
  };
  auto load_post = [&](Params& p, int i) {
    p.post_w = param(a.post.gamma, i, T(1)), p.post_b = param(a.post.beta, i, T(0));
    p.gate = param(gate, i, T(1));
  };
  auto load_pre = [&](Params& p, int i) {
    p.pre_w = param(a.pre.gamma, i, T(1)), p.pre_b = param(a.pre.beta, i, T(0));
  };
  Params early[EARLY ? VPL : 1];
  if constexpr (EARLY) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) load_post(early[i], i), load_pre(early[i], i);
  }

  const RowStats ps = stats(a.post, 0, [&](int i, int j) { return tof(h[i][j]); });
  float y[VPL][N];
  T* yr = static_cast<T*>(a.y) + rv * a.ldy;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    Params& q = early[EARLY ? i : 0];
    if constexpr (!EARLY) load_post(q, i);
    const bool all = whole(i);
    RawVec<T> o;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float p =
          fmaf((tof(h[i][j]) - ps.mean) * ps.rstd, tof(q.post_w[j]), tof(q.post_b[j]));
      const float v = fmaf(a.block_scale * tof(q.gate[j]), p, a.residual_scale * tof(x[i][j]));
      y[i][j] = all || col0(i) + j < cols ? v : 0.0f;
      o[j] = fromf<T>(v);
    }
    if (valid) store_at(yr, i, o);
  }
  if (!a.z) return;
  const RowStats zs = stats(a.pre, 2, [&](int i, int j) { return y[i][j]; });
  T* zr = static_cast<T*>(a.z) + rv * a.ldz;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    Params& q = early[EARLY ? i : 0];
    if constexpr (!EARLY) load_pre(q, i);
    RawVec<T> o;
#pragma unroll
    for (int j = 0; j < N; ++j)
      o[j] = fromf<T>(fmaf((y[i][j] - zs.mean) * zs.rstd, tof(q.pre_w[j]), tof(q.pre_b[j])));
    if (valid) store_at(zr, i, o);
  }
}

// Rows too long for the registers: 16 waves re-read h and x in every pass and
// compute y again.  y and z are written in the last pass alone, each element by
// the thread that has read it, so that they may be h or x.  Every statistic is a pass:
// 512 x 32768 f32, 268 MB, takes 69 us with an RMSNorm after, 77 with one on either side and
// 101 with LayerNorms, where the same bytes in rows of half the length, held in registers,
// take 43 to 45.
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_stream_kernel(ResidualArgs a) {
  constexpr int N = RowVec<T>::N, S = 16;
  const int64_t r = blockIdx.x, cols = a.cols;
  const T* hr = static_cast<const T*>(a.h) + r * a.ldh;
  const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
  const T* gate = static_cast<const T*>(a.gate);
  if (gate && a.rows_per_gate)
    gate += static_cast<int64_t>(static_cast<uint32_t>(r) / a.rows_per_gate) * a.ldg;
  __shared__ float red[4][S];
  auto row_sum = [&](float v, int slot) {
    v = wave_reduce(v, OpSum());
    if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    return wave_totals<S>(red[slot], OpSum());
  };
  auto at = [&](const void* p, int64_t c0, int n, T none) -> RawVec<T> {
    if (!p) return RawVec<T>(none);
    const T* q = static_cast<const T*>(p);
    return n == N ? load_any(q + c0) : load_tail(q, c0, cols, none);
  };
  // f(first column, elements inside the row) over this thread's vectors.
  auto each = [&](auto f) {
    const int64_t nfull = cols / N;
    for (int64_t i = threadIdx.x; i < nfull; i += S * 64) f(i * N, N);
    const int rem = static_cast<int>(cols - nfull * N);
    if (rem && static_cast<int64_t>(threadIdx.x) == nfull % (S * 64)) f(nfull * N, rem);
  };
  auto stats = [&](const NormArgs& n, int slot, auto value) {
    RowStats s{0.0f, 1.0f};
    if (n.kind == HXM_NORM_LAYER) {
      float t = 0.0f;
      each([&](int64_t c0, int m) {
        float v[N];
        value(c0, m, v);
#pragma unroll
        for (int j = 0; j < N; ++j) t += j < m ? v[j] : 0.0f;
      });
      s.mean = row_sum(t, slot) / static_cast<float>(cols);
    }
    if (n.kind != HXM_NORM_NONE) {
      float q = 0.0f;
      each([&](int64_t c0, int m) {
        float v[N];
        value(c0, m, v);
#pragma unroll
        for (int j = 0; j < N; ++j) q = j < m ? fmaf(v[j] - s.mean, v[j] - s.mean, q) : q;
      });
      s.rstd = 1.0f / sqrtf(row_sum(q, slot + 1) / static_cast<float>(cols) + n.eps);
    }
    return s;
  };
  const RowStats ps = stats(a.post, 0, [&](int64_t c0, int m, float (&v)[N]) {
    const RawVec<T> h = at(hr, c0, m, T(0));
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = tof(h[j]);
  });
  auto stream_y = [&](int64_t c0, int m, float (&v)[N]) {
    const RawVec<T> h = at(hr, c0, m, T(0)), x = at(xr, c0, m, T(0)),
                    w = at(a.post.gamma, c0, m, T(1)), b = at(a.post.beta, c0, m, T(0)),
                    g = at(gate, c0, m, T(1));
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float p = fmaf((tof(h[j]) - ps.mean) * ps.rstd, tof(w[j]), tof(b[j]));
      v[j] = fmaf(a.block_scale * tof(g[j]), p, a.residual_scale * tof(x[j]));
    }
  };
  RowStats zs{0.0f, 1.0f};
  if (a.z) zs = stats(a.pre, 2, stream_y);
  T* yr = static_cast<T*>(a.y) + r * a.ldy;
  T* zr = static_cast<T*>(a.z) + (a.z ? r * a.ldz : 0);
  auto store = [&](T* p, int64_t c0, int m, RawVec<T> v) {
    if (m == N) store_any(p + c0, v);
    else store_tail(p, c0, cols, v);
  };
  each([&](int64_t c0, int m) {
    float v[N];
    stream_y(c0, m, v);
    RawVec<T> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = fromf<T>(v[j]);
    store(yr, c0, m, o);
    if (a.z) {
      const RawVec<T> w = at(a.pre.gamma, c0, m, T(1)), b = at(a.pre.beta, c0, m, T(0));
#pragma unroll
      for (int j = 0; j < N; ++j)
        o[j] = fromf<T>(fmaf((v[j] - zs.mean) * zs.rstd, tof(w[j]), tof(b[j])));
      store(zr, c0, m, o);
    }
  });
}

// Waves per row and vectors per lane by the row's vectors, as the row kernels
// choose them; rows beyond 4096 vectors would need more than the 128
// registers a lane of 16 waves has.
template <typename T>
hxm_status launch_residual(const ResidualArgs& a, hipStream_t stream) {
  const int64_t nv = ceil_div(a.cols, RowVec<T>::N);
  hxm_status st = HXM_OK;
  auto launch = [&](auto kernel, int threads, int per_group) {
    const int64_t groups = ceil_div(a.rows, per_group);
    if ((st = check_grid("residual norm", groups, threads)) != HXM_OK) return;
    kernel<<<static_cast<unsigned>(groups), threads, 0, stream>>>(a);
    st = check_launch("residual norm");
  };
#define HXM_RESIDUAL(V, S)                                                                      \
  ceil_div(a.rows, row_waves(S) / (S)) <= 256                                                  \
      ? launch(residual_norm_kernel<T, V, S, (S < 16)>, 64 * row_waves(S), row_waves(S) / (S)) \
      : launch(residual_norm_kernel<T, V, S, false>, 64 * row_waves(S), row_waves(S) / (S))
  if (nv <= 64) HXM_RESIDUAL(1, 1);
  else if (nv <= 128) HXM_RESIDUAL(2, 1);
  else if (nv <= 192) HXM_RESIDUAL(3, 1);
  else if (nv <= 256) HXM_RESIDUAL(4, 1);
  else if (nv <= 512) HXM_RESIDUAL(2, 4);
  else if (nv <= 768) HXM_RESIDUAL(3, 4);
  else if (nv <= 1024) HXM_RESIDUAL(4, 4);
  else if (nv <= 1536) HXM_RESIDUAL(3, 8);
  else if (nv <= 2048) HXM_RESIDUAL(4, 8);
  else if (nv <= 3 * 1024) HXM_RESIDUAL(3, 16);
  else if (nv <= 4096) HXM_RESIDUAL(4, 16);
  else launch(residual_norm_stream_kernel<T>, 1024, 1);
#undef HXM_RESIDUAL
  return st;
}

// The matrices a [rows, cols] at lda and b at ldb (elements of eb bytes) share
// no element, as far as one span test or, for equal strides, their columns
// tell.
bool rows_disjoint(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows,
                   int64_t cols, int64_t eb) {
  return matrices_disjoint(reinterpret_cast<uintptr_t>(a), lda, reinterpret_cast<uintptr_t>(b),
                           ldb, rows, cols, cols, eb);
}

hxm_status check_norm(const char* which, const hxm_row_norm* n) {
  if (!n || n->kind < HXM_NORM_NONE || n->kind > HXM_NORM_LAYER)
    return fail(HXM_INVALID_ARG, "invalid-argument: residual_norm %s norm of kind %d", which,
                n ? n->kind : -1);
  if (n->kind == HXM_NORM_NONE && (n->gamma || n->beta))
    return fail(HXM_INVALID_ARG, "invalid-argument: residual_norm %s gamma or beta without a norm",
                which);
  if (n->kind != HXM_NORM_NONE && !(n->eps >= 0.0f))
    return fail(HXM_INVALID_ARG, "invalid-argument: residual_norm %s eps must be >= 0", which);
  return HXM_OK;
}

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_residual_norm_rows(
    const void* h, int64_t ldh, const void* x, int64_t ldx, const hxm_row_norm* post,
    const void* gate, int64_t ldg, int64_t gate_rows, float block_scale, float residual_scale,
    const hxm_row_norm* pre, void* y, int64_t ldy, void* z, int64_t ldz, int64_t rows,
    int64_t cols, int32_t dtype, void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16 && dtype != HXM_F32)
    return fail(HXM_UNSUPPORTED_DTYPE,
                "unsupported-dtype: residual_norm takes f16, bf16 or f32 (got %d)", dtype);
  hxm_status st = check_norm("post", post);
  if (st == HXM_OK) st = check_norm("pre", pre);
  if (st != HXM_OK) return st;
  // 2^40 elements in a row or between rows keep every byte offset below 2^63.
  constexpr int64_t kMax = int64_t(1) << 40;
  if (rows < 0 || cols < 1 || cols > kMax || gate_rows < 0)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: residual_norm rows=%lld cols=%lld gate_rows=%lld",
                (long long)rows, (long long)cols, (long long)gate_rows);
  if (rows > INT32_MAX)
    return fail(HXM_UNSUPPORTED_SHAPE, "tile-alignment: residual_norm rows=%lld too many",
                (long long)rows);
  const bool has_z = pre->kind != HXM_NORM_NONE;
  if (rows > 0 && (!h || !x || !y || (has_z && !z) || (gate_rows > 0 && !gate)))
    return fail(HXM_INVALID_ARG, "invalid-argument: residual_norm null tensor");
  if ((z && !has_z) || (gate && gate_rows == 0))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: residual_norm z without a norm, or a gate of no rows");
  auto bad_ld = [&](int64_t ld) { return ld < cols || ld > kMax; };
  if (bad_ld(ldh) || bad_ld(ldx) || bad_ld(ldy) || (has_z && bad_ld(ldz)) ||
      (gate_rows > 0 && bad_ld(ldg)))
    return fail(HXM_INVALID_ARG,
                "invalid-argument: residual_norm leading dimension below cols=%lld",
                (long long)cols);
  if (gate_rows > 0 && rows % gate_rows != 0)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: residual_norm %lld rows under %lld gate rows", (long long)rows,
                (long long)gate_rows);
  if (rows > 0) {
    const int64_t eb = dtype_bytes(dtype);
    const void* in[2] = {h, x};
    const int64_t ldi[2] = {ldh, ldx};
    void* out[2] = {y, z};
    const int64_t ldo[2] = {ldy, ldz};
    for (int o = 0; o < (has_z ? 2 : 1); ++o)
      for (int i = 0; i < 2; ++i) {
        const bool same = out[o] == in[i] && (ldo[o] == ldi[i] || rows == 1);
        if (!same && !rows_disjoint(out[o], ldo[o], in[i], ldi[i], rows, cols, eb))
          return fail(HXM_INVALID_ARG,
                      "invalid-argument: residual_norm an output overlaps an input without "
                      "being it");
      }
    if (has_z && !rows_disjoint(y, ldy, z, ldz, rows, cols, eb))
      return fail(HXM_INVALID_ARG, "invalid-argument: residual_norm y and z overlap");
  }
  if ((st = require_device(nullptr)) != HXM_OK) return st;
  if (rows == 0) return ok();
  const ResidualArgs a{h, x, y, has_z ? z : nullptr, gate, ldh, ldx, ldy, ldz, ldg, cols,
                       NormArgs{post->kind, post->eps, post->gamma, post->beta},
                       NormArgs{pre->kind, pre->eps, pre->gamma, pre->beta},
                       block_scale, residual_scale, static_cast<uint32_t>(rows),
                       gate_rows > 1 ? static_cast<uint32_t>(rows / gate_rows) : 0u};
  switch (dtype) {
    case HXM_F16: return launch_residual<_Float16>(a, as_stream(stream));
    case HXM_BF16: return launch_residual<__bf16>(a, as_stream(stream));
    default: return launch_residual<float>(a, as_stream(stream));
  }
}
