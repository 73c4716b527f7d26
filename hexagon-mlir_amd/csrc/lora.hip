// Low-rank adapters of many requests beside a projection they share:
//   out[m] = y[m] + scale[a] * (x[m] A[a]^T) B[a]^T,  a = index[m].
//
// Two launches.  The first makes t = x A^T, R values a row, split over K (fp32
// partial planes in the stream's workspace, added in order by the second); the
// second makes t B^T and adds it to y in one read and one write of y.  Bound by
// memory: y twice, x once, and R * (K + N) elements of each adapter in use,
// against 2 R operations for each element of x and y.
//
// Both work on tiles of 16 rows, any order of adapters among them: a tile's
// MFMAs run once for each adapter it holds, all 16 rows as one operand, and a
// row keeps the results of its own adapter alone (chosen, not multiplied by
// zero: what another adapter's weights hold does not reach it).  Few rows of
// many adapters cost what reading those adapters costs; a long run of one
// adapter one pass.
//
// t enters the second product as two 16-bit halves, t = hi + lo: 22 bits of it
// in f16, 16 in bf16, where one would round t to the weights' 11 or 8.  f16 rows
// are scaled by a power of two first, so that no t over- or underflows; it
// comes back in fp32 with the adapter's scale.
#include <algorithm>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kRows = 16;   // rows of a tile
constexpr int kWaves = 4;

struct LoraArgs {
  const void* y;
  const void* x;
  const void* A;
  const void* B;
  void* out;
  float* t;  // [splits][M][R]
  const int32_t* index;
  const float* scale;
  int64_t ldy, ldx, ldo, K, N;
  int M, R, adapters, splits;
  int k_per_split;  // a multiple of 32 * kWaves
  int n_per_group;  // columns of a workgroup of the second launch
};

template <typename T>
struct Mma;
template <>
struct Mma<_Float16> {
  typedef v8f16 V;
  static __device__ __forceinline__ v4f32 run(V a, V b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  typedef v8bf16 V;
  static __device__ __forceinline__ v4f32 run(V a, V b, v4f32 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));

// The adapter of this lane's row of the tile (lane % 16), -1 past the last row.
__device__ __forceinline__ int row_adapter(const LoraArgs& a, int m0, int c) {
  return m0 + c < a.M ? a.index[m0 + c] : -1;
}

// Workgroup (tile, j, split): t of the tile's rows under the adapter of row j,
// unless an earlier row has the same.  Its waves take 32 of K in turn.
template <typename T, int RT>
__global__ __launch_bounds__(kWaves * 64) void lora_shrink_kernel(LoraArgs a) {
  using V = typename Mma<T>::V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int m0 = blockIdx.x * kRows, j = blockIdx.y, split = blockIdx.z;
  const int mine = row_adapter(a, m0, c);
  const int id = __builtin_amdgcn_readlane(mine, j);
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.adapters)) return;
  const uint32_t same = static_cast<uint32_t>(__ballot(mine == id)) & 0xffffu;
  if (same & ((1u << j) - 1)) return;
  const bool hit = mine == id;

  const T* x = static_cast<const T*>(a.x) + static_cast<int64_t>(hit ? m0 + c : m0 + j) * a.ldx;
  const T* A = static_cast<const T*>(a.A) + static_cast<int64_t>(id) * a.R * a.K;
  v4f32 acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = v4f32(0.0f);
  const int64_t k_end = min(a.K, static_cast<int64_t>(split + 1) * a.k_per_split);
  for (int64_t k0 = static_cast<int64_t>(split) * a.k_per_split + wave * 32; k0 < k_end;
       k0 += 32 * kWaves) {
    const int64_t k = k0 + 8 * g;
    const bool in = k < a.K;
    v4u32_t xw = *reinterpret_cast<const any4*>(x + (in ? k : 0));
    if (!in) xw = v4u32_t(0u);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = min(r * 16 + c, a.R - 1);
      v4u32_t w = *reinterpret_cast<const any4*>(A + row * a.K + (in ? k : 0));
      if (!in) w = v4u32_t(0u);
      acc[r] = Mma<T>::run(__builtin_bit_cast(V, w), __builtin_bit_cast(V, xw), acc[r]);
    }
  }
  // acc[r][i]: rank 16r + 4g + i of row c.
  __shared__ __align__(16) float sum[kWaves][RT * 16][kRows + 1];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[wave][16 * r + 4 * g + i][c] = acc[r][i];
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * a.R; e += kWaves * 64) {
    const int row = e / a.R, r = e - row * a.R;
    if (!((same >> row) & 1)) continue;
    const float v = (sum[0][r][row] + sum[1][r][row]) + (sum[2][r][row] + sum[3][r][row]);
    a.t[(static_cast<int64_t>(split) * a.M + m0 + row) * a.R + r] = v;
  }
}

// Workgroup (columns, tile): 32 columns of 16 rows per wave and step.  KS: steps
// of 32 ranks.
template <typename T, int KS>
__global__ __launch_bounds__(kWaves * 64) void lora_expand_kernel(LoraArgs a) {
  using V = typename Mma<T>::V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int m0 = blockIdx.y * kRows, m = m0 + c;
  const int mine = row_adapter(a, m0, c);
  const bool live = static_cast<uint32_t>(mine) < static_cast<uint32_t>(a.adapters);

  // t of row c, ranks 32 s + 8 g ..+8, as hi + lo.
  V hi[KS], lo[KS];
  float factor = 0.0f;
  {
    float t[KS][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int r = 32 * s + 8 * g;
      const bool in = live && r < a.R;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[s][e] = 0.0f;
      if (in)
        for (int p = 0; p < a.splits; ++p) {
          const v4f32* tp = reinterpret_cast<const v4f32*>(
              a.t + (static_cast<int64_t>(p) * a.M + m) * a.R + r);
          const v4f32 u = tp[0], w = tp[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[s][e] += u[e], t[s][4 + e] += w[e];
        }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(t[s][e]));
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // Power of two that takes the row's largest |t| to [1/2, 1); 0, infinities
    // and NaN stay as they are.
    int ex = 0;
    if (top > 0.0f && top < __builtin_huge_valf()) ex = __builtin_amdgcn_frexp_expf(top);
    factor = live ? __builtin_amdgcn_ldexpf(a.scale ? a.scale[mine] : 1.0f, ex) : 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_ldexpf(t[s][e], -ex);
        hi[s][e] = fromf<T>(v);
        // An infinite or NaN hi needs no remainder (it would be NaN).
        const float rest = v - tof(hi[s][e]);
        lo[s][e] = fromf<T>(rest == rest ? rest : 0.0f);
      }
  }

  const int n_end = static_cast<int>(
      min(a.N, static_cast<int64_t>(blockIdx.x + 1) * a.n_per_group));
  for (int n0 = blockIdx.x * a.n_per_group + wave * 32; n0 < n_end; n0 += 32 * kWaves) {
    v4f32 acc[2] = {v4f32(0.0f), v4f32(0.0f)};
    // The tile's adapters, each at its first row.
    uint64_t todo = __ballot(live) & 0xffffull;
    while (todo) {
      const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      const bool hit = mine == id;
      todo &= ~__ballot(hit);
      const T* B = static_cast<const T*>(a.B) + static_cast<int64_t>(id) * a.N * a.R;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        v4f32 d = v4f32(0.0f);
        // Row c of the product is column 8 (c / 4) + 4u + c % 4, so that a lane
        // ends with 8 neighbouring columns.
        const int64_t n = min(a.N - 1, static_cast<int64_t>(n0 + 8 * (c >> 2) + 4 * u + (c & 3)));
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int r = 32 * s + 8 * g;
          v4u32_t w = *reinterpret_cast<const any4*>(B + n * a.R + (r < a.R ? r : 0));
          if (r >= a.R) w = v4u32_t(0u);
          d = Mma<T>::run(__builtin_bit_cast(V, w), hi[s], d);
          d = Mma<T>::run(__builtin_bit_cast(V, w), lo[s], d);
        }
        acc[u] = hit ? d : acc[u];
      }
    }
    if (m >= a.M) continue;
    const int n = n0 + 8 * g;
    if (n >= n_end) continue;
    if (mine < 0 && a.out == a.y) continue;
    const T* y = static_cast<const T*>(a.y) + m * a.ldy + n;
    T* out = static_cast<T*>(a.out) + m * a.ldo + n;
    const int left = n_end - n;
    RawVec<T> v = left >= 8 ? load_any(y) : load_tail(y, 0, left, T(0));
    if (mine >= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = e < 4 ? acc[0][e & 3] : acc[1][e & 3];
        v[e] = fromf<T>(live ? fmaf(factor, d, tof(v[e])) : __builtin_nanf(""));
      }
    }
    if (left >= 8) store_any(out, v);
    else store_tail(out, 0, left, v);
  }
}

template <typename T>
hxm_status launch_lora(const LoraArgs& a, hipStream_t stream) {
  const int tiles = static_cast<int>(ceil_div(a.M, kRows));
  hxm_status st = HXM_OK;
  const dim3 gs(tiles, std::min(kRows, a.M), a.splits);
  if (a.adapters > 0) {
#define HXM_LORA_SHRINK(RT) lora_shrink_kernel<T, RT><<<gs, kWaves * 64, 0, stream>>>(a)
    if (a.R <= 16) HXM_LORA_SHRINK(1);
    else if (a.R <= 32) HXM_LORA_SHRINK(2);
    else if (a.R <= 64) HXM_LORA_SHRINK(4);
    else if (a.R <= 128) HXM_LORA_SHRINK(8);
    else HXM_LORA_SHRINK(16);
#undef HXM_LORA_SHRINK
    if ((st = check_launch("lora shrink")) != HXM_OK) return st;
  }
  const dim3 ge(static_cast<unsigned>(ceil_div(a.N, a.n_per_group)), tiles);
#define HXM_LORA_EXPAND(KS) lora_expand_kernel<T, KS><<<ge, kWaves * 64, 0, stream>>>(a)
  if (a.R <= 32) HXM_LORA_EXPAND(1);
  else if (a.R <= 64) HXM_LORA_EXPAND(2);
  else if (a.R <= 128) HXM_LORA_EXPAND(4);
  else HXM_LORA_EXPAND(8);
#undef HXM_LORA_EXPAND
  return check_launch("lora expand");
}

// Rows of one pair of launches: a t plane of at most 64 MiB, at most 2^15 tiles.
constexpr int64_t kLoraPlaneBytes = int64_t(64) << 20, kLoraRows = int64_t(1) << 19;

}  // namespace
}  // namespace hxm

using namespace hxm;

extern "C" hxm_status hxm_lora_add(const void* y, int64_t ldy, const void* x, int64_t ldx,
                                   const void* A, const void* B, int64_t adapters, int64_t R,
                                   const int32_t* index, const float* scale, void* out,
                                   int64_t ldo, int64_t M, int64_t N, int64_t K, int32_t dtype,
                                   void* stream) {
  if (dtype != HXM_F16 && dtype != HXM_BF16)
    return fail(HXM_UNSUPPORTED_DTYPE, "unsupported-dtype: lora_add takes f16 or bf16 (got %d)",
                dtype);
  constexpr int64_t kMax = INT32_MAX / 4;
  if (M < 0 || N < 0 || K < 1 || adapters < 0 || R < 1)
    return fail(HXM_INVALID_ARG, "invalid-argument: lora_add M=%lld N=%lld K=%lld adapters=%lld R=%lld",
                (long long)M, (long long)N, (long long)K, (long long)adapters, (long long)R);
  if (K % 8 != 0 || R % 8 != 0 || R > 256)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: lora_add K=%lld and R=%lld must be multiples of 8, R at most 256",
                (long long)K, (long long)R);
  if (M > kMax || N > kMax || K > kMax || adapters > kMax)
    return fail(HXM_UNSUPPORTED_SHAPE, "tile-alignment: lora_add M=%lld N=%lld K=%lld too large",
                (long long)M, (long long)N, (long long)K);
  if (!stride_ok(ldy) || !stride_ok(ldx) || !stride_ok(ldo) || ldy < N || ldx < K || ldo < N)
    return fail(HXM_INVALID_ARG, "invalid-argument: lora_add leading dimensions %lld, %lld, %lld",
                (long long)ldy, (long long)ldx, (long long)ldo);
  if (M > 0 && N > 0 && (!y || !x || !out || !index || (adapters > 0 && (!A || !B))))
    return fail(HXM_INVALID_ARG, "invalid-argument: lora_add null tensor");
  if (M > 0 && N > 0) {
    const uintptr_t o = reinterpret_cast<uintptr_t>(out), yy = reinterpret_cast<uintptr_t>(y),
                    xx = reinterpret_cast<uintptr_t>(x);
    const bool same = out == y && (ldo == ldy || M == 1);
    if ((!same && !matrices_disjoint(o, ldo, yy, ldy, M, N, N, 2)) ||
        !matrices_disjoint(o, ldo, xx, ldx, M, N, K, 2))
      return fail(HXM_INVALID_ARG,
                  "invalid-argument: lora_add out overlaps y (without being it) or x");
  }
  hxm_status st = require_device(nullptr);
  if (st != HXM_OK) return st;
  if (M == 0 || N == 0) return ok();
  LoraArgs a{};
  a.A = A, a.B = B, a.scale = scale;
  a.ldy = ldy, a.ldx = ldx, a.ldo = ldo, a.K = K, a.N = N;
  a.R = static_cast<int>(R), a.adapters = static_cast<int>(adapters);
  const int64_t piece = std::min(std::min(M, kLoraRows), (kLoraPlaneBytes / (R * 4)) & ~int64_t(15));
  // K split until about 512 workgroups, each with 512 of K or more.
  const int64_t tiles = ceil_div(piece, kRows);
  int64_t splits = std::max<int64_t>(1, std::min(ceil_div(512, tiles), K / 512));
  const int64_t step = 32 * kWaves;
  a.k_per_split = static_cast<int>(ceil_div(ceil_div(K, splits), step) * step);
  a.splits = static_cast<int>(ceil_div(K, a.k_per_split));
  // Columns of a workgroup: as few as keep 1024 workgroups busy.
  const int64_t want = std::max<int64_t>(1, 1024 / tiles);
  a.n_per_group = static_cast<int>(ceil_div(ceil_div(N, want), step) * step);
  void* ws = nullptr;
  if (adapters > 0 &&
      (st = stream_workspace(as_stream(stream), static_cast<size_t>(a.splits * piece * R * 4), &ws,
                             kWsLayer)) != HXM_OK)
    return st;
  a.t = static_cast<float*>(ws);
  for (int64_t m = 0; m < M; m += piece) {
    a.M = static_cast<int>(std::min(piece, M - m));
    a.y = static_cast<const char*>(y) + m * ldy * 2;
    a.x = static_cast<const char*>(x) + m * ldx * 2;
    a.out = static_cast<char*>(out) + m * ldo * 2;
    a.index = index + m;
    st = dtype == HXM_F16 ? launch_lora<_Float16>(a, as_stream(stream))
                          : launch_lora<__bf16>(a, as_stream(stream));
    if (st != HXM_OK) return st;
  }
  return ok();
}
