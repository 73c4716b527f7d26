// Low-rank adapters of many requests beside a projection they share:
//   out[m] = y[m] + scale[a] * (x[m] A[a]^T) B[a]^T,  a = index[m].
//
// The first launch makes t = x A^T, R values a row, split over K (fp32 partial
// planes in the stream's workspace, added in order); the last makes t B^T and adds it to
// y in one read and one write of y.  Bound by memory: y twice, x once, and R * (K + N)
// elements of each adapter in use, against 2 R operations for each element of x and y.
//
// Both work on tiles of 16 rows, any order of adapters among them: a tile's MFMAs
// run once for each adapter it holds, all its rows as one operand, and a row
// keeps the results of its own adapter alone (chosen, not multiplied by zero: what
// another adapter's weights hold does not reach it).
//
// Few rows are a matter of latency and of reading many adapters: each adapter of a tile is
// a workgroup of the first launch and a wave of the second, every load under way at once.
// Many rows mostly share one adapter per tile: there a tile is 64 rows, whose waves share
// the adapter's weights through LDS, read in whole rows, and a launch between makes the
// second operand once.
//
// 48 rows of 16 adapters, 4096 -> 4096, R 16: 9.8 us, two launches of 4.4 and 5.5.  2048
// rows of 4, 4096 -> 11008, R 64, bf16: 36.4, of them 10 the first launch, 4 the second,
// and 22 the last, which moves 90 MB of y and out (17 us at a large copy's rate).  With
// each wave reading its own operands of the weights and of y, 16 rows of 64 bytes an
// instruction, they were 19, 5 and 39.  2048 rows of 16 mixed adapters, 4096 -> 4096, R 16:
// 44, sixteen turns for each tile (52 before conversions and selects took two elements
// each).
//
// t enters the second product as two 16-bit halves, t = hi + lo: 22 bits of it
// in f16, 16 in bf16, where one would round t to the weights' 11 or 8.  Rows
// are scaled by a power of two first, which comes back in fp32 with the adapter's scale: in
// f16 the largest |t| goes to [2^14, 2^15), as high as it can, so that the smallest lo,
// 2^-24, is 2^-38 of it or less (22 bits of a rank down to 2^-17 of the row's largest; with the
// largest in [1/2, 1) lo was subnormal for nearly all of them, and a rank 2^-20 of the largest
// kept 5 bits).  bf16 has fp32's exponents and needs no room.
#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "hxm_internal.h"
#include "row_vec.h"

namespace hxm {

namespace {

constexpr int kRows = 16;   // rows of an MFMA operand
constexpr int kWaves = 4;
// Rows from which the form for many is taken (R 16, 4096 -> 4096: 256 rows of 4 adapters
// 10.8 us with it, 14.0 without; 512 rows of 16 mixed adapters 22.8 and 31).
constexpr int64_t kManyRows = 256;

struct LoraArgs {
  const void* y;
  const void* x;
  const void* A;
  const void* B;
  void* out;
  float* t;        // [splits][M][R]
  void* halves;    // [M][2][R] of the rows' type, and
  float* factors;  // [M], for many rows
  const int32_t* index;
  const float* scale;
  int64_t ldy, ldx, ldo, K, N;
  int M, R, adapters, splits;
  int tiles;        // of 64 rows, of the last launch
  int k_per_split;  // a multiple of what a workgroup's waves take together
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

// The adapter of row m, -1 past the last row.
__device__ __forceinline__ int row_adapter(const LoraArgs& a, int m) {
  return m < a.M ? a.index[m] : -1;
}

// 32-wide steps of K whose loads a wave has under way together.
constexpr int shrink_steps(int rt) { return rt <= 1 ? 8 : rt <= 4 ? 4 : 2; }

// t of 16 rows, RT * 16 ranks, a part of K.  Workgroup (tile, y, ranks and part) takes the
// tile's adapter y in the order of their first rows (a tile has no more of them than rows, nor
// the grid fewer); its waves take steps of K in turn and are summed in order.
template <typename T, int RT>
__global__ __launch_bounds__(kWaves * 64) void lora_shrink_kernel(LoraArgs a) {
  using V = typename Mma<T>::V;
  constexpr int U = shrink_steps(RT);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int m0 = blockIdx.x * kRows;
  const int split = blockIdx.z % a.splits, r0 = blockIdx.z / a.splits * (RT * 16);
  const int mine = row_adapter(a, m0 + c);
  uint64_t todo = __ballot(static_cast<uint32_t>(mine) < static_cast<uint32_t>(a.adapters)) &
                  0xffffull;
  int row0 = 0, id = -1;
  uint64_t same = 0;
  for (int y = 0; todo && y <= static_cast<int>(blockIdx.y); ++y) {
    row0 = __builtin_ctzll(todo);
    id = __builtin_amdgcn_readlane(mine, row0);
    same = __ballot(mine == id);
    todo &= ~same;
    if (y < static_cast<int>(blockIdx.y)) same = 0;
  }
  if (!same) return;
  const int64_t k_begin = static_cast<int64_t>(split) * a.k_per_split;
  const int64_t k_end = min(a.K, k_begin + a.k_per_split);
  __shared__ __align__(16) float sum[kWaves][RT * 16][kRows + 1];
  // Rows of another adapter are read as row0; their results are not kept.
  const T* x = static_cast<const T*>(a.x) +
               static_cast<int64_t>(m0 + (mine == id ? c : row0)) * a.ldx;
  const T* A = static_cast<const T*>(a.A) + static_cast<int64_t>(id) * a.R * a.K;
  v4f32 acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = v4f32(0.0f);
  for (int64_t k0 = k_begin + wave * (32 * U); k0 < k_end; k0 += 32 * U * kWaves) {
    v4u32_t xv[U], av[U][RT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + 32 * u + 8 * g;
      const int64_t kc = k < k_end ? k : 0;
      xv[u] = *reinterpret_cast<const any4*>(x + kc);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        av[u][r] = *reinterpret_cast<const any4*>(
            A + static_cast<int64_t>(min(r0 + r * 16 + c, a.R - 1)) * a.K + kc);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = k0 + 32 * u + 8 * g < k_end;
      xv[u] = in ? xv[u] : v4u32_t(0u);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        av[u][r] = in ? av[u][r] : v4u32_t(0u);
        acc[r] = Mma<T>::run(__builtin_bit_cast(V, av[u][r]), __builtin_bit_cast(V, xv[u]),
                             acc[r]);
      }
    }
  }
  // acc[r][i]: rank 16r + 4g + i of row c.
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[wave][16 * r + 4 * g + i][c] = acc[r][i];
  __syncthreads();
  const int ranks = min(RT * 16, a.R - r0);
  for (int e = threadIdx.x; e < kRows * ranks; e += kWaves * 64) {
    const int row = e / ranks, r = e - row * ranks;
    if (!((same >> row) & 1)) continue;
    const float v = (sum[0][r][row] + sum[1][r][row]) + (sum[2][r][row] + sum[3][r][row]);
    a.t[(static_cast<int64_t>(split) * a.M + m0 + row) * a.R + r0 + r] = v;
  }
}

// 2^-ex takes a row's largest |t|, top, to [2^14, 2^15) in f16 (hi of at most 2^15 stays
// finite) and to [1/2, 1) in bf16; 0, infinities and NaN stay as they are.
template <typename T>
__device__ __forceinline__ int row_exponent(float top) {
  constexpr int kUp = std::is_same<T, _Float16>::value ? 15 : 0;
  return top > 0.0f && top < __builtin_huge_valf() ? __builtin_amdgcn_frexp_expf(top) - kUp : 0;
}
template <typename T>
__device__ __forceinline__ void split_halves(float v, T* hi, T* lo) {
  *hi = fromf<T>(v);
  // An infinite or NaN hi needs no remainder (it would be NaN).
  const float rest = v - tof(*hi);
  *lo = fromf<T>(rest == rest ? rest : 0.0f);
}

// t of a row, ranks 32 s + 8 g .. + 8, as two halves scaled by 2^-ex, and the factor
// that takes the product back: the adapter's scale times 2^ex.
template <typename T, int KS>
struct RowFactors {
  typename Mma<T>::V hi[KS], lo[KS];
  float factor;
};
// For row m0 + c.  The planes are added in order, P of their loads under way at once (past
// the last plane, its own again, which is not added).
template <typename T, int KS>
__device__ __forceinline__ void load_factors(const LoraArgs& a, int m0, int id, bool live, int g,
                                             int c, RowFactors<T, KS>& f) {
  constexpr int P = KS >= 4 ? 1 : 4 / KS;
  float t[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) t[s][e] = 0.0f;
  auto inside = [&](int s) { return live && 32 * s + 8 * g < a.R; };
  if (a.adapters > 0)
    for (int p0 = 0; p0 < a.splits; p0 += P) {
      v4f32 v[P][KS][2];
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          // A row without an adapter, or ranks past the last, read the plane's start.
          const int64_t at =
              static_cast<int64_t>(min(p0 + i, a.splits - 1)) * a.M * a.R +
              (inside(s) ? static_cast<int64_t>(m0 + c) * a.R + 32 * s + 8 * g : 0);
          const v4f32* tp = reinterpret_cast<const v4f32*>(a.t + at);
          v[i][s][0] = tp[0], v[i][s][1] = tp[1];
        }
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (p0 + i < a.splits)
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) t[s][e] += inside(s) ? v[i][s][e / 4][e % 4] : 0.0f;
    }
  float top = 0.0f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(t[s][e]));
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const int ex = row_exponent<T>(top);
  f.factor = live ? __builtin_amdgcn_ldexpf(a.scale ? a.scale[id] : 1.0f, ex) : 0.0f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      T hi, lo;
      split_halves(__builtin_amdgcn_ldexpf(t[s][e], -ex), &hi, &lo);
      f.hi[s][e] = hi, f.lo[s][e] = lo;
    }
}

// Many rows: t of 64 rows, a part of K; workgroup (tile, y, part) takes the tile's adapters
// y, y + ways, .. in the order of their first rows.  A wave's 16 rows of x stay in
// registers, 256 of K at a time; 16 RT ranks of an adapter's A lie in LDS for all four
// waves, read in whole rows.
constexpr int kManyTile = kRows * kWaves;
constexpr int kManyK = 256;
template <typename T, int RT, int NC>
__global__ __launch_bounds__(kWaves * 64) void lora_shrink_many_kernel(LoraArgs a) {
  using V = typename Mma<T>::V;
  constexpr int U = kManyK / 32, CHUNKS = 2 * RT;  // 16-byte chunks of A a thread brings
  constexpr int PITCH = kManyK / 8 + 1;            // of a rank's row in LDS, chunks
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int m0 = blockIdx.x * kManyTile, ways = gridDim.y;
  const int all = row_adapter(a, m0 + lane);
  const int64_t k_begin = static_cast<int64_t>(blockIdx.z) * a.k_per_split;
  const int64_t k_end = min(a.K, k_begin + a.k_per_split);
  const T* x = static_cast<const T*>(a.x) +
               static_cast<int64_t>(min(m0 + wave * kRows + c, a.M - 1)) * a.ldx;
  __shared__ __align__(16) v4u32_t la[RT * 16 * PITCH];
  v4f32 acc[NC][RT];
#pragma unroll
  for (int h = 0; h < NC; ++h)
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[h][r] = v4f32(0.0f);
  uint64_t done = 0;
  for (int64_t k0 = k_begin; k0 < k_end; k0 += kManyK) {
    v4u32_t xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + 32 * u + 8 * g;
      xv[u] = *reinterpret_cast<const any4*>(x + (k < k_end ? k : 0));
      xv[u] = k < k_end ? xv[u] : v4u32_t(0u);
    }
    const int mine = __shfl(all, wave * kRows + c, 64);
    int seen = 0;
    for (uint64_t todo = __ballot(static_cast<uint32_t>(all) < static_cast<uint32_t>(a.adapters));
         todo; ++seen) {
      const int id = __builtin_amdgcn_readlane(all, __builtin_ctzll(todo));
      const uint64_t same = __ballot(all == id);
      todo &= ~same;
      if (seen % ways != static_cast<int>(blockIdx.y)) continue;
      done |= same;
      const bool hit = mine == id;
#pragma unroll
      for (int h = 0; h < NC; ++h) {
        if (16 * RT * h >= a.R) break;
        v4u32_t st[CHUNKS];
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int q = i * (kWaves * 64) + threadIdx.x, col = q % (kManyK / 8);
          const int rank = min(16 * RT * h + q / (kManyK / 8), a.R - 1);
          const int64_t k = k0 + 8 * col;
          st[i] = *reinterpret_cast<const any4*>(
              static_cast<const T*>(a.A) + (static_cast<int64_t>(id) * a.R + rank) * a.K +
              (k < k_end ? k : 0));
          st[i] = k < k_end ? st[i] : v4u32_t(0u);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int q = i * (kWaves * 64) + threadIdx.x;
          la[q / (kManyK / 8) * PITCH + q % (kManyK / 8)] = st[i];
        }
        __syncthreads();
        if ((same >> (kRows * wave)) & 0xffff) {
          v4f32 d[RT];
#pragma unroll
          for (int r = 0; r < RT; ++r) d[r] = acc[h][r];
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < RT; ++r)
              d[r] = Mma<T>::run(__builtin_bit_cast(V, la[(16 * r + c) * PITCH + 4 * u + g]),
                                 __builtin_bit_cast(V, xv[u]), d[r]);
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[h][r] = hit ? d[r] : acc[h][r];
        }
      }
    }
    if (!done) return;
  }
  // acc[h][r][i]: rank 16 (RT h + r) + 4g + i of row c.
  if (!((done >> (kRows * wave + c)) & 1)) return;
  float* t = a.t + (static_cast<int64_t>(blockIdx.z) * a.M + m0 + wave * kRows + c) * a.R;
#pragma unroll
  for (int h = 0; h < NC; ++h)
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int rank = 16 * (RT * h + r) + 4 * g;
      if (rank < a.R) *reinterpret_cast<v4f32*>(t + rank) = acc[h][r];
    }
}

// Many rows: each row's factors made once, for the many workgroups that read them: halves
// [M][hi, lo][R] and the factors [M].  A row is LANES neighbouring lanes, four ranks
// each; the planes are added in order, eight loads under way at once (past the last plane,
// its own again, which is not added).
template <typename T, int LANES>
__global__ __launch_bounds__(256) void lora_halves_kernel(LoraArgs a) {
  constexpr int P = 8;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  const int m = static_cast<int>(min<int64_t>(at, a.M - 1));
  const int r = threadIdx.x % LANES * 4, id = a.index[m];
  const bool live = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.adapters);
  const bool in = live && at < a.M && r < a.R;
  const float* tp = a.t + (in ? static_cast<int64_t>(m) * a.R + r : 0);
  v4f32 t = v4f32(0.0f);
  for (int p0 = 0; p0 < a.splits; p0 += P) {
    v4f32 v[P];
#pragma unroll
    for (int i = 0; i < P; ++i)
      v[i] = *reinterpret_cast<const v4f32*>(
          tp + static_cast<int64_t>(min(p0 + i, a.splits - 1)) * a.M * a.R);
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (p0 + i < a.splits) t += v[i];
  }
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = in ? fmaxf(top, fabsf(t[e])) : 0.0f;
#pragma unroll
  for (int i = LANES / 2; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
  if (!in) return;
  const int ex = row_exponent<T>(top);
  typedef T half4 __attribute__((ext_vector_type(4)));
  half4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    T h, l;
    split_halves(__builtin_amdgcn_ldexpf(t[e], -ex), &h, &l);
    hi[e] = h, lo[e] = l;
  }
  T* halves = static_cast<T*>(a.halves) + static_cast<int64_t>(m) * 2 * a.R + r;
  *reinterpret_cast<half4*>(halves) = hi;
  *reinterpret_cast<half4*>(halves + a.R) = lo;
  if (r == 0) a.factors[m] = __builtin_amdgcn_ldexpf(a.scale ? a.scale[id] : 1.0f, ex);
}
// A row's factors as lora_halves_kernel left them (zeros past the last rank; a row
// without an adapter: whatever is there, and not used).
template <typename T, int KS>
__device__ __forceinline__ void load_halves(const LoraArgs& a, int m, int g,
                                            RowFactors<T, KS>& f) {
  using V = typename Mma<T>::V;
  const int row = min(m, a.M - 1);
  const T* halves = static_cast<const T*>(a.halves) + static_cast<int64_t>(row) * 2 * a.R;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int r = 32 * s + 8 * g;
    const V hi = *reinterpret_cast<const V*>(halves + (r < a.R ? r : 0));
    const V lo = *reinterpret_cast<const V*>(halves + a.R + (r < a.R ? r : 0));
    f.hi[s] = r < a.R ? hi : V(T(0));
    f.lo[s] = r < a.R ? lo : V(T(0));
  }
  f.factor = a.factors[row];
}

// Rows r of B (columns of the output) as the left operand of 32 columns: product
// u, row c is column 8 (c / 4) + 4u + c % 4, so that a lane ends with 8 neighbouring
// columns of one row.
template <typename T, int KS>
__device__ __forceinline__ void load_b(const LoraArgs& a, int id, int n0, int u, int g, int c,
                                       v4u32_t (&w)[KS]) {
  const int64_t n = min(a.N - 1, static_cast<int64_t>(n0 + 8 * (c >> 2) + 4 * u + (c & 3)));
  const T* B = static_cast<const T*>(a.B) + (static_cast<int64_t>(id) * a.N + n) * a.R;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int r = 32 * s + 8 * g;
    w[s] = *reinterpret_cast<const any4*>(B + (r < a.R ? r : 0));
    if (r >= a.R) w[s] = v4u32_t(0u);
  }
}
template <typename T, int KS>
__device__ __forceinline__ v4f32 times_b(const v4u32_t (&w)[KS], const RowFactors<T, KS>& f) {
  using V = typename Mma<T>::V;
  v4f32 d = v4f32(0.0f);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    d = Mma<T>::run(__builtin_bit_cast(V, w[s]), f.hi[s], d);
    d = Mma<T>::run(__builtin_bit_cast(V, w[s]), f.lo[s], d);
  }
  return d;
}
// Eight columns n .. of row m: y + factor * d, `left` of them inside.
template <typename T>
__device__ __forceinline__ RawVec<T> load_y(const LoraArgs& a, int m, int n, int left) {
  const T* y = static_cast<const T*>(a.y) + m * a.ldy + n;
  return left >= 8 ? load_any(y) : load_tail(y, 0, left, T(0));
}
template <typename T>
__device__ __forceinline__ void store_out(const LoraArgs& a, int m, int n, int left, int id,
                                          RawVec<T> y, v4f32 d0, v4f32 d1, float factor) {
  if (id < 0 && a.out == a.y) return;
  if (id >= 0) {
    const bool live = id < a.adapters;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = e < 4 ? d0[e & 3] : d1[e & 3];
      y[e] = fromf<T>(live ? fmaf(factor, d, tof(y[e])) : __builtin_nanf(""));
    }
  }
  // Plain stores: the next operator reads them.
  T* out = static_cast<T*>(a.out) + m * a.ldo + n;
  if (left >= 8) *reinterpret_cast<AnyVec<T>*>(out) = y;
  else store_tail(out, 0, left, y);
}

// Few rows: workgroup (32 columns, 16 rows), wave w the tile's adapters w, w + 4, ..
// by first row, and their rows; rows without an adapter go to wave 0.
template <typename T, int KS>
__global__ __launch_bounds__(kWaves * 64) void lora_expand_few_kernel(LoraArgs a) {
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int m = blockIdx.y * kRows + c, n0 = blockIdx.x * 32;
  const int mine = row_adapter(a, m);
  const bool live = static_cast<uint32_t>(mine) < static_cast<uint32_t>(a.adapters);
  constexpr int PER = kRows / kWaves;
  int ids[PER], count = 0, seen = 0;
  bool here = wave == 0 && !live && m < a.M;
  for (uint64_t todo = __ballot(live) & 0xffffull; todo; ++seen) {
    const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__ballot(mine == id);
    if (seen % kWaves != wave) continue;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i == count) ids[i] = id;
    ++count;
    here |= mine == id;
  }
  if (!__any(here)) return;
  // As many adapters' weights at once as 64 registers hold.
  constexpr int BATCH = KS >= 8 ? 1 : KS >= 4 ? 2 : PER;
  const int n = n0 + 8 * g;
  const int left = static_cast<int>(min<int64_t>(a.N - n, 8));
  RawVec<T> y;
  if (here && left > 0) y = load_y<T>(a, m, n, left);
  v4f32 acc[2] = {v4f32(0.0f), v4f32(0.0f)};
  RowFactors<T, KS> f;
#pragma unroll
  for (int i0 = 0; i0 < PER; i0 += BATCH) {
    v4u32_t w[BATCH][2][KS];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (i0 + i < count)
#pragma unroll
        for (int u = 0; u < 2; ++u) load_b<T, KS>(a, ids[i0 + i], n0, u, g, c, w[i][u]);
    if (i0 == 0)
      load_factors<T, KS>(a, blockIdx.y * kRows, mine, live && here, g, c, f);
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (i0 + i < count) {
        const bool hit = mine == ids[i0 + i];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const v4f32 d = times_b<T, KS>(w[i][u], f);
          acc[u] = hit ? d : acc[u];
        }
      }
  }
  if (here && left > 0) store_out<T>(a, m, n, left, mine, y, acc[0], acc[1], f.factor);
}

// Many rows: workgroup (64 rows, 32 NB columns), a wave 16 of the rows.  Everything a wave
// needs of y is under way before its adapters are known; the columns' rows of B, one
// block of memory, lie in LDS for the four waves, one adapter after another (the next
// one's on their way during the products), and a row's y takes its sum in place when its
// adapter's turn comes.
//
// Tiles are numbered down the rows and each XCD (workgroups go to them in turn) takes a run
// of them, so that its L2 holds the columns' weights.
constexpr int expand_blocks(int ks) { return ks <= 4 ? 4 : 2; }  // of 32 columns each
// Waves a SIMD that the compiler keeps its registers to.  R 256 needs two (2048 rows of 2,
// 4096 -> 4096: 61.4 us, 65.6 with one); up to R 128 the kernel takes no more registers than
// these leave it and one wave more or fewer is the same (R 64: 36.4 to 36.6 with
// 3, 4 or 5; R 128, 4096 -> 4096, 38.2 with 2 or 3).
constexpr int expand_waves(int ks) { return ks <= 2 ? 4 : ks <= 4 ? 3 : 2; }
template <typename T, int KS>
__global__ __launch_bounds__(kWaves * 64)
__attribute__((amdgpu_waves_per_eu(expand_waves(KS)))) void lora_expand_kernel(LoraArgs a) {
  using V = typename Mma<T>::V;
  constexpr int NB = expand_blocks(KS), COLS = 32 * NB;
  constexpr int ROW = 4 * KS, PITCH = ROW + 1;  // 16-byte chunks of a row of B, and its pitch
  constexpr int CHUNKS = COLS * ROW / (kWaves * 64);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const uint32_t run = gridDim.x / 8, turn = blockIdx.x % 8 * run + blockIdx.x / 8;
  const int col = turn / a.tiles;
  const int m0 = (turn - col * a.tiles) * kManyTile, m = m0 + wave * kRows + c;
  const int64_t n_begin = static_cast<int64_t>(col) * COLS;
  if (n_begin >= a.N) return;
  const int n0 = static_cast<int>(n_begin);
  const int all = row_adapter(a, m0 + lane);
  __shared__ __align__(16) v4u32_t lb[COLS * PITCH];
  // y and then out of a wave: whole rows to and from memory, operands to the products.
  constexpr int SEG = COLS / 8, SROW = SEG + 1, PER = 64 / SEG, NL = kRows / PER;
  __shared__ __align__(16) RawVec<T> ly[kWaves][kRows * SROW];
  const int lrow = lane / SEG, lcol = lane % SEG;
  const int left = static_cast<int>(min<int64_t>(a.N - (n0 + 8 * lcol), 8));
  RawVec<T> yl[NL];
  auto row_at = [&](int j) { return m0 + wave * kRows + PER * j + lrow; };
#pragma unroll
  for (int j = 0; j < NL; ++j)
    if (row_at(j) < a.M && left > 0) yl[j] = load_y<T>(a, row_at(j), n0 + 8 * lcol, left);
  uint64_t todo =
      __ballot(static_cast<uint32_t>(all) < static_cast<uint32_t>(a.adapters));
  // Zeros past the last rank and the last column, put there when the loads have arrived.
  auto inside = [&](int i) {
    const int q = i * (kWaves * 64) + threadIdx.x;
    return q % ROW * 8 < a.R && q / ROW < a.N - n0;
  };
  v4u32_t st[CHUNKS];
  auto fetch = [&](int id) {
    const T* B = static_cast<const T*>(a.B) + (static_cast<int64_t>(id) * a.N + n0) * a.R;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int q = i * (kWaves * 64) + threadIdx.x;
      st[i] = *reinterpret_cast<const any4*>(B + (inside(i) ? q / ROW * a.R + q % ROW * 8 : 0));
    }
  };
  // With ways, this workgroup's adapters alone, and the rows of no adapter in the first
  // one.
  const int way = blockIdx.y, ways = gridDim.y;
  uint64_t rows = ~0ull;
  if (ways > 1) {
    rows = way == 0 ? ~todo : 0ull;
    int seen = 0;
    for (uint64_t left_ids = todo; left_ids; ++seen) {
      const uint64_t same =
          __ballot(all == __builtin_amdgcn_readlane(all, __builtin_ctzll(left_ids)));
      left_ids &= ~same;
      if (seen % ways == way) rows |= same;
    }
    if (!rows) return;
    todo &= rows;
  }
  int id = -1;
  if (todo) {
    id = __builtin_amdgcn_readlane(all, __builtin_ctzll(todo));
    fetch(id);
  }
  RowFactors<T, KS> f;
  load_halves<T, KS>(a, m, g, f);
  const int mine = __shfl(all, wave * kRows + c, 64);
  RawVec<T> y[NB];
  auto swap_in = [&] {
#pragma unroll
    for (int j = 0; j < NL; ++j) ly[wave][(PER * j + lrow) * SROW + lcol] = yl[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < NB; ++k) y[k] = ly[wave][c * SROW + 4 * k + g];
  };
  if (!todo) swap_in();
  for (bool first = true; todo; first = false) {
    const uint64_t same = __ballot(all == id);
    const bool hit = mine == id;
    todo &= ~same;
    if (!first) __syncthreads();
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int q = i * (kWaves * 64) + threadIdx.x;
      lb[q / ROW * PITCH + q % ROW] = inside(i) ? st[i] : v4u32_t(0u);
    }
    __syncthreads();
    if (todo) {
      id = __builtin_amdgcn_readlane(all, __builtin_ctzll(todo));
      fetch(id);
    }
    if (first) swap_in();
    if ((same >> (kRows * wave)) & 0xffff) {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        v4f32 d[2] = {v4f32(0.0f), v4f32(0.0f)};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            // Columns 8 (c / 4) + 4u + c % 4 of the 32: a lane ends with 8 neighbours.
            const V w = __builtin_bit_cast(
                V, lb[(32 * k + 8 * (c >> 2) + 4 * u + (c & 3)) * PITCH + 4 * s + g]);
            d[u] = Mma<T>::run(w, f.hi[s], d[u]);
            d[u] = Mma<T>::run(w, f.lo[s], d[u]);
          }
        typedef float v8f32 __attribute__((ext_vector_type(8)));
        v8f32 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(f.factor, d[e / 4][e % 4], tof(y[k][e]));
        // Conversions and selects of two elements each.
        const v4u32_t sum = __builtin_bit_cast(v4u32_t, __builtin_convertvector(v, RawVec<T>));
        y[k] = __builtin_bit_cast(RawVec<T>, hit ? sum : __builtin_bit_cast(v4u32_t, y[k]));
      }
    }
  }
  if (mine >= a.adapters)
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[k][e] = fromf<T>(__builtin_nanf(""));
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int k = 0; k < NB; ++k) ly[wave][c * SROW + 4 * k + g] = y[k];
  __builtin_amdgcn_wave_barrier();
  // Nontemporal, like the other row operators: 45 MB of them 2.8 us faster.
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const RawVec<T> v = ly[wave][(PER * j + lrow) * SROW + lcol];
    const int of = __shfl(all, wave * kRows + PER * j + lrow, 64);
    if (row_at(j) >= a.M || left <= 0 || (of < 0 && a.out == a.y) ||
        !((rows >> (wave * kRows + PER * j + lrow)) & 1))
      continue;
    T* out = static_cast<T*>(a.out) + row_at(j) * a.ldo + n0 + 8 * lcol;
    if (left >= 8) store_any(out, v);
    else store_tail(out, 0, left, v);
  }
}

template <typename T>
hxm_status launch_lora(LoraArgs a, hipStream_t stream) {
  const bool few = a.M < kManyRows;
  hxm_status st = HXM_OK;
  if (a.adapters > 0 && !few) {
    const int64_t tiles = ceil_div(a.M, kManyTile);
    // A tile's adapters go to workgroups of their own while there are CUs without any
    // (256 rows of one adapter a tile, R 16: 10.8 us, 13.5 with four a CU, most of which
    // find no adapter; 256 rows of 16 mixed ones 18.2 and 20.8).
    const dim3 grid(static_cast<unsigned>(tiles),
                    static_cast<unsigned>(std::max<int64_t>(
                        1, std::min<int64_t>(16, 256 / (tiles * a.splits)))),
                    static_cast<unsigned>(a.splits));
#define HXM_MANY(RT, NC) lora_shrink_many_kernel<T, RT, NC><<<grid, kWaves * 64, 0, stream>>>(a)
    if (a.R <= 16) HXM_MANY(1, 1);
    else if (a.R <= 32) HXM_MANY(2, 1);
    else if (a.R <= 64) HXM_MANY(4, 1);
    else if (a.R <= 128) HXM_MANY(4, 2);
    else HXM_MANY(4, 4);
#undef HXM_MANY
    if ((st = check_launch("lora shrink")) != HXM_OK) return st;
#define HXM_HALVES(LANES)                                                       \
  lora_halves_kernel<T, LANES><<<static_cast<unsigned>(ceil_div(a.M, 256 / LANES)), 256, 0, \
                                 stream>>>(a)
    if (a.R <= 16) HXM_HALVES(4);
    else if (a.R <= 32) HXM_HALVES(8);
    else if (a.R <= 64) HXM_HALVES(16);
    else if (a.R <= 128) HXM_HALVES(32);
    else HXM_HALVES(64);
#undef HXM_HALVES
    if ((st = check_launch("lora halves")) != HXM_OK) return st;
  } else if (a.adapters > 0) {
    // All adapters of a tile at once, each a workgroup.
    const dim3 grid(static_cast<unsigned>(ceil_div(a.M, kRows)), std::min(kRows, a.M),
                    static_cast<unsigned>(a.splits * ceil_div(a.R, 128)));
    if (a.R <= 16) lora_shrink_kernel<T, 1><<<grid, kWaves * 64, 0, stream>>>(a);
    else if (a.R <= 32) lora_shrink_kernel<T, 2><<<grid, kWaves * 64, 0, stream>>>(a);
    else if (a.R <= 64) lora_shrink_kernel<T, 4><<<grid, kWaves * 64, 0, stream>>>(a);
    else lora_shrink_kernel<T, 8><<<grid, kWaves * 64, 0, stream>>>(a);
    if ((st = check_launch("lora shrink")) != HXM_OK) return st;
  }
#define HXM_LORA_EXPAND(KS)                                                                    \
  do {                                                                                         \
    if (few) {                                                                                 \
      lora_expand_few_kernel<T, KS>                                                            \
          <<<dim3(static_cast<unsigned>(ceil_div(a.N, 32)),                                    \
                  static_cast<unsigned>(ceil_div(a.M, kRows))),                                \
             kWaves * 64, 0, stream>>>(a);                                                     \
    } else {                                                                                   \
      a.tiles = static_cast<int>(ceil_div(a.M, kManyTile));                                    \
      const int64_t groups =                                                                   \
          ceil_div(a.tiles * ceil_div(a.N, 32 * expand_blocks(KS)), 8) * 8;                    \
      if ((st = check_grid("lora expand", groups, kWaves * 64)) != HXM_OK) return st;          \
      /* Ways until two workgroups a CU (256 rows of 16 mixed adapters 18.2 us, 25.5        */ \
      /* without). */                                                                          \
      lora_expand_kernel<T, KS>                                                                \
          <<<dim3(static_cast<unsigned>(groups),                                               \
                  static_cast<unsigned>(std::max<int64_t>(                                     \
                      1, std::min<int64_t>(16, 512 / groups)))),                               \
             kWaves * 64, 0, stream>>>(a);                                                     \
    }                                                                                          \
  } while (0)
  if (a.R <= 32) HXM_LORA_EXPAND(1);
  else if (a.R <= 64) HXM_LORA_EXPAND(2);
  else if (a.R <= 128) HXM_LORA_EXPAND(4);
  else HXM_LORA_EXPAND(8);
#undef HXM_LORA_EXPAND
  return check_launch("lora expand");
}

// Rows of one set of launches: a t plane of at most 64 MiB, at most 2^15 tiles of 16 rows.
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
  constexpr int64_t kMax = INT32_MAX / 4, kMaxN = int64_t(1) << 28;
  if (M < 0 || N < 0 || K < 1 || adapters < 0 || R < 1)
    return fail(HXM_INVALID_ARG,
                "invalid-argument: lora_add M=%lld N=%lld K=%lld adapters=%lld R=%lld",
                (long long)M, (long long)N, (long long)K, (long long)adapters, (long long)R);
  if (K % 8 != 0 || R % 8 != 0 || R > 256)
    return fail(HXM_UNSUPPORTED_SHAPE,
                "tile-alignment: lora_add K=%lld and R=%lld must be multiples of 8, R at most 256",
                (long long)K, (long long)R);
  if (M > kMax || N > kMaxN || K > kMax || adapters > kMax)
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
  // Rows of one set of launches: their planes fit the workspace, their tiles of 64 rows and
  // 64 columns or more a grid.
  const int64_t piece =
      std::min({M, kLoraRows, (kLoraPlaneBytes / (R * 4)) & ~int64_t(15),
                kManyTile * ((int64_t(1) << 23) / ceil_div(N, 64))});
  // K split until about 512 workgroups, in 8 parts at most, each a step of all its waves
  // or more; many rows, tiles of 64, in 16 parts (2048 rows, 4096 -> 11008, R 64: 36.4 us with
  // 512 workgroups in sight, 37.6 with 256; 8192 rows, R 32: 56.4 and 63.8).
  const bool few = piece < kManyRows;
  const int64_t tiles = ceil_div(piece, few ? kRows : kManyTile);
  const int64_t step = few ? 32 * kWaves * shrink_steps(R <= 16 ? 1 : R <= 64 ? 4 : 8) : kManyK;
  const int64_t splits = std::min(std::min<int64_t>(few ? 8 : 16, ceil_div(512, tiles)),
                                  ceil_div(K, step));
  a.k_per_split = static_cast<int>(ceil_div(ceil_div(K, splits), step) * step);
  a.splits = static_cast<int>(ceil_div(K, a.k_per_split));
  void* ws = nullptr;
  const int64_t plane_bytes = a.splits * piece * R * 4, halves_bytes = piece * R * 4;
  if ((st = stream_workspace(as_stream(stream),
                             static_cast<size_t>(plane_bytes + halves_bytes + piece * 4), &ws,
                             kWsLayer)) != HXM_OK)
    return st;
  a.t = static_cast<float*>(ws);
  a.halves = static_cast<char*>(ws) + plane_bytes;
  a.factors = reinterpret_cast<float*>(static_cast<char*>(ws) + plane_bytes + halves_bytes);
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
