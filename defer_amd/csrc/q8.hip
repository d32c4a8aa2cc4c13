// q8.hip -- the 8-bit operators: rows to codes, the norm that leaves codes,
// the product of codes, the cache in codes and the attention over it.
//
// Sums of code products are exact in 32-bit integers (v_mfma_i32_16x16x64_i8),
// so they have no order; every other sum has one that depends on its own row
// only. Nothing here keeps state, allocates or waits.
#include "q8_attn.h"

#include <algorithm>
#include <type_traits>

namespace q8 {

namespace {

struct NormArgs {
  const void *x, *r, *w;
  int64_t xs, rs, zs;
  void* z;
  int8_t* codes;
  float* scale;
  uint32_t n;
  float eps;
};

// One workgroup per row: z = x + r, sum z^2, max |z w|, then the codes. The
// squares and products are formed in 64 bits (24 + 24 bits: the products
// exactly), so that codes are those of the formula and not of a rounding;
// memory hides that (2048 x 4096: 5.0 M vector instructions, 8 of the 15.6 us at 4
// cycles each). Bound by memory: 2048 x 4096 bf16 with residual, 58.7 MB in
// 15.6 us (3.8 TB/s; a large copy moves 4.7); codes alone of 2047 x 14336 f32, 147
// MB in 37.0 us (4.0 TB/s); 1 x 576: 2.6 us, all latency.
struct RowSum {
  double ss = 0.0, top = 0.0;
  float bad = 0.0f;  // NaN once a value is not finite
  template <bool NORM>
  __device__ __forceinline__ double add(float v, float w) {
    const double d = (double)v, y = NORM ? d * (double)w : d;
    if (NORM) ss = fma(d, d, ss);
    top = fmax(top, fabs(y));
    bad = fmaf(v, 0.0f, bad);
    if (NORM) bad = fmaf(w, 0.0f, bad);
    return y;
  }
  // over the workgroup: lanes by halves, waves in order
  __device__ __forceinline__ void join() {
    __shared__ double s_ss[16], s_top[16];
    __shared__ float s_bad[16];
    ss = wave_add(ss);
    top = wave_max(top);
    bad = wave_add(bad);
    const uint32_t w = threadIdx.x / WAVE, waves = blockDim.x / WAVE;
    if (threadIdx.x % WAVE == 0) {
      s_ss[w] = ss;
      s_top[w] = top;
      s_bad[w] = bad;
    }
    __syncthreads();
    ss = s_ss[0];
    top = s_top[0];
    bad = s_bad[0];
    for (uint32_t i = 1; i < waves; ++i) {
      ss += s_ss[i];
      top = fmax(top, s_top[i]);
      bad += s_bad[i];
    }
  }
};

// Threads take 16 bytes of values in turn, as k_rows_vec's do, so that the sum
// of squares has the same order in both.
template <class T, bool NORM, int BLOCK>
__global__ __launch_bounds__(BLOCK) void k_rows(NormArgs a) {
  constexpr uint32_t V = 16 / sizeof(T);
  const size_t row = blockIdx.x;
  const uint32_t n = a.n;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.rs : nullptr;
  const T* w = static_cast<const T*>(a.w);
  T* z = a.z ? static_cast<T*>(a.z) + row * a.zs : nullptr;
  auto value = [&](uint32_t i) { return NORM && r ? (T)((float)x[i] + (float)r[i]) : x[i]; };
  RowSum s;
  for (uint64_t i0 = V * threadIdx.x; i0 < n; i0 += V * BLOCK)
#pragma unroll
    for (uint32_t e = 0; e < V; ++e)
      if (i0 + e < n) s.add<NORM>((float)value((uint32_t)i0 + e), NORM ? (float)w[i0 + e] : 1.0f);
  s.join();
  const double inv = NORM ? 1.0 / sqrt(s.ss / n + (double)a.eps) : 1.0;
  const float scale = scale_of(s.top * inv, isnan(s.bad));
  if (threadIdx.x == 0) a.scale[row] = scale;
  const double f = NORM && scale > 0.0f ? inv / (double)scale : 0.0;
  const Coder code(scale);
  int8_t* c = a.codes + row * (size_t)n;
  for (uint64_t i = threadIdx.x; i < n; i += BLOCK) {
    const T v = value((uint32_t)i);
    c[i] = (int8_t)(NORM ? (f > 0.0 ? (int)rint((double)(float)v * (double)(float)w[i] * f) : 0) : code((float)v));
    if (NORM && z) z[i] = v;
  }
}

// The same where every row is a multiple of 16 bytes apart and long: 16-byte
// loads, and the row stays in registers between its two passes (2048 x 4096:
// 34 us through k_rows, 15.6 so).
template <class T, bool NORM, int BLOCK, int C>
__global__ __launch_bounds__(BLOCK) void k_rows_vec(NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  typedef T vt __attribute__((ext_vector_type(V)));
  typedef int8_t vc __attribute__((ext_vector_type(V)));
  const size_t row = blockIdx.x;
  const uint32_t n = a.n;
  const vt* x = reinterpret_cast<const vt*>(static_cast<const T*>(a.x) + row * a.xs);
  const vt* r = a.r ? reinterpret_cast<const vt*>(static_cast<const T*>(a.r) + row * a.rs) : nullptr;
  const vt* w = static_cast<const vt*>(a.w);
  vt* z = a.z ? reinterpret_cast<vt*>(static_cast<T*>(a.z) + row * a.zs) : nullptr;
  const uint32_t nv = n / V;
  vt v[C], rv[C], wv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = c * BLOCK + threadIdx.x;
    if (i < nv) {
      v[c] = x[i];
      if (NORM && r) rv[c] = r[i];
      if (NORM) wv[c] = w[i];
    }
  }
  RowSum s;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = c * BLOCK + threadIdx.x;
    if (i >= nv) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (NORM && r) v[c][e] = (T)((float)v[c][e] + (float)rv[c][e]);
      s.add<NORM>((float)v[c][e], NORM ? (float)wv[c][e] : 1.0f);
    }
    if (NORM && z) z[i] = v[c];
  }
  s.join();
  const double inv = NORM ? 1.0 / sqrt(s.ss / n + (double)a.eps) : 1.0;
  const float scale = scale_of(s.top * inv, isnan(s.bad));
  if (threadIdx.x == 0) a.scale[row] = scale;
  const double f = NORM && scale > 0.0f ? inv / (double)scale : 0.0;
  const Coder code(scale);
  vc* codes = reinterpret_cast<vc*>(a.codes + row * (size_t)n);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t i = c * BLOCK + threadIdx.x;
    if (i >= nv) continue;
    vc o;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y = (float)v[c][e];
      o[e] = (int8_t)(NORM ? (f > 0.0 ? (int)rint((double)y * (double)(float)wv[c][e] * f) : 0) : code(y));
    }
    codes[i] = o;
  }
}

// ------------------------------------------------------------- the product

struct LinearArgs {
  const int8_t *x, *w;
  const float *xs, *ws;
  int64_t xst, wst, yst;
  void* y;
  uint32_t rows, m, k, type;
};

// 16 codes from p[k0 ..], zeros from k on. Unaligned rows are read by unaligned
// 16-byte loads, their last codes one by one: nothing behind a row is read.
template <bool ALIGNED>
__device__ __forceinline__ v4i load16(const int8_t* p, uint32_t k0, uint32_t k) {
  v4i v = {0, 0, 0, 0};
  if (ALIGNED) {
    if (k0 < k) v = *reinterpret_cast<const v4i*>(p + k0);
  } else if (k0 + 16 <= k) {
    __builtin_memcpy(&v, p + k0, 16);
  } else {
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      uint32_t x = 0;
      for (uint32_t i = 0; i < 4; ++i)
        if (k0 + 4 * w + i < k) x |= (uint32_t)(uint8_t)p[k0 + 4 * w + i] << (8 * i);
      v[w] = (int)x;
    }
  }
  return v;
}

// A sum of code products as the value it stands for. The scales are 2^-107 or
// more: sum and row scale first, so that no factor is lost below f32's range
// (the scales' own product would be) where the value is not.
__device__ __forceinline__ float scaled(int sum, float xs, float ws) { return (float)sum * xs * ws; }
// ... of a row whose scale may be over 2^64, where the sum would pass f32's range
// above it and the value does not: the scale is taken 2^64 times smaller until
// the channel's is in. Powers of two are exact: in range the bits are the same.
__device__ __forceinline__ bool large_scale(float xs) { return xs > 0x1p64f; }
__device__ __forceinline__ float scaled_any(int sum, float xs, float ws) {
  const bool large = large_scale(xs);
  return scaled(sum, large ? xs * 0x1p-64f : xs, ws) * (large ? 0x1p64f : 1.0f);
}

// Few rows: a workgroup owns 16 MT channels and 16 NT rows, its waves share k
// in steps of 128 codes; a lane's 32 bytes of a step go straight into two
// matrix instructions. The waves' sums meet in LDS. Bound by memory, which reads
// every weight once: 1 x 28672 x 4096 in 21.8 us (5.4 TB/s of the 6.0 that a large
// read reaches); 1 x 960 x 576 in 3.2 us, latency.
template <int MT, int NT, int NW, bool ALIGNED>
__global__ __launch_bounds__(NW * WAVE) void k_linear_few(LinearArgs a) {
  const uint32_t lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, r16 = lane % 16, kg = lane / 16;
  const uint32_t m0 = blockIdx.x * 16 * MT, n0 = blockIdx.y * 16 * NT;
  const int8_t *w[MT], *x[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) w[t] = a.w + (int64_t)min(m0 + 16 * t + r16, a.m - 1) * a.wst;
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = a.x + (int64_t)min(n0 + 16 * t + r16, a.rows - 1) * a.xst;
  v4i acc[MT][NT];
#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[u][t] = v4i{0, 0, 0, 0};
  for (uint32_t s0 = wave * 128; s0 < a.k; s0 += NW * 128) {
    const uint32_t k0 = s0 + kg * 32;
    v4i wv[MT][2], xv[NT][2];
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[u][h] = load16<ALIGNED>(w[u], k0 + 16 * h, a.k);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[t][h] = load16<ALIGNED>(x[t], k0 + 16 * h, a.k);
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[u][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u][h], xv[t][h], acc[u][t], 0, 0, 0);
  }
  __shared__ v4i part[NW][MT * NT][WAVE];
#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][u * NT + t][lane] = acc[u][t];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += NW) {
    v4i s = part[0][f][lane];
#pragma unroll
    for (int u = 1; u < NW; ++u) s += part[u][f][lane];
    const uint32_t row = n0 + 16 * (f % NT) + r16, c0 = m0 + 16 * (f / NT) + 4 * kg;
    if (row >= a.rows) continue;
    const float xs = a.xs[row];
    for (int i = 0; i < 4; ++i)
      if (c0 + i < a.m) store_value(a.y, (int64_t)row * a.yst + c0 + i, a.type, scaled_any(s[i], xs, a.ws[c0 + i]));
  }
}

// Many rows: a workgroup of 2 x 2 waves owns BR = 64 TM rows and BC = 64 TN
// channels and takes both operands through LDS, 128 codes of k a stage: a
// copy instruction moves 8 whole 128-byte lines. A row's eight 16-byte chunks
// lie in LDS in an order that depends on the row, so that the same chunk of
// 8, or of 16, rows in turn lies in different banks. A wave's 32 x 32 products
// take 16 bytes a lane of each side per 32 codes.
typedef int v16i __attribute__((ext_vector_type(16)));

template <int TM, int TN>
struct Tile {
  static constexpr int BR = 64 * TM, BC = 64 * TN, BK = 128;
  static constexpr int CHUNKS = BK / 16, ROWS = 64 / CHUNKS;  // of a row, rows of a copy instruction
  static constexpr int NI = (BR + BC) / (4 * ROWS);           // copies of each wave
  uint32_t r0, c0, xn, wn;                                    // the tile's first row and channel, and how many of each
  uint32_t lane, wave, wr, wc, l32, half;

  __device__ __forceinline__ Tile() {
    lane = threadIdx.x % WAVE;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    wr = wave / 2 * 32 * TM;
    wc = wave % 2 * 32 * TN;
    l32 = lane % 32;
    half = lane / 32;
  }
  __device__ __forceinline__ void at(const LinearArgs& a, uint32_t nrt, uint32_t id) {
    r0 = id % nrt * BR;
    c0 = id / nrt * BC;
    xn = min((uint32_t)BR, a.rows - r0);
    wn = min((uint32_t)BC, a.m - c0);
  }
  // the lane's row (of rows, then channels) and chunk in this wave's copy i
  __device__ __forceinline__ uint32_t copy_row(int i) const { return ROWS * (4 * i + wave) + lane / CHUNKS; }
  __device__ __forceinline__ uint32_t copy_chunk() const { return lane % CHUNKS ^ order(copy_row(0)); }  // any i: the same
  __device__ __forceinline__ uint32_t copy_to(int i) const { return ROWS * (4 * i + wave) * BK; }
  static constexpr bool copies_x(int i) { return ROWS * 4 * i < BR; }
  // the place of a row's chunk c is c ^ order(row)
  __device__ __forceinline__ static uint32_t order(uint32_t row) { return (row % 8) ^ (row / 8 % 2); }
  // operands of the stage's ks-th 32 codes; wr and wc are multiples of 32, so
  // the order of chunks goes by l32
  __device__ __forceinline__ void read(const int8_t* stage, int ks, v4i* xv, v4i* wv) const {
    const uint32_t at = ((2 * ks + half) ^ order(l32)) * 16;
    const int8_t *xl = stage + (wr + l32) * BK + at, *wl = stage + (BR + wc + l32) * BK + at;
#pragma unroll
    for (int i = 0; i < TM; ++i) xv[i] = *reinterpret_cast<const v4i*>(xl + 32 * i * BK);
#pragma unroll
    for (int j = 0; j < TN; ++j) wv[j] = *reinterpret_cast<const v4i*>(wl + 32 * j * BK);
  }
  // ... multiplied, with between(n) after the n-th product
  template <class F>
  __device__ __forceinline__ static void multiply(const v4i* xv, const v4i* wv, v16i (*acc)[TN], F between) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xv[i], wv[j], acc[i][j], 0, 0, 0);
        between(i * TN + j);
      }
  }
  // Register e of a product: row 8 (e / 4) + 4 half + e % 4, channel l32. Two
  // neighbouring lanes exchange a register each, so that one stores row e's two
  // channels and the other row e + 1's: half the stores, of twice the bytes.
  template <class T, bool LARGE>
  __device__ __forceinline__ void store_as(const LinearArgs& a, const v16i (*acc)[TN], const float* xsl, const float* ws) const {
    auto value = [](int sum, float x, float w) { return LARGE ? scaled_any(sum, x, w) : scaled(sum, x, w); };
    typedef T T2 __attribute__((ext_vector_type(2)));
    T* y = static_cast<T*>(a.y);
    const bool odd = lane & 1, pairs = (a.yst % 2 | (uintptr_t)a.y % sizeof(T2)) == 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const uint32_t r = wr + 32 * i + 4 * half + 8 * e4;
        const v4f xs = *reinterpret_cast<const v4f*>(xsl + r);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t row = r0 + r + e, mine = row + odd;
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const uint32_t c = c0 + wc + 32 * j + l32;
            const float v0 = value(acc[i][j][4 * e4 + e], xs[e], ws[j]);
            const float v1 = value(acc[i][j][4 * e4 + e + 1], xs[e + 1], ws[j]);
            const float got = dpp<0xb1>(odd ? v0 : v1);  // quad_perm 1 0 3 2
            const uint32_t c2 = c - odd;
            if (pairs && mine < a.rows && c2 + 1 < a.m) {
              const T2 v = {(T)(odd ? got : v0), (T)(odd ? v1 : got)};
              *reinterpret_cast<T2*>(y + (int64_t)mine * a.yst + c2) = v;
            } else if (c < a.m && !(pairs && c2 + 1 < a.m)) {
              if (row < a.rows) y[(int64_t)row * a.yst + c] = (T)v0;
              if (row + 1 < a.rows) y[(int64_t)(row + 1) * a.yst + c] = (T)v1;
            }
          }
        }
      }
    }
  }
  // (Apart: the factors in every value are 8 of 260 us at 2047 x 28672 x 4096.)
  template <bool LARGE>
  __device__ __forceinline__ void store_typed(const LinearArgs& a, const v16i (*acc)[TN], const float* xsl, const float* ws) const {
    if (a.type == DEFER_GPU_F32)
      store_as<float, LARGE>(a, acc, xsl, ws);
    else if (a.type == DEFER_GPU_BF16)
      store_as<__bf16, LARGE>(a, acc, xsl, ws);
    else
      store_as<_Float16, LARGE>(a, acc, xsl, ws);
  }
  __device__ __forceinline__ void store(const LinearArgs& a, const v16i (*acc)[TN], const float* xsl, const float* ws) const {
    bool large = false;
    for (int i = 0; i < TM; ++i) large = large || large_scale(xsl[wr + 32 * i + l32]);
    if (__any(large))
      store_typed<true>(a, acc, xsl, ws);
    else
      store_typed<false>(a, acc, xsl, ws);
  }
  // The tile's scales: this lane's channels', and a row's for each thread to
  // leave in LDS (before a barrier).
  __device__ __forceinline__ float scales(const LinearArgs& a, float* ws) const {
#pragma unroll
    for (int j = 0; j < TN; ++j) ws[j] = a.ws[min(c0 + wc + 32 * j + l32, a.m - 1)];
    return a.xs[min(r0 + threadIdx.x, a.rows - 1)];
  }
  static_assert(BR <= 256, "a row for each thread");
};

// The tile of a workgroup: an XCD (workgroups w % 8) takes a run of tiles, the
// rows of one stripe of channels, then the next stripe.
__device__ __forceinline__ bool tile_of_workgroup(uint32_t tiles, uint32_t* id) {
  const uint32_t per = (tiles + 7) / 8;
  *id = blockIdx.x % 8 * per + blockIdx.x / 8;
  return blockIdx.x / 8 < per && *id < tiles;
}

// Aligned rows. Copies go memory -> LDS with no registers between (buffer
// loads, which write zeros for what is outside the operand or behind k), two
// stages ahead or more. They are issued one at a time between the products:
// in a row they keep a wave from its next product for as long as the memory
// pipeline takes them (2047 x 28672 x 4096: 320 us so, 257 now: 1,870 Tops/s, and
// 268 on operands that were not there a call before; the matrix cores alone reach
// 4,100, the library's i8 product of the same sizes takes 243 us). Wider tiles (256 x 256: 310 us, half the LDS reads but one
// stage of 64 codes less in flight), and one workgroup per CU that goes on to its
// next tile's copies while it stores (312), were slower. A stage's last reads are waited for before the barrier in
// it; behind that the next stage's first operands are read while its last
// products run.
template <int TM, int TN, int NBUF>
__global__ __launch_bounds__(256) void k_linear_tile(LinearArgs a, uint32_t nrt, uint32_t tiles) {
  typedef Tile<TM, TN> T;
  constexpr int NI = T::NI, BK = T::BK, STAGE = (T::BR + T::BC) * BK, KS = BK / 32;
  // one object: beside a second one the compiler waits for every copy before
  // each read of LDS
  __shared__ __align__(16) int8_t lds[NBUF * STAGE + 4 * T::BR];
  float* xsl = reinterpret_cast<float*>(lds + NBUF * STAGE);
  T t;
  uint32_t id;
  if (!tile_of_workgroup(tiles, &id)) return;
  t.at(a, nrt, id);
  float ws[TN];
  const float xs = t.scales(a, ws);
  auto* xb = const_cast<int8_t*>(a.x + (int64_t)t.r0 * a.xst);
  auto* wb = const_cast<int8_t*>(a.w + (int64_t)t.c0 * a.wst);
  auto xrs = __builtin_amdgcn_make_buffer_rsrc(xb, 0, (int)((t.xn - 1) * a.xst + a.k), 0x00020000);
  auto wrs = __builtin_amdgcn_make_buffer_rsrc(wb, 0, (int)((t.wn - 1) * a.wst + a.k), 0x00020000);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  uint32_t off[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const bool is_x = T::copies_x(i);
    const uint32_t r = t.copy_row(i) - (is_x ? 0 : T::BR);
    off[i] = r < (is_x ? t.xn : t.wn) ? (uint32_t)(r * (is_x ? a.xst : a.wst)) + t.copy_chunk() * 16 : OUTSIDE;
  }
  auto copy = [&](uint32_t k0, int buf, int i) {
    const bool in = k0 + t.copy_chunk() * 16 < a.k;
    auto* to = (__attribute__((address_space(3))) void*)(lds + buf * STAGE + t.copy_to(i));
    const int from = (int)(in ? off[i] : OUTSIDE);
    if (T::copies_x(i))
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xrs, to, 16, from, (int)k0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs, to, 16, from, (int)k0, 0, 0);
  };
  v16i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v16i{};
  v4i xv[2][TM], wv[2][TN];
#pragma unroll
  for (int b = 0; b < NBUF - 1; ++b)
#pragma unroll
    for (int i = 0; i < NI; ++i) copy(b * BK, b, i);
  if (threadIdx.x < T::BR) xsl[threadIdx.x] = xs;
  // Every wave's copies of the oldest stage have arrived (the younger ones may
  // be on their way), and what it has read so far is in its registers.
#define Q8_STAGE_WAIT(YOUNGER)                                                                         \
  do {                                                                                                 \
    constexpr int n_ = (YOUNGER)*NI;                                                                   \
    static_assert(n_ < 64, "vmcnt");                                                                   \
    asm volatile("" ::: "memory");                                                                     \
    __builtin_amdgcn_s_waitcnt((n_ & 15) | (n_ >> 4) << 14 | 0x0070); /* vmcnt(n_) lgkmcnt(0) */ \
    __builtin_amdgcn_s_barrier();                                                                      \
    asm volatile("" ::: "memory");                                                                     \
    __builtin_amdgcn_sched_barrier(0);                                                                 \
  } while (0)
  Q8_STAGE_WAIT(NBUF - 2);
  t.read(lds, 0, xv[0], wv[0]);
  int buf = 0, free_buf = NBUF - 1;
  for (uint32_t k0 = 0; k0 < a.k; k0 += BK) {
    const int next = buf + 1 == NBUF ? 0 : buf + 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks < KS - 1) {
        t.read(lds + buf * STAGE, ks + 1, xv[(ks + 1) % 2], wv[(ks + 1) % 2]);
      } else {
        Q8_STAGE_WAIT(NBUF - 2);
        t.read(lds + next * STAGE, 0, xv[0], wv[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // this wave's copies of the stage NBUF - 1 on, evenly among the products
      // before the barrier
      constexpr int PRODUCTS = (KS - 1) * TM * TN;
      T::multiply(xv[ks % 2], wv[ks % 2], acc, [&](int n) {
        const int done = ks * TM * TN + n;
        if (ks < KS - 1) {
#pragma unroll
          for (int i = done * NI / PRODUCTS; i < (done + 1) * NI / PRODUCTS; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            copy(k0 + (NBUF - 1) * BK, free_buf, i);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    }
    free_buf = buf;
    buf = next;
  }
#undef Q8_STAGE_WAIT
  __builtin_amdgcn_s_waitcnt(0x0f70);  // nothing may still be on its way into LDS at the end
  t.store(a, acc, xsl, ws);
}

// Unaligned rows go through registers: the next stage is on its way there while
// one is multiplied.
template <int TM, int TN>
__global__ __launch_bounds__(256) void k_linear_tile_odd(LinearArgs a, uint32_t nrt, uint32_t tiles) {
  typedef Tile<TM, TN> T;
  constexpr int NI = T::NI, STAGE = (T::BR + T::BC) * T::BK;
  __shared__ __align__(16) int8_t lds[2 * STAGE];
  __shared__ __align__(16) float xsl[T::BR];
  T t;
  uint32_t id;
  if (!tile_of_workgroup(tiles, &id)) return;
  t.at(a, nrt, id);
  float ws[TN];
  const float xs = t.scales(a, ws);
  const int8_t* p[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const bool is_x = T::copies_x(i);
    const uint32_t r = t.copy_row(i) - (is_x ? 0 : T::BR);
    p[i] = is_x ? a.x + (int64_t)(t.r0 + min(r, t.xn - 1)) * a.xst : a.w + (int64_t)(t.c0 + min(r, t.wn - 1)) * a.wst;
  }
  v4i reg[NI];
  auto fetch = [&](uint32_t k0) {
#pragma unroll
    for (int i = 0; i < NI; ++i) reg[i] = load16<false>(p[i], k0 + t.copy_chunk() * 16, a.k);
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      *reinterpret_cast<v4i*>(lds + buf * STAGE + t.copy_to(i) + t.lane * 16) = reg[i];
  };
  v16i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v16i{};
  v4i xv[2][TM], wv[2][TN];
  fetch(0);
  put(0);
  if (threadIdx.x < T::BR) xsl[threadIdx.x] = xs;
  __syncthreads();
  int buf = 0;
  for (uint32_t k0 = 0; k0 < a.k; k0 += T::BK, buf ^= 1) {
    const bool more = k0 + T::BK < a.k;
    if (more) fetch(k0 + T::BK);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      t.read(lds + buf * STAGE, ks, xv[ks % 2], wv[ks % 2]);
      T::multiply(xv[ks % 2], wv[ks % 2], acc, [](int) {});
    }
    if (more) put(buf ^ 1);
    __syncthreads();
  }
  t.store(a, acc, xsl, ws);
}

// ------------------------------------------------------------- the cache

struct KvArgs {
  Pages p;
  Rows r;
  void *k, *v;
  int64_t ks, vs;
  uint32_t type, hd;
  bool vec;  // eight values of a row are 16-byte loads and stores
};

// A workgroup owns the new rows of 16 positions of a page, one head. 16 lanes
// take a row's key or value, 8 values each: maximum, scale, codes; keys go out as they are,
// values through LDS into their transposed page, 16 positions (16 bytes) a store.
// No other workgroup of the call writes these positions of the sequence, and
// bytes of rows that are not the call's are not touched. (2000 rows of 8 heads of
// 128 in bf16, 12.4 MB: 40 us with a wave per row and a whole page per workgroup,
// 14.6 with 16 lanes per row, 9.4 with a quarter page. Bound by the latency of
// one load, a reduction and one store; so a row's key and value go side by side:
// 64 sequences' single rows 4.8 us, 6.5 one after the other.)
__global__ __launch_bounds__(256) void k_kv_write(KvArgs a) {
  const uint32_t per = kv_runs(a.r.most_rows);
  const uint32_t g = blockIdx.x % a.p.heads, b = blockIdx.x / a.p.heads % per, seq = blockIdx.x / a.p.heads / per;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const int64_t first = max((int64_t)0, sp.pos(0)), end = sp.len;  // positions [first, end)
  const int64_t run = first / KV_RUN + b, t0 = max(first, run * KV_RUN), t1 = min(end, (run + 1) * KV_RUN);
  if (t0 >= t1) return;
  const int64_t block = run * KV_RUN / PAGE;
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const int page = page_of(table, width, q.pages, block);
  if (page < 0) return;
  const size_t hp = (size_t)page * a.p.heads + g;
  int8_t* kc = q.keys + hp * PAGE * a.p.dp;
  int8_t* vc = q.values + hp * PAGE * a.p.dp;
  const uint32_t n16 = threadIdx.x % 16, quad = threadIdx.x / 16, quads = blockDim.x / 16, hd = a.hd;
  const int a0 = (int)(t0 - block * PAGE), a1 = (int)(t1 - block * PAGE);
  const int64_t row0 = sp.start + (block * PAGE - sp.pos(0));  // the row of the block's first position
  __shared__ __align__(16) int8_t tile[KV_RUN * KV_ROW];
  const int tr = (int)(run * KV_RUN - block * PAGE);  // the run's first place in its page
  // every other 16 lanes a key, those between its value
  const bool which = quad % 2;
  for (int at = a0 + (int)quad / 2; at < a1; at += (int)quads / 2) {
    const int64_t row = row0 + at;
    float y[2][8], top = 0.0f, bad = 0.0f;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      if (h == 0 || hd > 128)
        load8(which ? a.v : a.k, row * (which ? a.vs : a.ks) + (int64_t)g * hd, 128 * h + 8 * n16, hd, a.type, a.vec, y[h]);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      if (h == 0 || hd > 128)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          top = fmaxf(top, fabsf(y[h][e]));
          bad = fmaf(y[h][e], 0.0f, bad);
        }
    const float scale = scale_of(row_max(top), isnan(row_sum(bad)));
    const Coder code(scale);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t d = 128 * h + 8 * n16;
      if (d >= hd) continue;
      uint64_t c = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) c |= (uint64_t)(uint8_t)code(y[h][e]) << (8 * e);
      // a page's row is a multiple of 64 codes: those behind hd are zeros
      *reinterpret_cast<uint64_t*>(which ? tile + (at - tr) * KV_ROW + d : kc + at * a.p.dp + d) = c;
    }
    if (n16 == 0) (which ? q.value_scale : q.key_scale)[hp * PAGE + at] = scale;
  }
  __syncthreads();
  if (a1 - a0 < KV_RUN) {  // some of the run: byte by byte
    for (uint32_t i = threadIdx.x; i < (uint32_t)(a1 - a0) * hd; i += blockDim.x) {
      const uint32_t d = i % hd, t = a0 + i / hd;
      vc[d * PAGE + t] = tile[(t - tr) * KV_ROW + d];
    }
    return;
  }
  for (uint32_t d = 4 * threadIdx.x; d < hd; d += 4 * blockDim.x) {  // four channels a thread
    uint32_t w[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t in[4], out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = *reinterpret_cast<const uint32_t*>(tile + (4 * u + e) * KV_ROW + d);
      transpose4(in, out);
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c][u] = out[c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (d + c < hd)
        *reinterpret_cast<v4i*>(vc + (d + c) * PAGE + tr) = v4i{(int)w[c][0], (int)w[c][1], (int)w[c][2], (int)w[c][3]};
  }
}

// The same runs back: codes times scales (5001 rows of 8 heads of 128 to bf16,
// 31 MB in 10.1 us). What would be the runs of one more sequence clear the rows
// of none.
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a) {
  const uint32_t per = kv_runs(a.r.most_rows);
  const uint32_t g = blockIdx.x % a.p.heads, b = blockIdx.x / a.p.heads % per, seq = blockIdx.x / a.p.heads / per;
  const uint32_t n16 = threadIdx.x % 16, quad = threadIdx.x / 16, quads = blockDim.x / 16, hd = a.hd;
  if (seq == a.r.sequences) {
    const int64_t lo = min((int64_t)max(a.r.row_start[0], 0), (int64_t)a.r.rows);
    const int64_t hi = min((int64_t)max(a.r.row_start[seq], (int)lo), (int64_t)a.r.rows);
    for (int64_t i = b; i < lo + ((int64_t)a.r.rows - hi); i += per) {
      const int64_t row = i < lo ? i : hi + (i - lo);
      for (uint32_t d = threadIdx.x; d < hd; d += blockDim.x) {
        if (a.k) store_value(a.k, (row * a.p.heads + g) * hd + d, a.type, 0.0f);
        if (a.v) store_value(a.v, (row * a.p.heads + g) * hd + d, a.type, 0.0f);
      }
    }
    return;
  }
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  // runs from the one of the first row on, which may be before position 0
  auto down = [](int64_t t, int n) { return t >= 0 ? t / n : -((-t + n - 1) / n); };
  const int64_t p0 = sp.pos(0), run = down(p0, KV_RUN) + b;
  const int64_t t0 = max(p0, run * KV_RUN), t1 = min((int64_t)sp.len, (run + 1) * KV_RUN);
  if (t0 >= t1) return;
  const int64_t block = down(run, PAGE / KV_RUN);
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const int page = page_of(table, width, q.pages, block);
  const size_t hp = (size_t)max(page, 0) * a.p.heads + g;
  const int8_t* kc = q.keys + hp * PAGE * a.p.dp;
  const int8_t* vc = q.values + hp * PAGE * a.p.dp;
  const int a0 = (int)(t0 - block * PAGE), a1 = (int)(t1 - block * PAGE);
  const int64_t row0 = sp.start + (block * PAGE - p0);
  __shared__ __align__(16) int8_t tile[KV_RUN * KV_ROW];
  const int tr = (int)(run * KV_RUN - block * PAGE);  // the run's first place in its page
  if (page >= 0 && a.v) {
    for (uint32_t d = 4 * threadIdx.x; d < hd; d += 4 * blockDim.x) {  // rows up to a multiple of 64 are there
      v4i w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const v4i*>(vc + (d + c) * PAGE + tr);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t in[4], out[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) in[c] = (uint32_t)w[c][u];
        transpose4(in, out);
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(tile + (4 * u + e) * KV_ROW + d) = out[e];
      }
    }
  }
  __syncthreads();
  for (int at = a0 + (int)quad; at < a1; at += (int)quads) {
    const float ks = page >= 0 ? q.key_scale[hp * PAGE + at] : 0.0f, vs = page >= 0 ? q.value_scale[hp * PAGE + at] : 0.0f;
    const int64_t o = ((row0 + at) * a.p.heads + g) * hd;
    for (uint32_t d = 8 * n16; d < hd; d += 128) {
      float k[8], v[8];
      const uint64_t ck = page >= 0 ? *reinterpret_cast<const uint64_t*>(kc + at * a.p.dp + d) : 0;
      const uint64_t cv = page >= 0 ? *reinterpret_cast<const uint64_t*>(tile + (at - tr) * KV_ROW + d) : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] = page >= 0 ? (float)(int8_t)(ck >> (8 * e)) * ks : 0.0f;
        v[e] = page >= 0 ? (float)(int8_t)(cv >> (8 * e)) * vs : 0.0f;
      }
      if (a.k) store8(a.k, o, d, hd, a.type, a.vec, k);
      if (a.v) store8(a.v, o, d, hd, a.type, a.vec, v);
    }
  }
}

// ------------------------------------------------------------- attention

enum AttnMode { DIRECT, SPLIT, GROUP };
constexpr uint32_t SPLIT_WAVES = 4096;

// What a wave does: the attention of R tiles of four (row, query head) pairs
// of one sequence and cache head, over blocks of 64 positions.
//
// Scores: the four digits of a pair's query (31 bits, relative to the power of
// two over its largest value: an exact scaling) are four rows of a 16-row
// operand, the codes of 16 keys the columns, so a lane ends up with the four
// digit sums of one (pair, key). Keys 4 n + j (j = 0..3) are column n of four
// such products: a lane holds four neighbouring positions of its pair. The
// block's probabilities become digits the same way, go through LDS into operand
// order (four words written, one 16-byte read) and meet the values, which lie
// transposed so that a lane's 16 bytes are 16 positions. All sums of a block
// are exact integers; only the softmax and the sums over blocks round.
//
// A block's probabilities (relative to its own largest score) times its value
// scales are held in 30 bits relative to the largest such product: so one token
// that takes nearly all of a softmax and has small values leaves the others'
// contributions their accuracy.
//
// A score is digit sum * key scale * the query's factor. The sum counts the
// query as some 2^30 and the codes as up to 2^15 more, so that its product with a large
// key scale would pass f32's range where the score does not, and the factor of a
// small query would lie below it: 2^45 goes from the sum to the factor, exactly
// (not for a query over 2^64, whose factor would pass the range). Scores over 2^26
// have the largest taken off before they are multiplied by the factor: behind it
// the largest is rounded and a fused product is not, which could put a block's
// probabilities above or below f32's range. Both by selects: 11 of a block's and
// tile's 200 instructions (2048 8B rows 234 -> 242 us, 272 -> 282 with hidden
// positions; sessions' single rows as before). Branches around what is seldom needed
// hold more registers (251 us); a wave that starts again once its key scales say
// that it must takes 233 us, but 301 with hidden positions, and 64 1B rows 15.5 in
// place of 11.5.
//
// The next block's keys are on their way once this one's scores are formed, the
// next values once this one's are used, or with the keys where registers
// allow (R = 1: few rows, bound by memory).
//
// A long cache is bound by memory (11 8B rows of 6000 positions: 140 MB in 36.7
// us; 512 of 2000: 2.2 GB in 403 us, 5.4 TB/s), a prompt by vector instructions
// (3500 360M rows: 180 us, 146 of them the vector unit's; a tile and block takes
// about 200 of them beside 8 matrix products), a short step by its chain of
// dependent loads (64 1B rows of 385 positions: 10.7 us with hidden ones, 8.6
// without: four byte loads more a block).
//
// DIRECT: a wave goes through all its positions, unit after unit (many rows;
// the four waves of a workgroup are neighbouring tiles and meet the same codes
// in L1). SPLIT: a few units for each wave, left in the workspace for
// k_attn_join. GROUP: the units of a tile are the waves of one workgroup, which
// joins them through LDS.
template <int KC, int R, AttnMode MODE>
__global__ __launch_bounds__(MODE == GROUP ? 512 : 256, MODE == DIRECT && KC == 1 ? 3 : MODE != GROUP && (KC == 1 || (KC == 2 && R == 1)) ? 2 : 1) void k_attn(AttnArgs a) {
  constexpr int DT = 4 * KC, DP = 64 * KC;
  constexpr bool AHEAD = R == 1 && KC <= 2 && MODE != GROUP;  // the next values wait in registers of their own
  extern __shared__ __align__(16) uint8_t lds[];  // [waves][R][16][P_ROW], GROUP: then [4 R][units][2 + DP] floats
  const uint32_t lane = threadIdx.x % WAVE, n16 = lane % 16, quad = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE;
  uint8_t* pl = lds + wave * R * 16 * P_ROW;

  // which wave does what: (tile, unit) slowest, (sequence, cache head) fastest
  const uint32_t shs = a.r.sequences * a.p.heads;
  const uint32_t sh = blockIdx.x % shs, item = MODE == GROUP ? blockIdx.x / shs : blockIdx.x / shs * 4 + wave;
  const uint32_t seq = sh / a.p.heads, g = sh % a.p.heads;
  const uint32_t chunks = (a.units + a.per_wave - 1) / a.per_wave;  // of a row's units (SPLIT)
  const uint32_t tile = MODE == SPLIT ? item / chunks : MODE == DIRECT ? a.tiles - 1 - min(item, a.tiles - 1) : item;
  if (a.clear && blockIdx.x == gridDim.x - 1) {  // the first ones have the longest rows
    // rows of no sequence lie before the first span and behind the last
    const int64_t lo = span_of(a.r.row_start, a.r.kv_len, 0, a.r.rows).start;
    const int64_t hi = max(lo, min((int64_t)a.r.row_start[a.r.sequences], (int64_t)a.r.rows));
    for (int64_t i = wave; i < lo + ((int64_t)a.r.rows - hi); i += waves) {
      const int64_t row = i < lo ? i : hi + (i - lo);
      for (uint32_t d = lane; d < a.nh * a.hd; d += WAVE) store_value(a.out, row * a.os + d, a.type, 0.0f);
    }
  }
  if (MODE == SPLIT ? tile >= a.tiles : item >= a.tiles) return;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const uint32_t pair0 = tile * 4 * R;
  if (sp.n <= 0 || pair0 >= (uint32_t)sp.n * a.group) return;
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const uint8_t* hid = a.hidden ? a.hidden + (int64_t)seq * a.hs : nullptr;

  // pairs: (row j of the sequence, query head of the group)
  int pos[R], max_pos = -1, min_pos = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t j = (pair0 + 4 * r + quad) / a.group;
    const int64_t t = j < (uint32_t)sp.n ? min(sp.pos((int)j), a.most_len - 1) : -1;
    pos[r] = t < 0 ? -1 : (int)t;
    max_pos = max(max_pos, pos[r]);
    min_pos = min(min_pos, pos[r] < 0 ? 0x7fffffff : pos[r]);
  }
  max_pos = max(max_pos, __shfl_xor(max_pos, 16));
  max_pos = __builtin_amdgcn_readfirstlane(max(max_pos, __shfl_xor(max_pos, 32)));
  min_pos = min(min_pos, __shfl_xor(min_pos, 16));
  min_pos = __builtin_amdgcn_readfirstlane(min(min_pos, __shfl_xor(min_pos, 32)));

  v4i k[4][KC], v[DT], vn[AHEAD ? DT : 1];
  v4f ks, vs, ksn, vsn;
  const int8_t* k0 = q.keys + (size_t)g * PAGE * DP + 4 * n16 * DP + quad * 16;
  const int8_t* v0 = q.values + (size_t)g * PAGE * DP + n16 * PAGE + quad * 16;
  auto load_k = [&](int page) {
    const int8_t* kb = k0 + (size_t)page * a.p.heads * PAGE * DP;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) k[j][kk] = *reinterpret_cast<const v4i*>(kb + j * DP + kk * 64);
    const size_t hp = ((size_t)page * a.p.heads + g) * PAGE + 4 * n16;
    ksn = *reinterpret_cast<const v4f*>(q.key_scale + hp);
    vsn = *reinterpret_cast<const v4f*>(q.value_scale + hp);
  };
  auto load_v = [&](int page, v4i* to) {
    const int8_t* vb = v0 + (size_t)page * a.p.heads * PAGE * DP;
#pragma unroll
    for (int t = 0; t < DT; ++t) to[t] = *reinterpret_cast<const v4i*>(vb + 16 * t * PAGE);
  };

  // the queries' digits; the scores' sign is the scale's, folded into them
  v4i aq[R][KC];
  float sq[R];  // queries' factors for digit sums times 2^-45; negative: for the sums as they are
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t pr = pair0 + 4 * r + n16 / 4, j = pr / a.group;
    const bool ok = j < (uint32_t)sp.n;
    const int64_t q0 = (int64_t)(sp.start + (ok ? j : 0)) * a.qs + (int64_t)(g * a.group + pr % a.group) * a.hd;
    const float s = query_digits<KC>(a, q0, ok, aq[r]);
    sq[r] = __shfl(s, (int)quad * 4);
  }

  // Units from u0 on, every `du`-th, of the rows whose units are `ul` long:
  // rows of a tile that spans a multiple of 8,192 positions go one length
  // after the other.
  const int ul_last = unit_len(max(max_pos, 0));
  const int ul_first = max_pos < 0 ? ul_last : unit_len(min_pos);
  for (int ul = ul_first; ul <= ul_last; ul += UNIT) {
    int ps[R], pmax = -1, pmin = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ps[r] = pos[r] >= 0 && unit_len(pos[r]) == ul ? pos[r] : -1;
      pmax = max(pmax, ps[r]);
      pmin = min(pmin, ps[r]);
    }
    pmax = max(pmax, __shfl_xor(pmax, 16));
    pmax = __builtin_amdgcn_readfirstlane(max(pmax, __shfl_xor(pmax, 32)));
    pmin = min(pmin, __shfl_xor(pmin, 16));
    pmin = __builtin_amdgcn_readfirstlane(min(pmin, __shfl_xor(pmin, 32)));

    float M[R], L[R], A[R][DT], m[R], l[R], acc[R][DT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = m[r] = -INFINITY;
      L[r] = l[r] = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t) A[r][t] = acc[r][t] = 0.0f;
    }

    // A block whose codes have been loaded: WHOLE if every row sees all of it.
    // next: the page to load meanwhile, or -1.
    auto block = [&](auto whole, int b, int next) {
      constexpr bool WHOLE = decltype(whole)::value;
      ks = ksn;
      vs = vsn;
      const int tb = b * PAGE + 4 * n16;  // this lane's first position
      bool hide[4] = {false, false, false, false};
      if (!WHOLE && hid) {
#pragma unroll
        for (int j = 0; j < 4; ++j) hide[j] = (uint32_t)(tb + j) < a.hidden_len && hid[tb + j] != 0;
      }
      // a NaN value scale of a visible position reaches the sum, and with it
      // every output (adding the zeros of the others changes nothing)
      float vbad = 0.0f;
      if (WHOLE) vbad = fmaf(vs[0], 0.0f, vs[1] * 0.0f) + fmaf(vs[2], 0.0f, vs[3] * 0.0f);
      float xw[R], be[R];  // the weights of what came before and of this block
#pragma unroll
      for (int r = 0; r < R; ++r) {
        v4i d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d[j] = v4i{0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < KC; ++kk) d[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[r][kk], k[j][kk], d[j], 0, 0, 0);
        }
        if (r == R - 1 && next >= 0) {
          load_k(next);
          if (AHEAD) load_v(next, vn);
        }
        float s[4];
        bool see[4];
        const float unit = sq[r] < 0.0f ? 1.0f : 0x1p-45f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          see[j] = WHOLE || (tb + j <= ps[r] && !hide[j]);
          const float x = undigit(d[j]) * unit * ks[j];
          s[j] = see[j] ? x : -INFINITY;
        }
        uint32_t y[4];
        block_weights<WHOLE>(s, see, vs, vbad, fabsf(sq[r]), m[r], l[r], &xw[r], &be[r], y);
        uint32_t* pw = reinterpret_cast<uint32_t*>(pl + (16 * r + 4 * quad) * P_ROW) + n16;
        uint32_t by_digit[4];
        transpose4(y, by_digit);
#pragma unroll
        for (int i = 0; i < 4; ++i) pw[i * P_ROW / 4] = by_digit[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const v4i pa = *reinterpret_cast<const v4i*>(pl + (16 * r + n16) * P_ROW + quad * 16);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const v4i zero = {0, 0, 0, 0};
          const v4i o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, v[t], zero, 0, 0, 0);
          acc[r][t] = fmaf(undigit(o), be[r], acc[r][t] * xw[r]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (!AHEAD && next >= 0) load_v(next, v);
      if (AHEAD) {
#pragma unroll
        for (int t = 0; t < DT; ++t) v[t] = vn[t];
      }
    };

    const int bpu = ul / PAGE, blocks = pmax < 0 ? 0 : pmax / PAGE + 1;
    const int du = MODE == GROUP ? (int)waves : 1;
    int u = MODE == SPLIT ? (int)(item % chunks * a.per_wave) : MODE == GROUP ? (int)wave : 0;
    const int u_end = MODE == SPLIT ? u + (int)a.per_wave : (blocks + bpu - 1) / bpu;
    int b = u * bpu;
    // pages of 64 blocks at a time, one a lane: a load for each block would have
    // to arrive before the block's own loads can go out
    int window = -1, window_page = -1;
    auto page_at = [&](int block) {
      if (block / WAVE != window) {
        window = block / WAVE;
        window_page = page_of(table, width, q.pages, (int64_t)window * WAVE + lane);
      }
      return __builtin_amdgcn_readlane(window_page, block % WAVE);
    };
    int page = u < u_end && b < blocks ? page_at(b) : -1;
    if (page >= 0) {
      load_k(page);
      load_v(page, v);
    }
    while (u < u_end && b < blocks) {
      const bool unit_ends = b + 1 == blocks || (b + 1) % bpu == 0;
      const int bn = unit_ends ? (u + du) * bpu : b + 1;
      const int next = bn < blocks && (!unit_ends || u + du < u_end) ? page_at(bn) : -1;
      if (page >= 0) {
        if (!hid && b * PAGE + PAGE - 1 <= pmin)
          block(std::true_type(), b, next);
        else
          block(std::false_type(), b, next);
      } else if (next >= 0) {
        load_k(next);
        load_v(next, v);
      }
      if (unit_ends) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float lu = row_sum(l[r]);
          if (MODE == DIRECT) {
            float x, y;
            join_weights(M[r], m[r], &x, &y);
#pragma unroll
            for (int t = 0; t < DT; ++t) A[r][t] = fmaf(acc[r][t], y, A[r][t] * x);
            L[r] = fmaf(lu, y, L[r] * x);
          } else if (ps[r] >= 0 && u < unit_count(ps[r])) {
            const uint32_t pr = pair0 + 4 * r + quad;
            float* o = MODE == SPLIT ? a.part + (((size_t)(sp.start + pr / a.group) * a.nh + g * a.group + pr % a.group) * a.units + u) * (2 + DP)
                                     : reinterpret_cast<float*>(lds + waves * R * 16 * P_ROW) +
                                           ((4 * r + quad) * a.units + u) * (2 + DP);
            if (n16 == 0) {
              o[0] = m[r];
              o[1] = lu;
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) o[2 + 16 * t + n16] = acc[r][t];
          }
          m[r] = -INFINITY;
          l[r] = 0.0f;
#pragma unroll
          for (int t = 0; t < DT; ++t) acc[r][t] = 0.0f;
        }
        u += du;
      }
      b = bn;
      page = next;
    }
    if (MODE == DIRECT) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // a pair without a position is written in the first pass
        const uint32_t pr = pair0 + 4 * r + quad, j = pr / a.group;
        if (j >= (uint32_t)sp.n || !(ps[r] >= 0 || (pos[r] < 0 && ul == ul_first))) continue;
        const int64_t o = (int64_t)(sp.start + j) * a.os + (int64_t)(g * a.group + pr % a.group) * a.hd;
        const float inv = L[r] == 0.0f ? 0.0f : 1.0f / L[r];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const uint32_t d = 16 * t + n16;
          if (d < a.hd) store_value(a.out, o + d, a.type, A[r][t] * inv);
        }
      }
    }
  }
  if (MODE == GROUP) {
    __syncthreads();
    const float* parts = reinterpret_cast<const float*>(lds + waves * R * 16 * P_ROW);
    for (uint32_t i = threadIdx.x; i < 4u * R * DP; i += blockDim.x) {
      const uint32_t pr = pair0 + i / DP, j = pr / a.group, d = i % DP;
      if (j >= (uint32_t)sp.n) continue;
      const int n = unit_count(min(sp.pos((int)j), a.most_len - 1));
      const float* p = parts + i / DP * a.units * (2 + DP);
      float M = -INFINITY, L = 0.0f, A = 0.0f;
      for (int u = 0; u < n; ++u, p += 2 + DP) {
        float x, y;
        join_weights(M, p[0], &x, &y);
        A = fmaf(p[2 + d], y, A * x);
        L = fmaf(p[1], y, L * x);
      }
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      if (d < a.hd)
        store_value(a.out, (int64_t)(sp.start + j) * a.os + (int64_t)(g * a.group + pr % a.group) * a.hd + d, a.type, A * inv);
    }
  }
}

// Joins a row's units in order, as the unsplit kernel does. One workgroup of
// dp lanes per (row of a sequence, head); a lane holds one unit's maximum and
// sum, the accumulators of 32 units are on their way at a time. Three dependent
// reads of what other XCDs wrote: 10 us for 11 x 32 heads of 47 units (8.6 MB);
// 64 units at a time changed nothing.
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
  const uint32_t h = blockIdx.x % a.nh, j = blockIdx.x / a.nh % a.r.most_rows, seq = blockIdx.x / a.nh / a.r.most_rows;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  if (j >= (uint32_t)sp.n) return;
  const int64_t pos = min(sp.pos((int)j), a.most_len - 1);
  const uint32_t row = sp.start + j, d = threadIdx.x, dp = a.p.dp, lane = threadIdx.x % WAVE;
  const float* p = a.part + ((size_t)row * a.nh + h) * a.units * (2 + dp);
  const int n = unit_count(pos);
  static_assert(MAX_UNITS <= WAVE, "a unit for each lane");
  const float ml = (int)lane < n ? p[lane * (2 + dp)] : 0.0f, ll = (int)lane < n ? p[lane * (2 + dp) + 1] : 0.0f;
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  constexpr int AT_ONCE = 32;
  for (int u0 = 0; u0 < n; u0 += AT_ONCE) {
    float acc[AT_ONCE];
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) acc[e] = u0 + e < n ? p[(u0 + e) * (2 + dp) + 2 + d] : 0.0f;
#pragma unroll
    for (int e = 0; e < AT_ONCE; ++e) {
      if (u0 + e < n) {
        float x, y;
        join_weights(M, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ml), u0 + e)), &x, &y);
        A = fmaf(acc[e], y, A * x);
        L = fmaf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ll), u0 + e)), y, L * x);
      }
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  if (d < a.hd) store_value(a.out, (int64_t)row * a.os + (int64_t)h * a.hd + d, a.type, A * inv);
}

// ------------------------------------------------------------- launches

template <class T, bool NORM>
int rows_launch_as(const NormArgs& a, uint32_t rows, hipStream_t s) {
  constexpr uint32_t V = 16 / sizeof(T);
  auto fits = [](const void* p, int64_t stride) { return ((uintptr_t)p | (uintptr_t)(stride * (int64_t)sizeof(T))) % 16 == 0; };
  const bool vec = a.n % V == 0 && fits(a.x, a.xs) && fits(a.w, 0) && (!a.r || fits(a.r, a.rs)) && (!a.z || fits(a.z, a.zs)) &&
                   ((uintptr_t)a.codes | a.n) % V == 0;
  const uint32_t nv = a.n / V;  // threads by n alone: they make the order of the sums
  if (vec && nv <= 256)
    return launch(k_rows_vec<T, NORM, 256, 1>, rows, 256, 0, s, a);
  if (vec && nv <= 512)
    return launch(k_rows_vec<T, NORM, 256, 2>, rows, 256, 0, s, a);
  if (vec && nv <= 1024)
    return launch(k_rows_vec<T, NORM, 256, 4>, rows, 256, 0, s, a);
  if (vec && nv <= 4096)
    return launch(k_rows_vec<T, NORM, 1024, 4>, rows, 1024, 0, s, a);
  if (nv <= 1024)
    return launch(k_rows<T, NORM, 256>, rows, 256, 0, s, a);
  return launch(k_rows<T, NORM, 1024>, rows, 1024, 0, s, a);
}
template <bool NORM>
int rows_launch(uint32_t type, const NormArgs& a, uint32_t rows, hipStream_t s) {
  if (type == DEFER_GPU_F32) return rows_launch_as<float, NORM>(a, rows, s);
  if (type == DEFER_GPU_BF16) return rows_launch_as<__bf16, NORM>(a, rows, s);
  return rows_launch_as<_Float16, NORM>(a, rows, s);
}

template <int R, AttnMode MODE>
int attn_launch(const AttnArgs& a, uint32_t blocks, uint32_t threads, size_t lds, hipStream_t s) {
  const uint32_t kc = a.p.dp / 64;
  if constexpr (R <= 2)
    if (kc == 1) return launch(k_attn<1, R, MODE>, blocks, threads, lds, s, a);
  if (kc == 2) return launch(k_attn<2, R, MODE>, blocks, threads, lds, s, a);
  if constexpr (MODE != GROUP && R <= 2)
    if (kc == 3) return launch(k_attn<3, R, MODE>, blocks, threads, lds, s, a);
  if constexpr (MODE != GROUP && R == 1)
    if (kc == 4) return launch(k_attn<4, R, MODE>, blocks, threads, lds, s, a);
  return defer_gpu_fail_(DEFER_GPU_E_INVALID, "no attention kernel for head_dim %u", a.hd);
}

// (Row, query head) pairs of a sequence and cache head. A call of more than
// MOST_PAIRS has too many workgroups anyway.
uint64_t pairs_of(const Rows& r, uint32_t heads, uint32_t kv_heads) { return (uint64_t)r.most_rows * (heads / kv_heads); }
constexpr uint64_t MOST_PAIRS = 0x7fffffff;

// How a call's pairs are dealt.
struct Plan {
  AttnMode mode;
  uint32_t R, tiles, units, per_wave, waves;  // tiles of 4 R pairs; units of a row at most, of a wave; waves of a workgroup
  size_t lds, workspace;
};
Plan plan_of(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t dp, uint32_t most_len) {
  const uint32_t pairs = (uint32_t)pairs_of(r, heads, kv_heads);
  Plan p;
  // Tiles share the codes a wave has loaded, so the more the better, as far as
  // registers allow and waves are left for the chip: a prompt of 2048 8B rows
  // takes 372, 276 and 242 us with 1, 2 and 4, one of 301 135M rows 9.0 and 12.5
  // with 1 and 2 (3500 360M rows: 307 and 180). Heads of 64 take three waves of R =
  // 2 a SIMD with 13 registers of each spilled, which hides more than sharing
  // between four rows saved at two waves (206 us with 4 where 2 took 191).
  auto waves_of = [&](uint32_t R) { return (uint64_t)r.sequences * kv_heads * ((pairs + 4 * R - 1) / (4 * R)); };
  p.R = pairs <= 4 || dp > 192 ? 1 : pairs > 8 && dp == 128 && waves_of(4) >= 2048 ? 4 : pairs <= 8 || waves_of(2) >= 1024 ? 2 : 1;
  p.tiles = (pairs + 4 * p.R - 1) / (4 * p.R);
  p.units = (uint32_t)most_units(most_len);
  p.waves = 4;
  p.per_wave = 1;
  p.workspace = 0;
  const uint64_t waves = waves_of(p.R);
  const size_t partials = (size_t)r.rows * heads * p.units * (2 + dp) * sizeof(float);
  const uint32_t w = std::min(p.units, 8u);
  // A wave for each of the chip's 1,024 SIMDs, and a row's units need no
  // dealing: 128 8B rows of 2000 positions take 98 us in one piece and 116 as
  // a workgroup's units; the 512 waves of 64 1B rows of 4000 take 70 in one piece
  // and 59 split.
  if (p.units > 1 && p.units <= 16 && p.R <= 2 && dp <= 128 && waves < 1024) {
    p.mode = GROUP;
    p.waves = w;
  } else if (p.units > 1 && waves < 1024 && partials <= ((size_t)128 << 20)) {
    // about four waves a SIMD: each has its rows' digits to form, so not more (11
    // 8B rows of 6000 positions: 37 us with the join, 101 in one piece; 16 of 8000:
    // 59, 158 in one piece, an eighth more with half as many waves)
    p.mode = SPLIT;
    p.per_wave = (uint32_t)std::max<uint64_t>(1, waves * p.units / SPLIT_WAVES);
    p.workspace = partials;
  } else {
    p.mode = DIRECT;
  }
  p.lds = p.waves * p.R * 16 * P_ROW + (p.mode == GROUP ? 4 * (size_t)p.R * p.units * (2 + dp) * sizeof(float) : 0);
  return p;
}

}  // namespace

int quantize(uint32_t type, const void* x, int64_t x_stride, uint32_t rows, uint32_t n, int8_t* codes,
             float* scale, hipStream_t s) {
  if (!rows) return DEFER_GPU_OK;
  NormArgs a{};
  a.x = x;
  a.xs = x_stride;
  a.codes = codes;
  a.scale = scale;
  a.n = n;
  return rows_launch<false>(type, a, rows, s);
}

int rms_norm(uint32_t type, const void* x, int64_t x_stride, const void* residual, int64_t r_stride,
             const void* weight, float eps, uint32_t rows, uint32_t n, void* sum, int64_t sum_stride,
             int8_t* codes, float* scale, hipStream_t s) {
  if (!rows) return DEFER_GPU_OK;
  const NormArgs a{x, residual, weight, x_stride, r_stride, sum_stride, sum, codes, scale, n, eps};
  return rows_launch<true>(type, a, rows, s);
}

template <int MT, int NT, int NW>
static int linear_few(const LinearArgs& a, bool aligned, hipStream_t s) {
  const dim3 grid((a.m + 16 * MT - 1) / (16 * MT), (a.rows + 16 * NT - 1) / (16 * NT));
  return launch(aligned ? k_linear_few<MT, NT, NW, true> : k_linear_few<MT, NT, NW, false>, grid, NW * WAVE, 0, s, a);
}
template <int TM, int TN, int NBUF>
static int linear_tile(const LinearArgs& a, hipStream_t s) {
  const uint32_t nrt = (a.rows + 64 * TM - 1) / (64 * TM), tiles = nrt * ((a.m + 64 * TN - 1) / (64 * TN));
  return launch(k_linear_tile<TM, TN, NBUF>, (tiles + 7) / 8 * 8, 256, 0, s, a, nrt, tiles);
}
template <int TM, int TN>
static int linear_tile_odd(const LinearArgs& a, hipStream_t s) {
  const uint32_t nrt = (a.rows + 64 * TM - 1) / (64 * TM), tiles = nrt * ((a.m + 64 * TN - 1) / (64 * TN));
  return launch(k_linear_tile_odd<TM, TN>, (tiles + 7) / 8 * 8, 256, 0, s, a, nrt, tiles);
}

int linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
           const float* w_scale, uint32_t rows, uint32_t m, uint32_t k, uint32_t type, void* y,
           int64_t y_stride, hipStream_t s) {
  if (!rows) return DEFER_GPU_OK;
  const LinearArgs a{x, w, x_scale, w_scale, x_stride, w_stride, y_stride, y, rows, m, k, type};
  const bool aligned = ((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_stride | (uintptr_t)w_stride | k) % 16 == 0;
  // offsets within a tile's operand fit 31 bits
  const bool near = std::max(x_stride, w_stride) <= (1 << 22);
  // Few rows read every weight once, at the rate of memory: 16 channels a
  // workgroup, whose waves share k; many waves of them where there are few
  // channels (1 x 4096 x 14336: 19.4 us with 4, 10.9 with 16; 1 x 28672 x
  // 4096: 21.8 and 25.9).
  const uint64_t m16 = (m + 15) / 16;
  if (rows <= 16)
    return m16 <= 512 && k >= 2048 ? linear_few<1, 1, 16>(a, aligned, s) : linear_few<1, 1, 4>(a, aligned, s);
  // Up to 64 rows and too few 64 x 64 tiles for the chip: k shared by eight
  // waves (64 x 2048 x 8192: 13.7 us, 14.5 in tiles; 64 x 16384 x 2048: 18.4
  // and 7.4), over 32 channels where 16 would be more than a workgroup per CU
  // (64 x 4096 x 14336: 39.7 with 16, 27.8 with 32). Between the two the tiles are
  // already ahead: 64 x 4096 x 14336 would take 24.3 in them, 64 x 8192 x 2048 6.6
  // where this takes 10.7.
  auto tiles_of = [&](uint32_t r, uint32_t c) { return (uint64_t)((rows + r - 1) / r) * ((m + c - 1) / c); };
  if (rows <= 64 && (tiles_of(64, 64) < 192 || !aligned))
    return m16 * ((rows + 31) / 32) <= 256 ? linear_few<1, 2, 8>(a, aligned, s) : linear_few<2, 2, 8>(a, aligned, s);
  if (!near) return linear_few<2, 2, 8>(a, aligned, s);
  // Unaligned: 301 x 577 x 1537 takes 20.5 us so and 23.8 in tiles, 130 x 9001 x
  // 3001 takes 113 and 42.
  if (!aligned)
    return tiles_of(128, 128) < 32 ? linear_few<1, 2, 8>(a, aligned, s) : linear_tile_odd<2, 2>(a, s);
  // The tile whose rounds over the chip take least: us a round and a stage as
  // measured (2047 x 28672 x 4096: 257 us in 256 x 128, 303 in 128 x 128; 1000
  // x 4096 x 4096: 32.2, 24.5, 31.7 in 64 x 64; 500 x 4096 x 4096: 29.3, 19.0,
  // 17.1). Two 64 x 64 tiles share a CU.
  const double stages = (k + 127) / 128;
  auto rounds = [&](uint64_t tiles, uint64_t at_once) { return (double)((tiles + at_once - 1) / at_once); };
  const uint64_t small = tiles_of(64, 64);
  const double t256 = rounds(tiles_of(256, 128), 256) * (6.0 + 1.0 * stages);
  const double t128 = rounds(tiles_of(128, 128), 256) * (3.0 + 0.7 * stages);
  const double t64 = rounds(small, 512) * (2.0 + (small <= 256 ? 0.34 : 0.5) * stages);
  if (t256 <= t128 && t256 <= t64) return linear_tile<4, 2, 3>(a, s);
  return t128 <= t64 ? linear_tile<2, 2, 4>(a, s) : linear_tile<1, 1, 4>(a, s);
}

static uint32_t kv_grid(const Pages& p, const Rows& r) {
  return r.sequences * p.heads * kv_runs(r.most_rows);
}

int kv_write(const Pages& p, const Rows& r, uint32_t type, const void* k, int64_t k_stride, const void* v,
             int64_t v_stride, uint32_t head_dim, hipStream_t s) {
  if (!r.rows || !r.sequences || !r.most_rows) return DEFER_GPU_OK;
  const int64_t vs = type == DEFER_GPU_F32 ? 4 : 2;
  const bool vec = head_dim % 8 == 0 && ((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_stride * vs) | (uintptr_t)(v_stride * vs)) % 16 == 0;
  const KvArgs a{p, r, const_cast<void*>(k), const_cast<void*>(v), k_stride, v_stride, type, head_dim, vec};
  return launch(k_kv_write, kv_grid(p, r), r.most_rows <= 2 ? 64 : 256, 0, s, a);
}

int kv_read(const Pages& p, const Rows& r, uint32_t type, void* k, void* v, uint32_t head_dim, hipStream_t s) {
  if (!r.rows) return DEFER_GPU_OK;
  if (!r.sequences || !r.most_rows) {
    const uint32_t n = p.heads * head_dim;
    const int rc = k ? launch(k_zero_rows, r.rows, 256, 0, s, k, n, n, type) : DEFER_GPU_OK;
    return rc || !v ? rc : launch(k_zero_rows, r.rows, 256, 0, s, v, n, n, type);
  }
  const bool vec = head_dim % 8 == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
  const KvArgs a{p, r, k, v, 0, 0, type, head_dim, vec};
  Rows and_one = r;
  and_one.sequences += r.row_start != nullptr;
  return launch(k_kv_read, kv_grid(p, and_one), r.most_rows <= 8 ? 64 : 256, 0, s, a);
}

size_t attention_workspace(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t most_len) {
  if (!r.rows || !r.sequences || !r.most_rows || pairs_of(r, heads, kv_heads) > MOST_PAIRS) return 0;
  const uint32_t dp = padded(head_dim);
  const Plan pl = plan_of(r, heads, kv_heads, dp, most_len);
  return pl.workspace;
}

int attention(const Pages& p, const Rows& r, const Attention& in, void* workspace, size_t workspace_bytes,
              hipStream_t s) {
  if (!r.rows) return DEFER_GPU_OK;
  if (!r.sequences || !r.most_rows) {
    return in.clear ? launch(k_zero_rows, r.rows, 256, 0, s, in.out, in.out_stride, in.heads * in.head_dim, in.type) : DEFER_GPU_OK;
  }
  if (pairs_of(r, in.heads, p.heads) > MOST_PAIRS)
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "too many rows for one call");
  const Plan pl = plan_of(r, in.heads, p.heads, p.dp, in.most_len);
  const size_t need = attention_workspace(r, in.heads, p.heads, in.head_dim, in.most_len);
  if (need && (!workspace || workspace_bytes < need))
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "attention needs a workspace of %zu bytes, got %zu", need,
                           workspace ? workspace_bytes : (size_t)0);
  AttnArgs a = attn_args(p, r, in, workspace);
  a.tiles = pl.tiles;
  a.units = pl.units;
  a.per_wave = pl.per_wave;
  const uint64_t items = (uint64_t)pl.tiles * (pl.mode == SPLIT ? (pl.units + pl.per_wave - 1) / pl.per_wave : 1);
  const uint64_t blocks = (pl.mode == GROUP ? items : (items + 3) / 4) * r.sequences * p.heads;
  if (blocks * pl.waves * WAVE > MAX_THREADS)
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "too many rows for one call");
  const uint32_t nb = (uint32_t)blocks, nt = pl.waves * WAVE;
  if (pl.mode == SPLIT) {
    const int rc = pl.R == 1 ? attn_launch<1, SPLIT>(a, nb, nt, pl.lds, s) : attn_launch<2, SPLIT>(a, nb, nt, pl.lds, s);
    return rc ? rc : launch(k_attn_join, r.sequences * r.most_rows * in.heads, p.dp, 0, s, a);
  }
  if (pl.mode == GROUP)
    return pl.R == 1 ? attn_launch<1, GROUP>(a, nb, nt, pl.lds, s) : attn_launch<2, GROUP>(a, nb, nt, pl.lds, s);
  if (pl.R == 1) return attn_launch<1, DIRECT>(a, nb, nt, pl.lds, s);
  return pl.R == 2 ? attn_launch<2, DIRECT>(a, nb, nt, pl.lds, s) : attn_launch<4, DIRECT>(a, nb, nt, pl.lds, s);
}

}  // namespace q8

// ------------------------------------------------------------- C entry points

using namespace q8;

extern "C" int defer_gpu_q8_quantize(uint32_t type, const void* x, int64_t x_stride, uint32_t rows, uint32_t n,
                                     int8_t* codes, float* scale, void* stream) {
  const int rc = check_rows_values(type, x, x_stride, rows, n, "x");
  if (rc) return rc;
  Q8_REQUIRE(rows == 0 || (codes && scale), "null output");
  return quantize(type, x, x_stride, rows, n, codes, scale, (hipStream_t)stream);
}

extern "C" int defer_gpu_q8_rms_norm(uint32_t type, const void* x, int64_t x_stride, const void* residual,
                                     int64_t residual_stride, const void* weight, float eps, uint32_t rows,
                                     uint32_t n, void* sum, int64_t sum_stride, int8_t* codes, float* scale,
                                     void* stream) {
  int rc = check_rows_values(type, x, x_stride, rows, n, "x");
  if (!rc && residual) rc = check_rows_values(type, residual, residual_stride, rows, n, "residual");
  if (!rc && sum) rc = check_rows_values(type, sum, sum_stride, rows, n, "sum");
  if (!rc) rc = check_rows_values(type, weight, n, 1, n, "weight");
  if (rc) return rc;
  if (sum) {
    const int64_t v = (int64_t)value_size(type);
    Q8_REQUIRE(!overlap(sum, sum_stride * v, rows, x, x_stride * v, rows, n * v), "sum overlaps x");
    Q8_REQUIRE(!residual || !overlap(sum, sum_stride * v, rows, residual, residual_stride * v, rows, n * v), "sum overlaps residual");
    Q8_REQUIRE(rows == 0 || (sum != weight && !overlap(sum, sum_stride * v, rows, weight, 0, 1, n * v)), "sum overlaps weight");
  }
  Q8_REQUIRE(eps >= 0.0f && eps < INFINITY, "eps %g", (double)eps);
  Q8_REQUIRE(rows == 0 || (codes && scale), "null output");
  return rms_norm(type, x, x_stride, residual, residual_stride, weight, eps, rows, n, sum, sum_stride, codes, scale,
                  (hipStream_t)stream);
}

extern "C" int defer_gpu_q8_linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w,
                                   int64_t w_stride, const float* w_scale, uint32_t rows, uint32_t m, uint32_t k,
                                   uint32_t type, void* y, int64_t y_stride, void* stream) {
  Q8_REQUIRE(k >= 1 && k < MAX_K, "k = %u: sums of code products are exact for 1 <= k < %u", k, MAX_K);
  int rc = check_rows_values(type, y, y_stride, rows, m, "y");
  if (rc) return rc;
  Q8_REQUIRE((rows + 31) / 32 <= 65535, "%u rows: at most 2,097,120 in one call", rows);
  Q8_REQUIRE(rows == 0 || (x && x_scale), "null x");
  constexpr uint32_t MOST_M = MAX_THREADS / 512 * 32;  // 512 threads for 32 channels, 256 for 16
  Q8_REQUIRE(m <= MOST_M, "%u channels: at most %u in one call", m, MOST_M);
  Q8_REQUIRE(w && w_scale, "null w");
  Q8_REQUIRE(rows <= 1 || x_stride >= (int64_t)k, "x: rows of %u codes %lld apart", k, (long long)x_stride);
  Q8_REQUIRE(m <= 1 || w_stride >= (int64_t)k, "w: rows of %u codes %lld apart", k, (long long)w_stride);
  return linear(x, x_stride, x_scale, w, w_stride, w_scale, rows, m, k, type, y, y_stride, (hipStream_t)stream);
}

extern "C" int defer_gpu_q8_kv_write(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                     const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* stream) {
  Pages p;
  Rows r;
  int rc = check_pages(pages, rows, &p, &r);
  if (rc) return rc;
  const uint32_t n = p.heads * pages->head_dim;
  rc = check_rows_values(type, k, k_stride, r.rows, n, "k");
  if (!rc) rc = check_rows_values(type, v, v_stride, r.rows, n, "v");
  if (rc) return rc;
  return kv_write(p, r, type, k, k_stride, v, v_stride, pages->head_dim, (hipStream_t)stream);
}

extern "C" int defer_gpu_q8_kv_read(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                    void* k, void* v, void* stream) {
  Pages p;
  Rows r;
  int rc = check_pages(pages, rows, &p, &r);
  if (rc) return rc;
  const uint32_t n = p.heads * pages->head_dim;
  if (k) rc = check_rows_values(type, k, n, r.rows, n, "k");
  if (!rc && v) rc = check_rows_values(type, v, n, r.rows, n, "v");
  if (rc) return rc;
  Q8_REQUIRE(type <= DEFER_GPU_F16, "value type %u", type);
  return kv_read(p, r, type, k, v, pages->head_dim, (hipStream_t)stream);
}

extern "C" size_t defer_gpu_q8_attention_workspace(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows,
                                                   uint32_t q_heads, uint32_t most_len) {
  if (!pages || !rows || !pages->heads || !q_heads || pages->head_dim > MAX_HEAD_DIM) return 0;
  const Rows r{rows->row_start, rows->kv_len, rows->sequences, rows->rows, rows->most_rows};
  return attention_workspace(r, q_heads, pages->heads, pages->head_dim, most_len);
}

extern "C" size_t defer_gpu_q8_tree_attention_workspace(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows,
                                                        uint32_t q_heads, uint32_t most_len) {
  if (!pages || !rows || !pages->heads || !q_heads || pages->head_dim > MAX_HEAD_DIM) return 0;
  const Rows r{rows->row_start, rows->kv_len, rows->sequences, rows->rows, rows->most_rows};
  return tree_attention_workspace(r, q_heads, pages->heads, pages->head_dim, most_len);
}

static int attend(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type, const void* q,
                  int64_t q_stride, uint32_t q_heads, const int32_t* parent, uint32_t most_len, float scale,
                  const uint8_t* hidden, int64_t hidden_stride, uint32_t hidden_len, void* out, int64_t out_stride,
                  uint32_t clear, void* workspace, size_t workspace_bytes, void* stream) {
  Pages p;
  Rows r;
  int rc = check_pages(pages, rows, &p, &r);
  if (!rc) rc = check_heads(pages, q_heads, most_len);
  if (rc) return rc;
  const uint32_t n = q_heads * pages->head_dim;
  rc = check_rows_values(type, q, q_stride, r.rows, n, "q");
  if (!rc) rc = check_rows_values(type, out, out_stride, r.rows, n, "out");
  if (rc) return rc;
  const int64_t v = (int64_t)value_size(type);
  Q8_REQUIRE(!overlap(out, out_stride * v, r.rows, q, q_stride * v, r.rows, n * v), "out overlaps q");
  Q8_REQUIRE(!hidden || r.sequences <= 1 || hidden_stride >= (int64_t)hidden_len, "hidden: rows of %u, %lld apart",
             hidden_len, (long long)hidden_stride);
  Q8_REQUIRE(aligned16(workspace), "workspace is not 16-byte aligned");
  Attention a{type, q, q_stride, out, out_stride, q_heads, pages->head_dim, scale, most_len, hidden, hidden_stride,
              hidden_len, clear != 0, parent};
  return (parent ? tree_attention : attention)(p, r, a, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int defer_gpu_q8_attention(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                      const void* q, int64_t q_stride, uint32_t q_heads, uint32_t most_len,
                                      float scale, const uint8_t* hidden, int64_t hidden_stride,
                                      uint32_t hidden_len, void* out, int64_t out_stride, uint32_t clear,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  return attend(pages, rows, type, q, q_stride, q_heads, nullptr, most_len, scale, hidden, hidden_stride, hidden_len, out,
                out_stride, clear, workspace, workspace_bytes, stream);
}

extern "C" int defer_gpu_q8_tree_attention(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                           const void* q, int64_t q_stride, uint32_t q_heads, const int32_t* parent,
                                           uint32_t most_len, float scale, const uint8_t* hidden, int64_t hidden_stride,
                                           uint32_t hidden_len, void* out, int64_t out_stride, uint32_t clear,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  Q8_REQUIRE(!rows || rows->most_rows <= MAX_TREE, "%u rows of a sequence: at most %u", rows->most_rows, MAX_TREE);
  Q8_REQUIRE(!rows || rows->rows == 0 || parent, "parent is null");
  Q8_REQUIRE(aligned_to(parent, 4), "parent is not aligned to its type");
  return attend(pages, rows, type, q, q_stride, q_heads, parent, most_len, scale, hidden, hidden_stride, hidden_len, out,
                out_stride, clear, workspace, workspace_bytes, stream);
}
