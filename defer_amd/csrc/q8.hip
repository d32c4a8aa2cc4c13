// q8.hip -- the 8-bit operators: rows to codes, the norm that leaves codes,
// the product of codes, the cache in codes and the attention over it.
//
// Sums of code products are exact in 32-bit integers (v_mfma_i32_16x16x64_i8),
// so they have no order; every other sum has one that depends on its own row
// only. Nothing here keeps state, allocates or waits.
#include "q8.h"

#include <math.h>

#include <algorithm>

namespace q8 {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int WAVE = 64;
constexpr double TINY = 0x1p-100;  // rows with a smaller maximum are held as zeros

// ------------------------------------------------------------- value types

__device__ __forceinline__ float load_value(const void* p, int64_t i, uint32_t type) {
  if (type == DEFER_GPU_F32) return static_cast<const float*>(p)[i];
  if (type == DEFER_GPU_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_value(void* p, int64_t i, uint32_t type, float v) {
  if (type == DEFER_GPU_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == DEFER_GPU_BF16)
    static_cast<__bf16*>(p)[i] = (__bf16)v;
  else
    static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// ------------------------------------------------------------- reductions

// Over the 16 lanes of a DPP row; every lane gets the result. Each step adds
// the same two numbers in both lanes of a pair, so all 16 hold the same bits.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp<0x128>(v));
  v = fmaxf(v, dpp<0x124>(v));
  v = fmaxf(v, dpp<0x122>(v));
  return fmaxf(v, dpp<0x121>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<0x128>(v);
  v += dpp<0x124>(v);
  v += dpp<0x122>(v);
  return v + dpp<0x121>(v);
}
template <class V>
__device__ __forceinline__ V wave_max(V v) {
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
template <class V>
__device__ __forceinline__ V wave_add(V v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// ------------------------------------------------------------- rows to codes

// Scale of a row with maximum `top`; nan: the row holds no finite values only.
__device__ __forceinline__ float scale_of(double top, bool nan) {
  const float s = top < TINY ? 0.0f : (float)(top / 127.0);
  return nan || !(s < INFINITY) ? __builtin_nanf("") : s;
}
// The code of y at a scale: in 64 bits, so that a quotient next to a half is
// on the side it belongs to. `scale` is 0 or NaN for a row of zeros.
__device__ __forceinline__ int code_of(double y, double scale) {
  return scale > 0.0 ? (int)rint(y / scale) : 0;
}

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
// exactly), which a kernel bound by memory does not notice, so that codes are
// those of the formula and not of a rounding.
template <class T, bool NORM>
__global__ __launch_bounds__(256) void k_rows(NormArgs a) {
  const size_t row = blockIdx.x;
  const uint32_t tid = threadIdx.x, n = a.n;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.rs : nullptr;
  const T* w = static_cast<const T*>(a.w);
  T* z = a.z ? static_cast<T*>(a.z) + row * a.zs : nullptr;
  auto value = [&](uint32_t i) {
    T v = x[i];
    if (NORM && r) v = (T)((float)v + (float)r[i]);
    return v;
  };
  double ss = 0.0, top = 0.0;
  float bad = 0.0f;  // NaN once a value is not finite
  for (uint32_t i = tid; i < n; i += 256) {
    const T v = value(i);
    const double d = (double)(float)v;
    const double y = NORM ? d * (double)(float)w[i] : d;
    if (NORM) ss = fma(d, d, ss);
    top = fmax(top, fabs(y));
    bad = fmaf((float)v, 0.0f, bad);
    if (NORM) bad = fmaf((float)w[i], 0.0f, bad);
  }
  __shared__ double s_ss[4], s_top[4];
  __shared__ float s_bad[4];
  ss = wave_add(ss);
  top = wave_max(top);
  bad = wave_add(bad);
  if (tid % WAVE == 0) {
    s_ss[tid / WAVE] = ss;
    s_top[tid / WAVE] = top;
    s_bad[tid / WAVE] = bad;
  }
  __syncthreads();
  ss = (s_ss[0] + s_ss[1]) + (s_ss[2] + s_ss[3]);
  top = fmax(fmax(s_top[0], s_top[1]), fmax(s_top[2], s_top[3]));
  bad = (s_bad[0] + s_bad[1]) + (s_bad[2] + s_bad[3]);
  const double inv = NORM ? 1.0 / sqrt(ss / n + (double)a.eps) : 1.0;
  const float scale = scale_of(top * inv, isnan(bad));
  if (tid == 0) a.scale[row] = scale;
  int8_t* c = a.codes + row * (size_t)n;
  for (uint32_t i = tid; i < n; i += 256) {
    const T v = value(i);
    const double d = (double)(float)v;
    c[i] = (int8_t)code_of(NORM ? d * (double)(float)w[i] * inv : d, (double)scale);
    if (NORM && z) z[i] = v;
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

// 16 codes from p[k0 ..], zeros from k on.
template <bool ALIGNED>
__device__ __forceinline__ v4i load16(const int8_t* p, uint32_t k0, uint32_t k) {
  v4i v = {0, 0, 0, 0};
  if (ALIGNED) {
    if (k0 < k) v = *reinterpret_cast<const v4i*>(p + k0);
  } else {
    union {
      int8_t b[16];
      v4i v;
    } u;
    u.v = v;
    for (uint32_t i = 0; i < 16; ++i)
      if (k0 + i < k) u.b[i] = p[k0 + i];
    v = u.v;
  }
  return v;
}

// Few rows: a workgroup owns 16 channels and 16 NT rows, its waves share k
// in steps of 128 codes; a lane's 32 bytes of a step go straight into two
// matrix instructions. The waves' sums meet in LDS.
template <int NT, bool ALIGNED>
__global__ __launch_bounds__(256) void k_linear_few(LinearArgs a) {
  constexpr int NW = 4;
  const uint32_t lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, r16 = lane % 16, kg = lane / 16;
  const uint32_t m0 = blockIdx.x * 16, n0 = blockIdx.y * 16 * NT;
  const int8_t* w = a.w + (int64_t)min(m0 + r16, a.m - 1) * a.wst;
  const int8_t* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = a.x + (int64_t)min(n0 + 16 * t + r16, a.rows - 1) * a.xst;
  v4i acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = v4i{0, 0, 0, 0};
  for (uint32_t k0 = wave * 128 + kg * 32; k0 - kg * 32 < a.k; k0 += NW * 128) {
    const v4i w0 = load16<ALIGNED>(w, k0, a.k), w1 = load16<ALIGNED>(w, k0 + 16, a.k);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, load16<ALIGNED>(x[t], k0, a.k), acc[t], 0, 0, 0);
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, load16<ALIGNED>(x[t], k0 + 16, a.k), acc[t], 0, 0, 0);
    }
  }
  __shared__ v4i part[NW][NT][WAVE];
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < NT; t += NW) {
    v4i s = part[0][t][lane];
    for (int u = 1; u < NW; ++u) s += part[u][t][lane];
    const uint32_t row = n0 + 16 * t + r16;
    if (row >= a.rows) continue;
    const float xs = a.xs[row];
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = m0 + 4 * kg + i;
      if (c < a.m) store_value(a.y, (int64_t)row * a.yst + c, a.type, (float)s[i] * (xs * a.ws[c]));
    }
  }
}

// ------------------------------------------------------------- the cache

__device__ __forceinline__ SeqPages pool_of(const Pages& p, uint32_t seq, const int32_t*& table, uint32_t& width) {
  if (p.seqs) {
    SeqPages s = p.seqs[seq];
    table = nullptr;
    width = s.pages;
    const int64_t off = p.seq_layer * s.pages * p.heads * PAGE;
    s.keys += off * p.dp;
    s.values += off * p.dp;
    s.key_scale += off;
    s.value_scale += off;
    return s;
  }
  table = p.table + (size_t)seq * p.width;
  width = p.width;
  return SeqPages{p.keys, p.values, p.key_scale, p.value_scale, p.pages};
}

struct KvArgs {
  Pages p;
  Rows r;
  void *k, *v;
  int64_t ks, vs;
  uint32_t type, hd;
};

constexpr int KV_ROW = 256 + 4;  // bytes of a token's codes in LDS, apart by an odd number of words

// A workgroup owns the new rows of one block of 64 positions, one head. A wave
// takes a row: maximum, scale, codes; keys go out as they are, values through
// LDS into their transposed page. No other workgroup of the call writes
// this block of the sequence, and bytes of rows that are not the call's are
// not touched.
__global__ __launch_bounds__(256) void k_kv_write(KvArgs a) {
  const uint32_t per = (a.r.most_rows + PAGE - 2) / PAGE + 1;
  const uint32_t g = blockIdx.x % a.p.heads, b = blockIdx.x / a.p.heads % per, seq = blockIdx.x / a.p.heads / per;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const int64_t first = max((int64_t)0, sp.pos(0)), end = sp.len;  // positions [first, end)
  const int64_t block = first / PAGE + b, t0 = max(first, block * PAGE), t1 = min(end, (block + 1) * PAGE);
  if (t0 >= t1) return;
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const int page = page_of(table, width, q.pages, block);
  if (page < 0) return;
  const size_t hp = (size_t)page * a.p.heads + g;
  int8_t* kc = q.keys + hp * PAGE * a.p.dp;
  int8_t* vc = q.values + hp * PAGE * a.p.dp;
  const uint32_t wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, hd = a.hd;
  __shared__ int8_t tile[PAGE * KV_ROW];
  for (int64_t t = t0 + wave; t < t1; t += 4) {
    const int64_t row = sp.start + (t - sp.pos(0));
    const int at = (int)(t - block * PAGE);
    for (int which = 0; which < 2; ++which) {
      const void* src = which ? a.v : a.k;
      const int64_t i0 = row * (which ? a.vs : a.ks) + (int64_t)g * hd;
      float y[4];
      float top = 0.0f, bad = 0.0f;
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t d = lane + WAVE * e;
        y[e] = d < hd ? load_value(src, i0 + d, a.type) : 0.0f;
        top = fmaxf(top, fabsf(y[e]));
        bad = fmaf(y[e], 0.0f, bad);
      }
      top = wave_max(top);
      const float scale = scale_of(top, isnan(wave_add(bad)));
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t d = lane + WAVE * e;
        if (d >= hd) continue;
        const int8_t c = (int8_t)code_of(y[e], scale);
        if (which)
          tile[at * KV_ROW + d] = c;
        else
          kc[at * a.p.dp + d] = c;
      }
      if (lane == 0) (which ? q.value_scale : q.key_scale)[hp * PAGE + at] = scale;
    }
  }
  __syncthreads();
  const int a0 = (int)(t0 - block * PAGE), a1 = (int)(t1 - block * PAGE);
  for (uint32_t i = threadIdx.x; i < hd * (PAGE / 4); i += 256) {
    const uint32_t d = i / (PAGE / 4);
    const int t = 4 * (int)(i % (PAGE / 4));
    if (t >= a0 && t + 4 <= a1) {
      uint32_t w = 0;
      for (int e = 0; e < 4; ++e) w |= (uint32_t)(uint8_t)tile[(t + e) * KV_ROW + d] << (8 * e);
      *reinterpret_cast<uint32_t*>(vc + d * PAGE + t) = w;
    } else {
      for (int e = 0; e < 4; ++e)
        if (t + e >= a0 && t + e < a1) vc[d * PAGE + t + e] = tile[(t + e) * KV_ROW + d];
    }
  }
}

// The same blocks back: codes times scales. What would be the blocks of one
// more sequence clear the rows of none.
__global__ __launch_bounds__(256) void k_kv_read(KvArgs a) {
  const uint32_t per = (a.r.most_rows + PAGE - 2) / PAGE + 1;
  const uint32_t g = blockIdx.x % a.p.heads, b = blockIdx.x / a.p.heads % per, seq = blockIdx.x / a.p.heads / per;
  if (seq == a.r.sequences) {
    const int64_t lo = min((int64_t)max(a.r.row_start[0], 0), (int64_t)a.r.rows);
    const int64_t hi = min((int64_t)max(a.r.row_start[seq], (int)lo), (int64_t)a.r.rows);
    for (int64_t row = b; row < (int64_t)a.r.rows; row += per) {
      if (row >= lo && row < hi) continue;
      for (uint32_t d = threadIdx.x; d < a.hd; d += 256) {
        if (a.k) store_value(a.k, (row * a.p.heads + g) * a.hd + d, a.type, 0.0f);
        if (a.v) store_value(a.v, (row * a.p.heads + g) * a.hd + d, a.type, 0.0f);
      }
    }
    return;
  }
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  // blocks from the one of the first row on, which may be before position 0
  const int64_t p0 = sp.pos(0), base = p0 >= 0 ? p0 / PAGE : -((-p0 + PAGE - 1) / PAGE);
  const int64_t block = base + b, t0 = max(p0, block * PAGE), t1 = min((int64_t)sp.len, (block + 1) * PAGE);
  if (t0 >= t1) return;
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const int page = page_of(table, width, q.pages, block);
  const size_t hp = (size_t)max(page, 0) * a.p.heads + g;
  const int8_t* kc = q.keys + hp * PAGE * a.p.dp;
  const int8_t* vc = q.values + hp * PAGE * a.p.dp;
  const uint32_t hd = a.hd;
  for (uint32_t i = threadIdx.x; i < (uint32_t)(t1 - t0) * hd; i += 256) {
    const int at = (int)(t0 - block * PAGE) + (int)(i / hd);
    const uint32_t d = i % hd;
    const int64_t row = sp.start + (block * PAGE + at - p0);
    float k = 0.0f, v = 0.0f;
    if (page >= 0) {
      k = (float)kc[at * a.p.dp + d] * q.key_scale[hp * PAGE + at];
      v = (float)vc[d * PAGE + at] * q.value_scale[hp * PAGE + at];
    }
    const int64_t o = (row * a.p.heads + g) * hd + d;
    if (a.k) store_value(a.k, o, a.type, k);
    if (a.v) store_value(a.v, o, a.type, v);
  }
}

// ------------------------------------------------------------- attention

struct AttnArgs {
  Pages p;
  Rows r;
  const void* q;
  void* out;
  int64_t qs, os;
  uint32_t type, nh, group, hd, tiles, units;
  int64_t most_len;
  float scale2;  // scale * log2(e)
  const uint8_t* hidden;
  int64_t hs;
  uint32_t hidden_len;
  float* part;  // [rows][nh][units][2 + dp]: maximum, sum, accumulators
};

// Four signed base-256 digits of x, one a byte: x = sum of byte_i 256^i.
__device__ __forceinline__ uint32_t digits(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }
// ... and back, from sums of products of each digit with codes.
__device__ __forceinline__ float undigit(v4i d) {
  return fmaf((float)((d[3] << 8) + d[2]), 65536.0f, (float)((d[1] << 8) + d[0]));
}
__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}

// A running softmax: maximum (in the exponent of 2), sum, accumulators.
// (M, L, A) joined with (m, l, acc) that follows it.
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.0f : m; }

constexpr int P_ROW = 80;  // bytes of a digit row of 64 probabilities in LDS: rows of four heads on other banks

// The attention of one wave: R tiles of four (row, head) pairs of one sequence
// and cache head, over blocks of 64 positions.
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
template <int KC, int R, bool SPLIT>
__global__ __launch_bounds__(256) void k_attn(AttnArgs a) {
  constexpr int DT = 4 * KC, DP = 64 * KC;
  __shared__ __align__(16) uint8_t lds[4][16 * P_ROW];
  const uint32_t lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, n16 = lane % 16, quad = lane / 16;
  uint8_t* pl = lds[wave];

  // which wave does what: (tile or unit) slowest, (sequence, cache head) fastest
  const uint32_t shs = a.r.sequences * a.p.heads;
  const uint32_t sh = blockIdx.x % shs, item = blockIdx.x / shs * 4 + wave;
  const uint32_t seq = sh / a.p.heads, g = sh % a.p.heads;
  const uint32_t tile = SPLIT ? item / a.units : a.tiles - 1 - min(item, a.tiles - 1);
  const uint32_t unit = SPLIT ? item % a.units : 0;
  if (SPLIT ? tile >= a.tiles : item >= a.tiles) return;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const uint32_t pair0 = tile * 4 * R;
  if (sp.n <= 0 || pair0 >= (uint32_t)sp.n * a.group) return;
  const int32_t* table;
  uint32_t width;
  const SeqPages q = pool_of(a.p, seq, table, width);
  const uint8_t* hid = a.hidden ? a.hidden + (int64_t)seq * a.hs : nullptr;

  // pairs: (row j of the sequence, query head of the group)
  int pos[R], max_pos = -1;
  uint32_t orow[R], ohead[R];
  bool have[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t pr = pair0 + 4 * r + quad, j = pr / a.group;
    have[r] = j < (uint32_t)sp.n;
    const int64_t t = have[r] ? min(sp.pos((int)j), a.most_len - 1) : -1;
    pos[r] = t < 0 ? -1 : (int)t;
    orow[r] = sp.start + j;
    ohead[r] = g * a.group + pr % a.group;
    max_pos = max(max_pos, pos[r]);
  }
  max_pos = max(max_pos, __shfl_xor(max_pos, 16));
  max_pos = max(max_pos, __shfl_xor(max_pos, 32));

  // the queries' digits
  v4i aq[R][KC];
  float sq[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t pr = pair0 + 4 * r + n16 / 4, j = pr / a.group;
    const bool ok = j < (uint32_t)sp.n;
    const int64_t q0 = (int64_t)(sp.start + (ok ? j : 0)) * a.qs + (int64_t)(g * a.group + pr % a.group) * a.hd;
    float x[KC][16], top = 0.0f, bad = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KC; ++kk)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t d = kk * 64 + quad * 16 + e;
        x[kk][e] = ok && d < a.hd ? load_value(a.q, q0 + d, a.type) : 0.0f;
        top = fmaxf(top, fabsf(x[kk][e]));
        bad = fmaf(x[kk][e], 0.0f, bad);
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    bad += __shfl_xor(bad, 16);
    bad += __shfl_xor(bad, 32);
    // top < 2^ex; values of rows under 2^-96 keep fewer digits
    int ex = 0;
    (void)frexpf(top, &ex);
    ex = top > 0.0f ? max(ex, -96) : 0;
    const float up = ldexpf(1.0f, 30 - ex);
    const float s = isnan(bad) ? __builtin_nanf("") : ldexpf(1.0f, ex - 30) * a.scale2;
#pragma unroll
    for (int kk = 0; kk < KC; ++kk)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int xi = isnan(bad) ? 0 : (int)(x[kk][4 * w + e] * up);
          v |= ((digits(xi) >> (8 * (n16 % 4))) & 0xffu) << (8 * e);
        }
        aq[r][kk][w] = (int)v;
      }
    sq[r] = __shfl(s, (int)quad * 4);
  }

  // Rows whose units have another length (sequences over 8,192 positions, where a
  // tile spans a multiple of that) go one length after the other.
  const int ul_last = unit_len(max(max_pos, 0));
  int lo = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < R; ++r) lo = min(lo, pos[r] < 0 ? 0x7fffffff : pos[r]);
  lo = min(lo, __shfl_xor(lo, 16));
  lo = min(lo, __shfl_xor(lo, 32));
  const int ul_first = lo == 0x7fffffff ? ul_last : unit_len(lo);
  for (int ul = ul_first; ul <= ul_last; ul += UNIT) {
    int ps[R];
    int pmax = -1, pmin = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ps[r] = pos[r] >= 0 && unit_len(pos[r]) == ul ? pos[r] : -1;
      pmax = max(pmax, ps[r]);
      pmin = min(pmin, ps[r]);
    }
    pmax = max(pmax, __shfl_xor(pmax, 16));
    pmax = max(pmax, __shfl_xor(pmax, 32));
    pmin = min(pmin, __shfl_xor(pmin, 16));
    pmin = min(pmin, __shfl_xor(pmin, 32));
    pmax = __builtin_amdgcn_readfirstlane(pmax);
    pmin = __builtin_amdgcn_readfirstlane(pmin);

    float M[R], L[R], A[R][DT], m[R], l[R], acc[R][DT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = m[r] = -INFINITY;
      L[r] = l[r] = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t) A[r][t] = acc[r][t] = 0.0f;
    }
    const int bpu = ul / PAGE;
    const int b0 = SPLIT ? (int)unit * bpu : 0;
    const int b1 = min(pmax < 0 ? 0 : pmax / PAGE + 1, SPLIT ? b0 + bpu : 0x7fffffff);
    for (int b = b0; b < b1; ++b) {
      const int page = page_of(table, width, q.pages, b);
      if (page >= 0) {
        const size_t hp = (size_t)page * a.p.heads + g;
        const int8_t* kb = q.keys + hp * PAGE * DP;
        const int8_t* vb = q.values + hp * PAGE * DP;
        v4i k[4][KC], v[DT];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int kk = 0; kk < KC; ++kk)
            k[j][kk] = *reinterpret_cast<const v4i*>(kb + (4 * n16 + j) * DP + kk * 64 + quad * 16);
        const v4f ks = *reinterpret_cast<const v4f*>(q.key_scale + hp * PAGE + 4 * n16);
        const v4f vs = *reinterpret_cast<const v4f*>(q.value_scale + hp * PAGE + 4 * n16);
#pragma unroll
        for (int t = 0; t < DT; ++t)
          v[t] = *reinterpret_cast<const v4i*>(vb + (16 * t + n16) * PAGE + quad * 16);
        const int tb = b * PAGE + 4 * n16;  // this lane's first position
        bool hide[4] = {false, false, false, false};
        if (hid) {
#pragma unroll
          for (int j = 0; j < 4; ++j) hide[j] = (uint32_t)(tb + j) < a.hidden_len && hid[tb + j] != 0;
        }
        // every row sees the whole block
        const bool whole = !hid && b * PAGE + PAGE - 1 <= pmin;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float s[4];
          bool see[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v4i d = {0, 0, 0, 0};
#pragma unroll
            for (int kk = 0; kk < KC; ++kk)
              d = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[r][kk], k[j][kk], d, 0, 0, 0);
            see[j] = whole || (tb + j <= ps[r] && !hide[j]);
            s[j] = see[j] ? undigit(d) * (sq[r] * ks[j]) : -INFINITY;
          }
          const float mb = row_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
          const float mb0 = finite_or_0(mb);
          float lp = 0.0f, w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = see[j] ? __builtin_amdgcn_exp2f(s[j] - mb0) : 0.0f;
            // a NaN value scale reaches the sum, and with it every output
            lp += see[j] ? fmaf(vs[j], 0.0f, p) : 0.0f;
            w[j] = see[j] ? p * vs[j] : 0.0f;
          }
          int ex = 0;
          (void)frexpf(row_max(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))), &ex);
          const float down = ldexpf(1.0f, ex - 30);
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = digits((int)fminf(fmaxf(ldexpf(w[j], 30 - ex), 0.0f), 0x1p30f));
          const uint32_t t01l = perm(y[1], y[0], 0x05010400u), t23l = perm(y[3], y[2], 0x05010400u);
          const uint32_t t01h = perm(y[1], y[0], 0x07030602u), t23h = perm(y[3], y[2], 0x07030602u);
          uint32_t* pw = reinterpret_cast<uint32_t*>(pl + 4 * quad * P_ROW) + n16;
          pw[0] = perm(t23l, t01l, 0x05040100u);
          pw[P_ROW / 4] = perm(t23l, t01l, 0x07060302u);
          pw[2 * P_ROW / 4] = perm(t23h, t01h, 0x05040100u);
          pw[3 * P_ROW / 4] = perm(t23h, t01h, 0x07060302u);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          const v4i pa = *reinterpret_cast<const v4i*>(pl + n16 * P_ROW + quad * 16);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          const float mn = fmaxf(m[r], mb), mn0 = finite_or_0(mn);
          const float al = __builtin_amdgcn_exp2f(m[r] - mn0), eb = __builtin_amdgcn_exp2f(mb - mn0);
          const float be = eb * down;
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const v4i zero = {0, 0, 0, 0};
            const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, v[t], zero, 0, 0, 0);
            acc[r][t] = fmaf(undigit(d), be, acc[r][t] * al);
          }
          l[r] = fmaf(lp, eb, l[r] * al);
          m[r] = mn;
        }
      }
      // the end of a unit, or of the row
      if (!SPLIT && ((b + 1) % bpu == 0 || b + 1 == b1)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float lu = row_sum(l[r]);
          const float mn = fmaxf(M[r], m[r]), mn0 = finite_or_0(mn);
          const float x = __builtin_amdgcn_exp2f(M[r] - mn0), y = __builtin_amdgcn_exp2f(m[r] - mn0);
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            A[r][t] = fmaf(acc[r][t], y, A[r][t] * x);
            acc[r][t] = 0.0f;
          }
          L[r] = fmaf(lu, y, L[r] * x);
          M[r] = mn;
          m[r] = -INFINITY;
          l[r] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (SPLIT) {
        if (ps[r] < 0 || (int)unit >= unit_count(ps[r])) continue;
        const float lu = row_sum(l[r]);
        float* o = a.part + (((size_t)orow[r] * a.nh + ohead[r]) * a.units + unit) * (2 + DP);
        if (n16 == 0) {
          o[0] = m[r];
          o[1] = lu;
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) o[2 + 16 * t + n16] = acc[r][t];
      } else {
        // a pair without a position is written in the first pass
        const bool mine = have[r] && (ps[r] >= 0 || (pos[r] < 0 && ul == ul_first));
        if (!mine) continue;
        const float inv = L[r] == 0.0f ? 0.0f : 1.0f / L[r];
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const uint32_t d = 16 * t + n16;
          if (d < a.hd) store_value(a.out, (int64_t)orow[r] * a.os + (int64_t)ohead[r] * a.hd + d, a.type, A[r][t] * inv);
        }
      }
    }
  }
}

// Joins a row's units in order, as the unsplit kernel does. One workgroup of
// dp lanes per (row of a sequence, head).
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
  const uint32_t h = blockIdx.x % a.nh, j = blockIdx.x / a.nh % a.r.most_rows, seq = blockIdx.x / a.nh / a.r.most_rows;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  if (j >= (uint32_t)sp.n) return;
  const int64_t pos = min(sp.pos((int)j), a.most_len - 1);
  const uint32_t row = sp.start + j, d = threadIdx.x, dp = a.p.dp;
  const float* p = a.part + ((size_t)row * a.nh + h) * a.units * (2 + dp);
  const int n = unit_count(pos);
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  for (int u = 0; u < n; ++u, p += 2 + dp) {
    const float m = p[0], l = p[1], acc = p[2 + d];
    const float mn = fmaxf(M, m), mn0 = finite_or_0(mn);
    const float x = __builtin_amdgcn_exp2f(M - mn0), y = __builtin_amdgcn_exp2f(m - mn0);
    A = fmaf(acc, y, A * x);
    L = fmaf(l, y, L * x);
    M = mn;
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  if (d < a.hd) store_value(a.out, (int64_t)row * a.os + (int64_t)h * a.hd + d, a.type, A * inv);
}

// ------------------------------------------------------------- launches

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DEFER_GPU_OK : defer_gpu_fail_(DEFER_GPU_E_HIP, "launch: %s", hipGetErrorString(e));
}

template <bool NORM>
int rows_launch(uint32_t type, const NormArgs& a, uint32_t rows, hipStream_t s) {
  if (type == DEFER_GPU_F32)
    k_rows<float, NORM><<<rows, 256, 0, s>>>(a);
  else if (type == DEFER_GPU_BF16)
    k_rows<__bf16, NORM><<<rows, 256, 0, s>>>(a);
  else
    k_rows<_Float16, NORM><<<rows, 256, 0, s>>>(a);
  return launched();
}

template <int R, bool SPLIT>
void attn_launch(const AttnArgs& a, uint32_t blocks, hipStream_t s) {
  switch (a.p.dp / 64) {
    case 1: k_attn<1, R, SPLIT><<<blocks, 256, 0, s>>>(a); break;
    case 2: k_attn<2, R, SPLIT><<<blocks, 256, 0, s>>>(a); break;
    case 3: k_attn<3, R, SPLIT><<<blocks, 256, 0, s>>>(a); break;
    default: k_attn<4, R, SPLIT><<<blocks, 256, 0, s>>>(a); break;
  }
}

// How a call's pairs are dealt: tiles of 4 R pairs, units (0: unsplit).
struct Plan {
  uint32_t R, tiles, units;
};
Plan plan_of(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t dp, uint32_t most_len) {
  const uint32_t pairs = r.most_rows * (heads / kv_heads);
  Plan p;
  p.R = pairs <= 4 ? 1 : pairs <= 8 ? 2 : 4;
  p.tiles = (pairs + 4 * p.R - 1) / (4 * p.R);
  const uint64_t waves = (uint64_t)r.sequences * kv_heads * p.tiles;
  const int u = most_units(most_len);
  p.units = waves < 1024 && u > 1 ? (uint32_t)u : 0;
  (void)dp;
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

int linear(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* w, int64_t w_stride,
           const float* w_scale, uint32_t rows, uint32_t m, uint32_t k, uint32_t type, void* y,
           int64_t y_stride, hipStream_t s) {
  if (!rows) return DEFER_GPU_OK;
  const LinearArgs a{x, w, x_scale, w_scale, x_stride, w_stride, y_stride, y, rows, m, k, type};
  const bool aligned = ((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_stride | (uintptr_t)w_stride | k) % 16 == 0;
  const dim3 grid((m + 15) / 16, (rows + 63) / 64);
  if (rows <= 16) {
    if (aligned)
      k_linear_few<1, true><<<grid, 256, 0, s>>>(a);
    else
      k_linear_few<1, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (aligned)
      k_linear_few<4, true><<<grid, 256, 0, s>>>(a);
    else
      k_linear_few<4, false><<<grid, 256, 0, s>>>(a);
  }
  return launched();
}

static uint32_t kv_grid(const Pages& p, const Rows& r) {
  return r.sequences * p.heads * ((r.most_rows + PAGE - 2) / PAGE + 1);
}

int kv_write(const Pages& p, const Rows& r, uint32_t type, const void* k, int64_t k_stride, const void* v,
             int64_t v_stride, uint32_t head_dim, hipStream_t s) {
  if (!r.rows || !r.sequences || !r.most_rows) return DEFER_GPU_OK;
  const KvArgs a{p, r, const_cast<void*>(k), const_cast<void*>(v), k_stride, v_stride, type, head_dim};
  k_kv_write<<<kv_grid(p, r), 256, 0, s>>>(a);
  return launched();
}

int kv_read(const Pages& p, const Rows& r, uint32_t type, void* k, void* v, uint32_t head_dim, hipStream_t s) {
  if (!r.rows || !r.sequences || !r.most_rows) return DEFER_GPU_OK;
  const KvArgs a{p, r, k, v, 0, 0, type, head_dim};
  Rows and_one = r;
  and_one.sequences += r.row_start != nullptr;
  k_kv_read<<<kv_grid(p, and_one), 256, 0, s>>>(a);
  return launched();
}

size_t attention_workspace(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t most_len) {
  if (!r.rows || !r.sequences || !r.most_rows) return 0;
  const uint32_t dp = padded(head_dim);
  const Plan pl = plan_of(r, heads, kv_heads, dp, most_len);
  return (size_t)r.rows * heads * pl.units * (2 + dp) * sizeof(float);
}

int attention(const Pages& p, const Rows& r, const Attention& in, void* workspace, size_t workspace_bytes,
              hipStream_t s) {
  if (!r.rows || !r.sequences || !r.most_rows) return DEFER_GPU_OK;
  const Plan pl = plan_of(r, in.heads, p.heads, p.dp, in.most_len);
  const size_t need = attention_workspace(r, in.heads, p.heads, in.head_dim, in.most_len);
  if (need && (!workspace || workspace_bytes < need))
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "attention needs a workspace of %zu bytes, got %zu", need,
                           workspace ? workspace_bytes : (size_t)0);
  AttnArgs a{};
  a.p = p;
  a.r = r;
  a.q = in.q;
  a.out = in.out;
  a.qs = in.q_stride;
  a.os = in.out_stride;
  a.type = in.type;
  a.nh = in.heads;
  a.group = in.heads / p.heads;
  a.hd = in.head_dim;
  a.tiles = pl.tiles;
  a.units = pl.units;
  a.most_len = in.most_len;
  a.scale2 = in.scale * 1.44269504088896340736f;
  a.hidden = in.hidden;
  a.hs = in.hidden_stride;
  a.hidden_len = in.hidden_len;
  a.part = static_cast<float*>(workspace);
  const uint64_t items = (uint64_t)pl.tiles * std::max(pl.units, 1u);
  const uint64_t blocks = (items + 3) / 4 * r.sequences * p.heads;
  if (blocks > 0x7fffffffu || (uint64_t)r.sequences * r.most_rows * in.heads > 0x7fffffffu)
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "too many rows for one call");
  const uint32_t nb = (uint32_t)blocks;
  if (pl.units) {
    if (pl.R == 1)
      attn_launch<1, true>(a, nb, s);
    else if (pl.R == 2)
      attn_launch<2, true>(a, nb, s);
    else
      attn_launch<4, true>(a, nb, s);
    k_attn_join<<<r.sequences * r.most_rows * in.heads, p.dp, 0, s>>>(a);
  } else {
    if (pl.R == 1)
      attn_launch<1, false>(a, nb, s);
    else if (pl.R == 2)
      attn_launch<2, false>(a, nb, s);
    else
      attn_launch<4, false>(a, nb, s);
  }
  return launched();
}

}  // namespace q8

// ------------------------------------------------------------- C entry points

using namespace q8;

#define Q8_REQUIRE(cond, ...)                                              \
  do {                                                                     \
    if (!(cond)) return defer_gpu_fail_(DEFER_GPU_E_INVALID, __VA_ARGS__); \
  } while (0)

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
static size_t value_size(uint32_t type) { return type == DEFER_GPU_F32 ? 4 : 2; }
static bool aligned_to(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

static int check_rows_values(uint32_t type, const void* x, int64_t stride, uint32_t rows, uint32_t n, const char* what) {
  Q8_REQUIRE(type <= DEFER_GPU_F16, "value type %u", type);
  Q8_REQUIRE(n >= 1 && n <= 0x7fffffffu && rows <= 0x7fffffffu, "%s: %u rows of %u values", what, rows, n);
  Q8_REQUIRE(rows == 0 || x, "%s is null", what);
  Q8_REQUIRE(rows <= 1 || stride >= (int64_t)n, "%s: rows of %u values %lld apart", what, n, (long long)stride);
  Q8_REQUIRE(aligned_to(x, value_size(type)), "%s is not aligned to its type", what);
  return DEFER_GPU_OK;
}

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
  Q8_REQUIRE((rows + 63) / 64 <= 65535, "%u rows: at most 4,194,240 in one call", rows);
  Q8_REQUIRE(rows == 0 || (x && x_scale), "null x");
  Q8_REQUIRE(w && w_scale, "null w");
  Q8_REQUIRE(rows <= 1 || x_stride >= (int64_t)k, "x: rows of %u codes %lld apart", k, (long long)x_stride);
  Q8_REQUIRE(m <= 1 || w_stride >= (int64_t)k, "w: rows of %u codes %lld apart", k, (long long)w_stride);
  return linear(x, x_stride, x_scale, w, w_stride, w_scale, rows, m, k, type, y, y_stride, (hipStream_t)stream);
}

static int check_pages(const defer_gpu_q8_pages* p, const defer_gpu_q8_rows* r, Pages* pages, Rows* rows) {
  Q8_REQUIRE(p && r, "null argument");
  Q8_REQUIRE(p->head_dim >= 1 && p->head_dim <= MAX_HEAD_DIM, "head_dim %u: 1 to %u", p->head_dim, MAX_HEAD_DIM);
  Q8_REQUIRE(p->heads >= 1 && p->heads <= 65535, "%u cache heads", p->heads);
  Q8_REQUIRE(p->pages <= 0x7fffffffu && p->table_width <= 0x7fffffffu / PAGE, "%u pages, %u a sequence", p->pages,
             p->table_width);
  Q8_REQUIRE(r->rows <= 0x7fffffffu && r->sequences <= 0x7fffffffu, "%u rows of %u sequences", r->rows, r->sequences);
  Q8_REQUIRE(r->most_rows <= r->rows, "most_rows %u of %u rows", r->most_rows, r->rows);
  *rows = Rows{r->row_start, r->kv_len, r->sequences, r->rows, r->most_rows};
  *pages = Pages{p->keys, p->values, p->key_scale, p->value_scale, p->table, p->pages, p->heads,
                 padded(p->head_dim), p->table_width, nullptr, 0};
  if (!r->rows || !r->sequences || !r->most_rows) return DEFER_GPU_OK;
  Q8_REQUIRE(r->row_start || r->rows == r->sequences, "%u rows of %u sequences without row_start", r->rows, r->sequences);
  Q8_REQUIRE(r->kv_len, "kv_len is null");
  Q8_REQUIRE(p->table_width == 0 || p->table, "table is null");
  Q8_REQUIRE(p->pages == 0 || (p->keys && p->values && p->key_scale && p->value_scale), "null pages");
  Q8_REQUIRE(aligned16(p->keys) && aligned16(p->values) && aligned16(p->key_scale) && aligned16(p->value_scale),
             "pages are not 16-byte aligned");
  Q8_REQUIRE(((uint64_t)r->sequences + 1) * p->heads * ((r->most_rows + PAGE - 2) / PAGE + 1) <= 0x7fffffffu,
             "too many rows for one call");
  return DEFER_GPU_OK;
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

static int check_heads(const defer_gpu_q8_pages* p, uint32_t q_heads, uint32_t most_len) {
  Q8_REQUIRE(q_heads >= 1 && q_heads <= 65535 && q_heads % p->heads == 0, "%u query heads on %u cache heads", q_heads,
             p->heads);
  Q8_REQUIRE(most_len <= 0x7fffffffu, "most_len %u", most_len);
  return DEFER_GPU_OK;
}

extern "C" size_t defer_gpu_q8_attention_workspace(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows,
                                                   uint32_t q_heads, uint32_t most_len) {
  if (!pages || !rows || !pages->heads || !q_heads || pages->head_dim > MAX_HEAD_DIM) return 0;
  const Rows r{rows->row_start, rows->kv_len, rows->sequences, rows->rows, rows->most_rows};
  return attention_workspace(r, q_heads, pages->heads, pages->head_dim, most_len);
}

extern "C" int defer_gpu_q8_attention(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                      const void* q, int64_t q_stride, uint32_t q_heads, uint32_t most_len,
                                      float scale, const uint8_t* hidden, int64_t hidden_stride,
                                      uint32_t hidden_len, void* out, int64_t out_stride, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  Pages p;
  Rows r;
  int rc = check_pages(pages, rows, &p, &r);
  if (!rc) rc = check_heads(pages, q_heads, most_len);
  if (rc) return rc;
  const uint32_t n = q_heads * pages->head_dim;
  rc = check_rows_values(type, q, q_stride, r.rows, n, "q");
  if (!rc) rc = check_rows_values(type, out, out_stride, r.rows, n, "out");
  if (rc) return rc;
  Q8_REQUIRE(!hidden || r.sequences <= 1 || hidden_stride >= (int64_t)hidden_len, "hidden: rows of %u, %lld apart",
             hidden_len, (long long)hidden_stride);
  Q8_REQUIRE(aligned16(workspace), "workspace is not 16-byte aligned");
  Attention a{type, q, q_stride, out, out_stride, q_heads, pages->head_dim, scale, most_len, hidden, hidden_stride,
              hidden_len};
  return attention(p, r, a, workspace, workspace_bytes, (hipStream_t)stream);
}
