// q8_draft.hip -- what a program that drafts tokens and verifies them needs
// around the attention: rows normed, rotated and appended to the cache in one
// launch, the log probabilities of given tokens, and the accepted path moved
// together in the cache. (The attention of a tree of drafts is in q8_tree.hip.)
#include "q8_common.h"

#include <float.h>

#include <algorithm>

namespace q8 {

namespace {

// ------------------------------------------------------------- append

struct AppendArgs {
  Pages p;
  Rows r;
  const void *q, *k, *v;
  void* out;
  int64_t qs, ks, vs, os;
  const int32_t* position;
  const double* freq;
  const void *qn, *kn;
  double eps, factor;
  uint32_t hd, nh, half;        // half: rotated pairs of a head
  uint32_t kv_shift, q_shift;   // a workgroup takes so many heads, as a power of 2: of the cache, or of the queries
  uint32_t kv_chunks, chunks;   // workgroups of a run for the cache's heads, and for all
  bool interleaved;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// (Written out: the compiler quiets both operands first. Another lane reads a register two wait
// states after it was written.)
__device__ __forceinline__ double max_abs(double v, double x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_max_f64 %0, %0, |%1|\n\ts_nop 1" : "+v"(v) : "v"(x));
#endif
  return v;
}
// Over the 16 lanes of a DPP row, as row_max and row_sum; the maximum of numbers that are not negative.
__device__ __forceinline__ double row_max64(double v) {
  v = max_abs(v, dpp64<0x128>(v));
  v = max_abs(v, dpp64<0x124>(v));
  v = max_abs(v, dpp64<0x122>(v));
  return max_abs(v, dpp64<0x121>(v));
}
__device__ __forceinline__ double row_sum64(double v) {
  v += dpp64<0x128>(v);
  v += dpp64<0x124>(v);
  v += dpp64<0x122>(v);
  return v + dpp64<0x121>(v);
}

// (cos, sin) of position times frequency, in 64 bits: as turns, of which the
// whole ones go, then the quarters; what is left is within an eighth of a turn,
// where the series to x^15 and x^16 are off by less than 2^-54 (their next terms,
// x^17 / 17! and x^18 / 18!). The turns are products in two parts each, so that no position is too far.
__device__ __forceinline__ double2 turn(int pos, double freq) {
  constexpr double PER = 0.15915494309189533577, LEFT = -9.839338337591251e-18;  // 1 / (2 pi) in two parts
  const double p = (double)pos, f = freq * PER, fl = fma(freq, PER, -f) + freq * LEFT;
  const double h = p * f;
  double t = (h - rint(h)) + (fma(p, f, -h) + p * fl);
  t -= rint(t);
  const double quarter = rint(4.0 * t), x = (t - 0.25 * quarter) * 6.28318530717958647693, x2 = x * x;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, x2, 1.0 / 6227020800.0);
  c = fma(c, x2, -1.0 / 87178291200.0);
  s = fma(s, x2, -1.0 / 39916800.0);
  s = fma(s, x2, 1.0 / 362880.0);
  s = fma(s, x2, -1.0 / 5040.0);
  s = fma(s, x2, 1.0 / 120.0);
  s = fma(s, x2, -1.0 / 6.0);
  s = fma(s * x2, x, x);
  c = fma(c, x2, 1.0 / 479001600.0);
  c = fma(c, x2, -1.0 / 3628800.0);
  c = fma(c, x2, 1.0 / 40320.0);
  c = fma(c, x2, -1.0 / 720.0);
  c = fma(c, x2, 1.0 / 24.0);
  c = fma(c, x2, -0.5);
  c = fma(c, x2, 1.0);
  const int n = (int)quarter & 3;
  const double a = n & 1 ? s : c, b = n & 1 ? c : s;
  return double2{n == 1 || n == 2 ? -a : a, n >= 2 ? -b : b};
}

// 8 values of a head.
template <class T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8), aligned(16)));
};

// Where pair `i` of a row's (cos, sin) lies in LDS: lanes that take 8 values each (and so 8 or,
// side by side, 4 pairs) read neighbouring ones.
struct Angles {
  uint32_t step, line;  // pairs of a lane, and places of each of them
  __device__ __forceinline__ Angles(uint32_t half, bool interleaved) : step(interleaved ? 4 : 8), line((half + step - 1) / step) {}
  __device__ __forceinline__ uint32_t at(uint32_t i) const { return i % step * line + i / step; }
};
// ... of a row.
Q8_HD uint32_t angles_of(uint32_t half, bool interleaved) {
  const uint32_t step = interleaved ? 4 : 8;
  return (half + step - 1) / step * step;
}

// The codes of a lane's values at a scale. A quotient in f32 is off by less than
// 2^-15 (three roundings of up to 127), so only where one of the wave's lies that near a half
// does it take 64 bits to say on which side.
template <uint32_t W>
struct Codes {
  uint64_t c[W];
  __device__ __forceinline__ Codes(const double (*y)[8], float scale) {
    const float r = scale > 0.0f ? 1.0f / scale : 0.0f;  // (zeros, and rows with what is no number: codes 0)
    float off = 0.0f;
    int q[W][8];
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) {
        const float x = r > 0.0f ? (float)y[w][e] * r : 0.0f, n = rintf(x);
        off = fmaxf(off, fabsf(x - n));
        q[w][e] = (int)n;
      }
    if (__any(!(off < 0.5f - 0x1p-14f) || scale > 0x1p118f)) {  // (values that f32 may not hold)
      const Coder code(scale);
#pragma unroll
      for (uint32_t w = 0; w < W; ++w)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) q[w][e] = code(y[w][e]);
    }
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      uint32_t h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        h[i] = perm(perm((uint32_t)q[w][4 * i + 3], (uint32_t)q[w][4 * i + 2], 0x0c0c0400u),
                    perm((uint32_t)q[w][4 * i + 1], (uint32_t)q[w][4 * i], 0x0c0c0400u), 0x05040100u);
      c[w] = (uint64_t)h[1] << 32 | h[0];
    }
  }
};

// A workgroup takes the rows of 16 places of a page (as k_kv_write's, whose
// places they are) and some heads: of the cache's keys and values, or of the
// queries. The rows' angles are formed once, 64 bits, in LDS; then 16 lanes take
// a row's head, 8 values each (WIDE: and the 8 from 128 on), the next one's already on its
// way. Keys, scales and codes are those of the formula in 64 bits, as everywhere here.
// VEC: 8 values are aligned, and so are the 8 they are paired with.
//
// y = x w / sqrt(mean(x^2) + eps), or x; a pair (a, b) at an angle t becomes factor (a cos t - b
// sin t, b cos t + a sin t). Every value is read once, but for the half layout's pairs, which lie
// 8 lanes off and come from L1 the second time.
//
// One row, 9 + 3 heads of 64, f32: 4.4 us, the chain of lengths, page, values and a launch. 64 such
// rows of 32 + 8 heads 6.2. 2000 rows of 32 + 8 bf16 heads of 128, 45 MB: 21.6 us, 2.1 TB/s, where
// a copy of the queries and a cache write alone take 7.9 + 9.1. The rotation is about 4 of them (without
// it 17.5); what bounds the rest is not measured. The half layout reads every rotated value twice,
// and the queries' workgroups hold the registers of the codes' path, four waves a SIMD. Two items on their
// way instead of one cost registers (27 us), angles formed anew by each lane 48.
template <class T, bool VEC, bool WIDE>
__global__ __launch_bounds__(256) void k_append(AppendArgs a) {
  typedef typename Eight<T>::type t8;
  constexpr uint32_t W = WIDE ? 2 : 1;
  extern __shared__ __align__(16) uint8_t lds[];  // the rows' angles, then [heads][rows][KV_ROW] value codes
  const uint32_t per = kv_runs(a.r.most_rows), most = min(a.r.most_rows, (uint32_t)KV_RUN);
  const uint32_t chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks % per, seq = blockIdx.x / a.chunks / per;
  const uint32_t n16 = threadIdx.x % 16, quad = threadIdx.x / 16, hd = a.hd, rotated = 2 * a.half;
  constexpr uint32_t quads = 16;
  T* const out = static_cast<T*>(a.out);
  if (seq >= a.r.sequences) {  // zeros for the rows of no sequence
    const int64_t lo = span_of(a.r.row_start, a.r.kv_len, 0, a.r.rows).start;
    const int64_t hi = max(lo, min((int64_t)a.r.row_start[a.r.sequences], (int64_t)a.r.rows));
    const uint32_t first = a.r.sequences * per * a.chunks;
    const int64_t n = a.nh * hd;
    for (int64_t i = blockIdx.x - first; i < lo + ((int64_t)a.r.rows - hi); i += gridDim.x - first) {
      const int64_t row = i < lo ? i : hi + (i - lo);
      for (int64_t d = threadIdx.x; d < n; d += blockDim.x) out[row * a.os + d] = (T)0.0f;
    }
    return;
  }
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  auto down = [](int64_t t, int n) { return t >= 0 ? t / n : -((-t + n - 1) / n); };
  const int64_t p0 = sp.pos(0), run = down(p0, KV_RUN) + b;
  const int64_t t0 = max(p0, run * KV_RUN), t1 = min((int64_t)sp.len, (run + 1) * KV_RUN);
  if (t0 >= t1) return;
  const uint32_t n = min((uint32_t)(t1 - t0), most);  // rows
  const int64_t row0 = sp.start + (t0 - p0);
  const bool queries = chunk >= a.kv_chunks;
  const uint32_t shift = queries ? a.q_shift : a.kv_shift, h0 = (queries ? chunk - a.kv_chunks : chunk) << shift;
  const uint32_t heads = min(1u << shift, (queries ? a.nh : a.p.heads) - h0);
  // keys and values that have a place and a page (places before 0 have none)
  const int64_t block = down(run, PAGE / KV_RUN);
  int page = 0;
  if (!queries) {
    page = page_of(a.p.table + (size_t)seq * a.p.width, a.p.width, a.p.pages, block);
    if (page < 0) return;
  }
  const uint32_t turning = n << shift, items = queries ? turning : 2 * turning;  // keys, then values; of 2^shift heads

  auto load = [&](const T* p, uint32_t d) {
    t8 v;
    if (VEC && d < hd) {
      v = *reinterpret_cast<const t8*>(p + d);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) v[e] = d + e < hd ? p[d + e] : (T)0.0f;
    }
    return v;
  };
  // the values that a half layout pairs with the 8 from d on
  auto load_pairs = [&](const T* p, uint32_t d) {
    t8 v;
    if (VEC && d < rotated) {
      v = *reinterpret_cast<const t8*>(p + (d < a.half ? d + a.half : d - a.half));
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) v[e] = d + e < rotated ? p[d + e < a.half ? d + e + a.half : d + e - a.half] : (T)0.0f;
    }
    return v;
  };
  t8 x[W], xp[W];
  auto fetch = [&](uint32_t i) {
    const uint32_t it = i < turning ? i : i - turning, j = it >> shift, hl = it & ((1u << shift) - 1);
    const T* p = queries       ? static_cast<const T*>(a.q) + (row0 + j) * a.qs
                 : i < turning ? static_cast<const T*>(a.k) + (row0 + j) * a.ks
                               : static_cast<const T*>(a.v) + (row0 + j) * a.vs;
    p += (int64_t)(h0 + min(hl, heads - 1)) * hd;  // (none: another's, not used)
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      x[w] = load(p, 128 * w + 8 * n16);
      if (!a.interleaved && i < turning) xp[w] = load_pairs(p, 128 * w + 8 * n16);
    }
  };
  if (quad < items) fetch(quad);
  const T* const norm = static_cast<const T*>(queries ? a.qn : a.kn);
  t8 weight[W], weight_p[W];
  if (norm) {
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      weight[w] = load(norm, 128 * w + 8 * n16);
      if (!a.interleaved) weight_p[w] = load_pairs(norm, 128 * w + 8 * n16);
    }
  }

  const uint32_t of_row = angles_of(a.half, a.interleaved);
  const Angles angles(a.half, a.interleaved);
  double2* const cs = reinterpret_cast<double2*>(lds);
  int8_t* const tile = reinterpret_cast<int8_t*>(cs + most * of_row);
  for (uint32_t i = threadIdx.x; i < n * a.half; i += 256) {
    const uint32_t j = i / a.half, pair = i - j * a.half;
    const double2 c = turn(a.position ? a.position[row0 + j] : (int)(t0 + j), a.freq[pair]);
    cs[j * of_row + angles.at(pair)] = double2{c.x * a.factor, c.y * a.factor};
  }
  __syncthreads();

  const int a0 = (int)(t0 - block * PAGE);  // the first row's place in its page
  for (uint32_t i = quad; i < items; i += quads) {
    const bool value = i >= turning;
    const uint32_t it = value ? i - turning : i, j = it >> shift, hl = it & ((1u << shift) - 1), h = h0 + hl;
    double y[W][8];
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) y[w][e] = (double)(float)x[w][e];
    if (!value) {
      double inv = 1.0;
      if (norm) {
        double ss = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w)
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) ss = fma(y[w][e], y[w][e], ss);
        inv = 1.0 / sqrt(row_sum64(ss) / (double)hd + a.eps);
#pragma unroll
        for (uint32_t w = 0; w < W; ++w)
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) y[w][e] *= (double)(float)weight[w][e] * inv;
      }
      const double2* const row = cs + j * of_row;
#pragma unroll
      for (uint32_t w = 0; w < W; ++w) {
        const uint32_t d = 128 * w + 8 * n16;
        if (VEC ? d >= rotated : false) continue;
        if (a.interleaved) {
#pragma unroll
          for (uint32_t e = 0; e < 8; e += 2) {
            if (!VEC && d + e >= rotated) continue;
            const double2 c = row[e / 2 * angles.line + d / 8];
            const double p = y[w][e], q = y[w][e + 1];
            y[w][e] = fma(p, c.x, -(q * c.y));
            y[w][e + 1] = fma(q, c.x, p * c.y);
          }
        } else {
          const bool all_second = d >= a.half;  // (VEC: all of them or none)
          const double2* const from = row + (all_second ? d - a.half : d) / 8;
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) {
            const uint32_t k = d + e;
            if (!VEC && k >= rotated) continue;
            const bool second = VEC ? all_second : k >= a.half;
            const double2 c = VEC ? from[e * angles.line] : row[angles.at(second ? k - a.half : k)];
            const float of = (float)xp[w][e];
            double o = (double)(second ? of : -of);
            if (norm) o *= (double)(float)weight_p[w][e] * inv;
            y[w][e] = fma(o, c.y, y[w][e] * c.x);
          }
        }
      }
    }
    if (i + quads < items) fetch(i + quads);
    if (hl >= heads) continue;
    if (queries) {
      T* const to = out + (row0 + j) * a.os + (int64_t)h * hd;
#pragma unroll
      for (uint32_t w = 0; w < W; ++w) {
        const uint32_t d = 128 * w + 8 * n16;
        t8 v;  // (through f32: at most half a step of it more than rounded at once)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = (T)(float)y[w][e];
        if (VEC && d < hd) {
          *reinterpret_cast<t8*>(to + d) = v;
        } else {
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e)
            if (d + e < hd) to[d + e] = v[e];
        }
      }
      continue;
    }
    double top = 0.0, bad = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) {
        top = max_abs(top, y[w][e]);
        bad = fma(y[w][e], 0.0, bad);
      }
    const float scale = scale_of(row_max64(top), isnan(row_sum64(bad)));
    const Codes<W> codes(y, scale);
    const size_t hp = (size_t)page * a.p.heads + h;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      const uint32_t d = 128 * w + 8 * n16;
      if (d >= hd) continue;
      // a page's row is a multiple of 64 codes: those behind hd are zeros
      if (value)
        *reinterpret_cast<uint64_t*>(tile + (hl * most + j) * KV_ROW + d) = codes.c[w];
      else
        *reinterpret_cast<uint64_t*>(a.p.keys + (hp * PAGE + a0 + j) * a.p.dp + d) = codes.c[w];
    }
    if (n16 == 0) (value ? a.p.value_scale : a.p.key_scale)[hp * PAGE + a0 + j] = scale;
  }
  if (queries) return;
  __syncthreads();
  // value codes into their transposed pages
  int8_t* const vc = a.p.values + ((size_t)page * a.p.heads + h0) * PAGE * a.p.dp;
  if (n < KV_RUN) {  // some of the run: byte by byte
    for (uint32_t i = threadIdx.x; i < heads * n * hd; i += 256) {
      const uint32_t d = i % hd, hj = i / hd, j = hj % n, hl = hj / n;
      vc[((size_t)hl * a.p.dp + d) * PAGE + a0 + j] = tile[(hl * most + j) * KV_ROW + d];
    }
    return;
  }
  const uint32_t quarters = (hd + 3) / 4;
  for (uint32_t i = threadIdx.x; i < heads * quarters; i += 256) {  // four channels a thread
    const uint32_t hl = i / quarters, d = 4 * (i % quarters);
    uint32_t w[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t in[4], by[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = *reinterpret_cast<const uint32_t*>(tile + (hl * most + 4 * u + e) * KV_ROW + d);
      transpose4(in, by);
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c][u] = by[c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (d + c < hd)
        *reinterpret_cast<v4i*>(vc + ((size_t)hl * a.p.dp + d + c) * PAGE + a0) =
            v4i{(int)w[c][0], (int)w[c][1], (int)w[c][2], (int)w[c][3]};
  }
}

template <class T>
int append_launch(const AppendArgs& a, uint32_t blocks, size_t lds, bool vec, hipStream_t s) {
  if (a.hd <= 128) return launch(vec ? k_append<T, true, false> : k_append<T, false, false>, blocks, 256, lds, s, a);
  return launch(vec ? k_append<T, true, true> : k_append<T, false, true>, blocks, 256, lds, s, a);
}

// ------------------------------------------------------------- keep

struct KeepArgs {
  Pages p;
  Rows r;
  const int32_t *keep, *kept;
  int32_t* kv_len_out;
  uint32_t hd;
};

// One workgroup for a sequence and head: its kept rows' codes and scales all
// come into LDS, then go to their new places, so that the order of rows and
// places that are both does not matter. A chain of dependent reads (lengths, entry, page,
// codes) bounds it: 4.1 us for one sequence of 3 heads of 64, 7.2 for 64 of 8 heads of 128, of
// whose values each byte lies in a line of its own.
__global__ __launch_bounds__(256) void k_keep(KeepArgs a) {
  const uint32_t g = blockIdx.x % a.p.heads, seq = blockIdx.x / a.p.heads;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const int move = min(min(max(a.kept[seq], 0), sp.n), (int)a.r.most_rows);  // rows that stay
  if (g == 0 && threadIdx.x == 0) a.kv_len_out[seq] = (int32_t)max(sp.pos(move), (int64_t)INT32_MIN);
  __shared__ __align__(16) int8_t keys[MAX_TREE * 256], values[MAX_TREE * 256];
  __shared__ float scales[2][MAX_TREE];
  __shared__ int64_t from[MAX_TREE], to[MAX_TREE];  // places: page * 64 + position, or -1
  if (move <= 0) return;
  auto place = [&](int64_t pos) -> int64_t {
    const int page = pos < 0 ? -1 : page_of(a.p.table + (size_t)seq * a.p.width, a.p.width, a.p.pages, pos / PAGE);
    return page < 0 ? -1 : (int64_t)page * PAGE + pos % PAGE;
  };
  for (int t = threadIdx.x; t < move; t += blockDim.x) {
    const int j = a.keep[sp.start + t];
    const int64_t f = j >= 0 && j < sp.n && j != t ? place(sp.pos(j)) : -1;
    from[t] = f;
    to[t] = f < 0 ? -1 : place(sp.pos(t));
  }
  __syncthreads();
  const uint32_t dp = a.p.dp;
  auto head = [&](int64_t at) { return (size_t)(at / PAGE) * a.p.heads + g; };  // of a place
  // keys by 16 bytes, values by the byte: rows fastest, so that lanes share a line
  for (uint32_t i = threadIdx.x; i < move * dp / 16; i += blockDim.x) {
    const uint32_t t = i / (dp / 16), d = i % (dp / 16) * 16;
    if (to[t] >= 0)
      *reinterpret_cast<v4i*>(keys + t * 256 + d) =
          *reinterpret_cast<const v4i*>(a.p.keys + (head(from[t]) * PAGE + from[t] % PAGE) * dp + d);
  }
  for (uint32_t i = threadIdx.x; i < move * a.hd; i += blockDim.x) {
    const uint32_t t = i % move, d = i / move;
    if (to[t] >= 0) values[t * 256 + d] = a.p.values[(head(from[t]) * dp + d) * PAGE + from[t] % PAGE];
  }
  for (int t = threadIdx.x; t < move; t += blockDim.x)
    if (to[t] >= 0) {
      scales[0][t] = a.p.key_scale[head(from[t]) * PAGE + from[t] % PAGE];
      scales[1][t] = a.p.value_scale[head(from[t]) * PAGE + from[t] % PAGE];
    }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < move * dp / 16; i += blockDim.x) {
    const uint32_t t = i / (dp / 16), d = i % (dp / 16) * 16;
    if (to[t] >= 0)
      *reinterpret_cast<v4i*>(a.p.keys + (head(to[t]) * PAGE + to[t] % PAGE) * dp + d) =
          *reinterpret_cast<const v4i*>(keys + t * 256 + d);
  }
  for (uint32_t i = threadIdx.x; i < move * a.hd; i += blockDim.x) {
    const uint32_t t = i % move, d = i / move;
    if (to[t] >= 0) a.p.values[(head(to[t]) * dp + d) * PAGE + to[t] % PAGE] = values[t * 256 + d];
  }
  for (int t = threadIdx.x; t < move; t += blockDim.x)
    if (to[t] >= 0) {
      a.p.key_scale[head(to[t]) * PAGE + to[t] % PAGE] = scales[0][t];
      a.p.value_scale[head(to[t]) * PAGE + to[t] % PAGE] = scales[1][t];
    }
}

// ------------------------------------------------------------- log probabilities

constexpr int SCORE_EACH = 16, SCORE_CHUNK = SCORE_EACH * WAVE;  // logits of a lane, and of a wave
constexpr int SCORE_THREADS = 256, SCORE_WAVES = SCORE_THREADS / WAVE;
constexpr int SCORE_GROUP = 8, SCORE_GROUPS = WAVE / SCORE_GROUP;  // lanes whose logits have a maximum together
constexpr uint32_t SCORE_FEW = 2048;               // candidates for the best that a row may have in LDS
constexpr uint32_t SCORE_LIST = 1024;              // ... and groups that they come from

// What a wave leaves of its chunk of a row.
struct ScorePart {
  float top, sum, moment;  // maximum m; sum of e = 2^t, t = scale log2(e) (x - m) + r, and of e t
  uint32_t above;          // logits over the target's; SCORE_FAR: r is 0
};
constexpr uint32_t SCORE_FAR = 1u << 31;
// A logit's t is one fused product: fma(x, unit, -c), c = unit m rounded, which is r too large for
// all of a wave's, r = fma(m, unit, -c) without a rounding: the sum is 2^r times too
// large, the moment has r times it to lose.
__device__ __forceinline__ float score_over(float m, float unit) { return fmaf(m, unit, -(m * unit)); }

struct ScoreArgs {
  const void* x;
  int64_t xs;
  const int32_t* target;
  uint32_t rows, n, top, chunks;
  float scale;
  float *log_p, *entropy, *top_log_p;
  int32_t *rank, *top_index;
  ScorePart* part;   // [rows][chunks]
  uint32_t* maxima;  // [rows][chunks][8], for the best: score_order's
};

// A whole number that orders logits by value (-0 is 0), and back; no logit's is 0. (A
// NaN's is anywhere: its row has no best.)
__device__ __forceinline__ uint32_t score_order(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b ^ (uint32_t)((int32_t)b >> 31 | (int32_t)0x80000000);
}
__device__ __forceinline__ float of_order(uint32_t o) {
  return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}
// ... and one that orders equal ones by the lower column.
__device__ __forceinline__ uint64_t score_key(float v, uint32_t column) {
  return (uint64_t)score_order(v) << 32 | (0xffffffffu - column);
}
__device__ __forceinline__ uint32_t column_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) { return of_order((uint32_t)(key >> 32)); }

// A bound that `top` of the wave's numbers reach and at most `slack` more, unless they are equal;
// 0 if fewer are over 0. Steps down from the largest, then halves.
__device__ __forceinline__ uint32_t score_bound(uint32_t o, uint32_t top, uint32_t slack) {
  uint32_t most = o;
  for (int s = 32; s > 0; s >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, s));
  most = (uint32_t)__builtin_amdgcn_readfirstlane((int)most);
  uint32_t lo = 0, hi = most + 1, step = 1u << 20;  // `top` reach lo (or it is 0), fewer reach hi
  while (hi - lo > 1) {
    const uint32_t t = lo ? lo + (hi - lo) / 2 : most > step ? most - step : 1;
    const uint32_t n = (uint32_t)__popcll(__ballot(o >= t));
    if (n >= top) {
      lo = t;
      if (n <= top + slack) break;
    } else {
      hi = t;
      step = step >= 1u << 30 ? 0xffffffffu : step * 4;
    }
  }
  return lo;
}

// The `top` largest of `count` different keys in LDS, in their order, by one wave, which
// gathers those over a bound at their front and ranks them; two of them a lane are enough
// but for rows of many equal logits.
template <class F>
__device__ __forceinline__ void score_pick(uint64_t* keys, uint32_t count, uint32_t top, F store) {
  const uint32_t lane = threadIdx.x % WAVE;
  auto meet = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  if (count > WAVE) {
    uint32_t o = 0;
    for (uint32_t i = lane; i < count; i += WAVE) o = max(o, (uint32_t)(keys[i] >> 32));
    const uint32_t bound = score_bound(o, top, top / 4);
    uint32_t n = 0;
    for (uint32_t i = lane; i < (count + WAVE - 1) / WAVE * WAVE; i += WAVE) {
      const uint64_t k = i < count ? keys[i] : 0;
      const bool is = k && (uint32_t)(k >> 32) >= bound;
      const uint64_t mask = __ballot(is);
      meet();
      if (is) keys[n + (uint32_t)__popcll(mask & ((1ull << lane) - 1))] = k;
      n += (uint32_t)__popcll(mask);
    }
    count = n;
    meet();
  }
  if (count <= 2 * WAVE) {
    const uint64_t k0 = lane < count ? keys[lane] : 0, k1 = lane + WAVE < count ? keys[lane + WAVE] : 0;
    uint32_t b0 = 0, b1 = 0;
    auto against = [&](uint64_t k, int n) {
      for (int i = 0; i < n; ++i) {
        const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), i) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, i);
        b0 += o > k0;
        b1 += o > k1;
      }
    };
    against(k0, (int)min(count, (uint32_t)WAVE));
    if (count > WAVE) against(k1, (int)(count - WAVE));
    if (lane < count && b0 < top) store(b0, k0);
    if (lane + WAVE < count && b1 < top) store(b1, k1);
    return;
  }
  for (uint32_t i = lane; i < count; i += WAVE) {
    const uint64_t k = keys[i];
    uint32_t before = 0;
    for (uint32_t j = 0; j < count; ++j) before += keys[j] > k;
    if (before < top) store(before, k);
  }
}

// Maxima and sums over lanes, a step an instruction: CTRL names the lanes that are read, ROWS the
// rows of 16 that read them.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t max_step(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float add_step(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
// Over 8 neighbouring lanes: in each of them.
__device__ __forceinline__ uint32_t max_of_8(uint32_t v) {
  return max_step<0x141>(max_step<0x4e>(max_step<0xb1>(v)));  // quad_perm 1 0 3 2, 2 3 0 1, row_half_mirror
}
// Over the wave, of numbers that are the same in 8 neighbouring lanes: in all of it.
__device__ __forceinline__ uint32_t max_of_wave(uint32_t v) {
  v = max_step<0x143, 0xc>(max_step<0x142, 0xa>(max_step<0x140>(v)));  // row_mirror, row_bcast 15, 31
  return (uint32_t)__builtin_amdgcn_readlane((int)v, WAVE - 1);
}
// Over the wave: in its last lane.
__device__ __forceinline__ float sum_of_wave(float v) { return add_step<0x143, 0xc>(add_step<0x142, 0xa>(row_sum(v))); }

// A wave takes a chunk of a row, in registers, 16 logits a lane, read once; its sums are
// relative to its own maximum m. For the best, the maxima of groups of lanes are left:
// k_score_join reads the few groups again that can hold one. Where m is so far out that the
// product that t comes from would be, or a logit is infinitely far below (t is -inf, the moment
// NaN), x - m comes first.
//
// 2047 rows of 128,256 bf16: 92 us, 5.7 TB/s, where a plain read takes 84; with the best's maxima
// and targets 98; f32 178 of 169. Rows that are not aligned to 16 bytes are read by the logit, each lane's
// 16 bytes from the next one's (61 of 128,256 f32, 31 MB: 11.2). A chunk with a logit of -inf, or with the
// row's end in it, is summed twice. Bound by memory and, nearly as much, by vector instructions (about 150 a
// wave's 1,024 logits). Workgroups of 8 waves joined through LDS took 117 with more instructions
// and 130 with fewer, waiting at their barrier; 32 logits a lane 94, and 30 more in the join, whose
// groups are larger then; workgroups that stay and fetch the next chunk ahead 137.
template <class T, bool VEC>
__global__ __launch_bounds__(SCORE_THREADS, 8) void k_score(ScoreArgs a) {
  constexpr int V = 16 / sizeof(T), NV = SCORE_EACH / V;
  typedef T vt __attribute__((ext_vector_type(V)));
  const uint32_t lane = threadIdx.x % WAVE, at = blockIdx.x * SCORE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  if (at >= a.rows * a.chunks) return;
  const uint32_t row = at / a.chunks, c0 = (at - row * a.chunks) * SCORE_CHUNK;
  const T* const p = static_cast<const T*>(a.x) + (int64_t)row * a.xs;
  const int32_t target = a.target ? a.target[row] : -1;
  vt w[NV];
  if (VEC && c0 + SCORE_CHUNK <= a.n) {
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = *reinterpret_cast<const vt*>(p + c0 + (v * WAVE + lane) * V);
  } else {
#pragma unroll
    for (int i = 0; i < SCORE_EACH; ++i) {
      const uint32_t c = c0 + (i / V * WAVE + lane) * V + i % V;
      w[i / V][i % V] = c < a.n ? p[c] : (T)-INFINITY;
    }
  }
  T wt = (T)INFINITY;
  if (target >= 0 && (uint32_t)target < a.n) wt = p[target];  // on its way with the others
  __builtin_amdgcn_sched_barrier(0);
  float x[SCORE_EACH];
#pragma unroll
  for (int i = 0; i < SCORE_EACH; ++i) x[i] = (float)w[i / V][i % V];
  float mine = x[0];
#pragma unroll
  for (int i = 1; i < SCORE_EACH; ++i) mine = fmaxf(mine, x[i]);
  const uint32_t group = max_of_8(score_order(mine));
  if (a.top && lane % SCORE_GROUP == 0) a.maxima[(size_t)at * SCORE_GROUPS + lane / SCORE_GROUP] = group;
  const float m = of_order(max_of_wave(group)), unit = a.scale * 1.44269504088896340736f, c = m * unit;
  float sum = 0.0f, moment = 0.0f;
  uint32_t above = 0;
  bool far = !(fabsf(c) <= 0x1p20f);  // (or m is not finite)
  if (!far) {
#pragma unroll
    for (int i = 0; i < SCORE_EACH; ++i) {
      const float t = fmaf(x[i], unit, -c), e = __builtin_amdgcn_exp2f(t);
      sum += e;
      moment = fmaf(t, e, moment);
    }
    far = __any(!(moment > -FLT_MAX));
  }
  if (__builtin_expect(far, 0)) {
    const float m0 = m == -INFINITY ? 0.0f : m;
    sum = moment = 0.0f;
    above = SCORE_FAR;
#pragma unroll
    for (int i = 0; i < SCORE_EACH; ++i) {
      const float t = (x[i] - m0) * unit, e = __builtin_amdgcn_exp2f(t);
      sum += e;
      moment = fmaf(fmaxf(t, -FLT_MAX), e, moment);  // so far below (or -inf): 0 of the sum
    }
  }
  const float xt = (float)wt;
  if (m > xt) {  // (the same in all lanes)
#pragma unroll
    for (int i = 0; i < SCORE_EACH; ++i) above += (uint32_t)__popcll(__ballot(x[i] > xt));
  }
  sum = sum_of_wave(sum);
  moment = sum_of_wave(moment);
  if (lane == WAVE - 1) a.part[at] = ScorePart{m, sum, moment, above};
}

// A row's chunks joined in order, in 64 bits, by the last wave; its best by the others:
// from the groups of logits whose maximum reaches a bound that `top` groups' maxima reach (the
// top-th of 64 maxima of groups), read again. Where more than LDS takes reach it, because
// many are equal to it: those over it, and of the equal ones the first in the row.
// Where those over it are too many still, one after the other, each by a pass over the row: where
// the best lie side by side, so that few groups hold more of them than LDS takes, or where a row of more logits
// than that has fewer groups than `top`. The 32 best of one row of 128,256 logits in order: 2.0 ms, of
// 1,024 such rows 8.1, the same where all but a run of 2,500 logits are -inf; of one row of 2,500 62 us.
//
// 20 best of 2047 rows of 128,256 bf16: 16 us (21 with the groups read by the value), of one row of
// 49,152: 5.7; without the best 4.7. Every
// row's workgroup is on the chip at once: a chain of reads (maxima, then the groups') and of the
// bound's and the ranking's serial steps.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_score_join(ScoreArgs a) {
  constexpr uint32_t V = 16 / sizeof(T), NV = SCORE_EACH / V;
  typedef T vt __attribute__((ext_vector_type(V)));
  constexpr uint32_t HELD = 4;  // groups' maxima that a thread keeps
  constexpr double LN2 = 0.69314718055994530942;
  __shared__ uint64_t s_key[SCORE_FEW], s_wave[4];
  __shared__ uint32_t s_max[4][WAVE];
  __shared__ uint16_t s_list[SCORE_LIST];
  __shared__ uint32_t s_count, s_groups;
  __shared__ double s_sum;
  __shared__ float s_top;
  static_assert(MAX_SCORE / SCORE_CHUNK * SCORE_GROUPS <= 0x10000 && MAX_TOP <= WAVE, "a group's number in 16 bits");
  const uint32_t row = blockIdx.x, lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const T* const x = static_cast<const T*>(a.x) + (int64_t)row * a.xs;
  const uint32_t groups = a.chunks * SCORE_GROUPS;
  const uint32_t* maxima = a.maxima + (size_t)row * groups;
  auto group_max = [&](uint32_t i) { return i < groups ? maxima[i] : 0u; };
  uint32_t held[HELD], most = 0;
  if (a.top) {
#pragma unroll
    for (uint32_t h = 0; h < HELD; ++h) held[h] = group_max(threadIdx.x + 256 * h);
#pragma unroll
    for (uint32_t h = 0; h < HELD; ++h) most = max(most, held[h]);
    for (uint32_t i = threadIdx.x + 256 * HELD; i < groups; i += 256) most = max(most, group_max(i));
    s_max[wave][lane] = most;
    if (threadIdx.x == 0) s_count = s_groups = 0;
  }

  if (wave == 3) {  // what the whole row's sums say
    const int32_t target = a.target ? a.target[row] : -1;
    const ScorePart* part = a.part + (size_t)row * a.chunks;
    const float unit = a.scale * 1.44269504088896340736f;
    float top = -INFINITY;
    double sum = 0.0, moment = 0.0;
    uint32_t above = 0;
    for (uint32_t c = lane; c < a.chunks; c += WAVE) top = fmaxf(top, part[c].top);
    top = wave_max(top);
    for (uint32_t c = lane; c < a.chunks; c += WAVE) {
      const ScorePart s = part[c];
      if (s.top == -INFINITY && s.sum == 0.0f) continue;  // nothing over -inf: nothing of the sum
      const float over = s.above & SCORE_FAR ? 0.0f : score_over(s.top, unit);
      // what its sum is times: that of a wave of one logit is 1
      const double own = (double)s.sum / (double)__builtin_amdgcn_exp2f(over);
      const double left = ((double)s.moment - (double)(over * s.sum)) / (double)__builtin_amdgcn_exp2f(over);
      const double t = (double)a.scale * ((double)s.top - (double)top), e = exp(t);
      sum += e * own;
      if (e > 0.0) moment += e * fma(t, own, LN2 * left);
      above += s.above & ~SCORE_FAR;
    }
    above = wave_add(above);
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
      sum += __shfl_xor(sum, o);
      moment += __shfl_xor(moment, o);
    }
    if (lane == 0) {
      const float nan = __builtin_nanf("");
      const bool none = !(sum >= 1.0);  // a NaN, an infinity, or nothing over -inf: no distribution
      const bool has = target >= 0 && (uint32_t)target < a.n && !none;
      const double scale = (double)a.scale, log_sum = none ? (double)nan : log(sum);
      a.log_p[row] = has ? (float)(scale * ((double)(float)x[target] - (double)top) - log_sum) : nan;
      a.entropy[row] = (float)(log_sum - moment / sum);
      a.rank[row] = has ? (int32_t)above : -1;
      s_sum = log_sum;
      s_top = top;
    }
  }
  if (!a.top) return;
  __syncthreads();
  const uint32_t o = max(max(s_max[0][lane], s_max[1][lane]), max(s_max[2][lane], s_max[3][lane]));
  // Keys of the logits that reach `from` (counts are 0); returns how many there are.
  auto gather = [&](uint32_t from) {
    auto list = [&](uint32_t i, uint32_t m) {
      if (i < groups && m >= from) {
        const uint32_t at = atomicAdd(&s_groups, 1u);
        if (at < SCORE_LIST) s_list[at] = (uint16_t)i;
      }
    };
#pragma unroll
    for (uint32_t h = 0; h < HELD; ++h) list(threadIdx.x + 256 * h, held[h]);
    for (uint32_t i = threadIdx.x + 256 * HELD; i < groups; i += 256) list(i, group_max(i));
    __syncthreads();
    const uint32_t n = s_groups;
    if (n > SCORE_LIST) return SCORE_FEW + 1;
    for (uint32_t i = threadIdx.x / 16; i < n; i += 16) {  // 16 lanes a group
      const uint32_t group = s_list[i], l = lane % 16;
      const uint32_t c0 = group / SCORE_GROUPS * SCORE_CHUNK + l / 8 * (WAVE * V) + (group % SCORE_GROUPS * SCORE_GROUP + l % 8) * V;
      vt w[NV / 2];
#pragma unroll
      for (uint32_t v = 0; v < NV / 2; ++v) {
        const uint32_t c = c0 + v * (2 * WAVE * V);
        if (VEC && c + V <= a.n) {
          w[v] = *reinterpret_cast<const vt*>(x + c);
        } else {
#pragma unroll
          for (uint32_t e = 0; e < V; ++e) w[v][e] = c + e < a.n ? x[c + e] : (T)-INFINITY;
        }
      }
#pragma unroll
      for (uint32_t v = 0; v < NV / 2; ++v)
#pragma unroll
        for (uint32_t e = 0; e < V; ++e) {
          const uint32_t c = c0 + v * (2 * WAVE * V) + e;
          const float value = (float)w[v][e];
          if (c < a.n && score_order(value) >= from) {
            const uint32_t at = atomicAdd(&s_count, 1u);
            if (at < SCORE_FEW) s_key[at] = score_key(value, c);
          }
        }
    }
    __syncthreads();
    return s_count;
  };
  uint32_t bound = score_bound(o, a.top, a.top / 4), count = gather(bound);
  const double log_sum = s_sum;
  const bool none = isnan(log_sum);
  if (count > SCORE_FEW && !none) {
    bound = score_bound(o, a.top, 0);  // a maximum's own number
    __syncthreads();
    if (threadIdx.x == 0) s_count = s_groups = 0;
    __syncthreads();
    count = gather(bound + 1);
    if (count < a.top) {  // ... and the first of the equal ones
      const float equal = value_of((uint64_t)bound << 32);
      if (wave == 0)
        for (uint32_t c0 = 0; c0 < a.n && count < a.top; c0 += WAVE) {
          const uint32_t c = c0 + lane;
          const float v = c < a.n ? (float)x[c] : 0.0f;
          const bool is = c < a.n && v == equal;
          const uint64_t mask = __ballot(is);
          const uint32_t at = count + (uint32_t)__popcll(mask & ((1ull << lane) - 1));
          if (is && at < a.top) s_key[at] = score_key(v, c);
          count += (uint32_t)__popcll(mask);
        }
      count = a.top;
    } else if (count > SCORE_FEW) {  // one after the other
      uint64_t last = ~0ull;
      for (uint32_t t = 0; t < a.top; ++t) {
        uint64_t k = 0;
        for (uint32_t c = threadIdx.x; c < a.n; c += 256) {
          const uint64_t key = score_key((float)x[c], c);
          k = key < last && key > k ? key : k;
        }
        for (int s = 32; s > 0; s >>= 1) {
          const uint64_t other = __shfl_xor((unsigned long long)k, s);
          k = other > k ? other : k;
        }
        __syncthreads();
        if (lane == 0) s_wave[wave] = k;
        __syncthreads();
        last = s_wave[0];
        for (int w = 1; w < 4; ++w) last = s_wave[w] > last ? s_wave[w] : last;
        if (threadIdx.x == 0) s_key[t] = last;
      }
      count = a.top;
    }
  }
  if (wave) return;
  const size_t out = (size_t)row * a.top;
  if (none) {
    if (lane < a.top) {
      a.top_index[out + lane] = -1;
      a.top_log_p[out + lane] = __builtin_nanf("");
    }
    return;
  }
  const double scale = (double)a.scale, top = (double)s_top;
  score_pick(s_key, count, a.top, [&](uint32_t t, uint64_t k) {
    a.top_index[out + t] = (int32_t)column_of(k);
    a.top_log_p[out + t] = (float)(scale * ((double)value_of(k) - top) - log_sum);
  });
}

template <class T>
int score_launch(const ScoreArgs& a, bool vec, hipStream_t s) {
  const uint32_t blocks = (a.rows * a.chunks + SCORE_WAVES - 1) / SCORE_WAVES;
  const int rc = launch(vec ? k_score<T, true> : k_score<T, false>, blocks, SCORE_THREADS, 0, s, a);
  return rc ? rc : launch(vec ? k_score_join<T, true> : k_score_join<T, false>, a.rows, 256, 0, s, a);
}

uint32_t score_chunks(uint32_t n) { return (n + SCORE_CHUNK - 1) / SCORE_CHUNK; }

}  // namespace

}  // namespace q8

// ------------------------------------------------------------- C entry points

using namespace q8;

extern "C" int defer_gpu_q8_kv_append(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, uint32_t type,
                                      const defer_gpu_q8_rotary* rotary, const void* q, int64_t q_stride, uint32_t q_heads,
                                      const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* out,
                                      int64_t out_stride, uint32_t clear, void* stream) {
  Pages p;
  Rows r;
  int rc = check_pages(pages, rows, &p, &r);
  if (!rc) rc = check_heads(pages, q_heads, 0);
  if (rc) return rc;
  const uint32_t hd = pages->head_dim, nkv = p.heads * hd, nq = q_heads * hd;
  rc = check_rows_values(type, q, q_stride, r.rows, nq, "q");
  if (!rc) rc = check_rows_values(type, k, k_stride, r.rows, nkv, "k");
  if (!rc) rc = check_rows_values(type, v, v_stride, r.rows, nkv, "v");
  if (!rc) rc = check_rows_values(type, out, out_stride, r.rows, nq, "out");
  if (rc) return rc;
  Q8_REQUIRE(rotary, "rotary is null");
  Q8_REQUIRE(rotary->rotated <= hd && rotary->rotated % 2 == 0, "%u values of %u rotated", rotary->rotated, hd);
  Q8_REQUIRE(rotary->rotated == 0 || (rotary->freq && aligned_to(rotary->freq, 8)), "freq is null or not aligned to its type");
  Q8_REQUIRE(aligned_to(rotary->position, 4), "position is not aligned to its type");
  Q8_REQUIRE(aligned_to(rotary->q_norm, value_size(type)) && aligned_to(rotary->k_norm, value_size(type)),
             "a norm's weight is not aligned to its type");
  Q8_REQUIRE(rotary->eps >= 0.0f && rotary->eps < INFINITY, "eps %g", (double)rotary->eps);
  Q8_REQUIRE(fabsf(rotary->factor) < INFINITY, "factor %g", (double)rotary->factor);
  const int64_t vs = (int64_t)value_size(type), row = nq * vs;
  Q8_REQUIRE(!overlap(out, out_stride * vs, r.rows, q, q_stride * vs, r.rows, row), "out overlaps q");
  // Of q a workgroup reads what it writes itself; all else is read by others while this one writes.
  auto shares = [&](const void* in, int64_t stride, uint32_t n, int64_t bytes) {
    return in && share(out, out_stride * vs, r.rows, row, in, stride, n, bytes);
  };
  Q8_REQUIRE(!shares(k, k_stride * vs, r.rows, nkv * vs), "out overlaps k");
  Q8_REQUIRE(!shares(v, v_stride * vs, r.rows, nkv * vs), "out overlaps v");
  Q8_REQUIRE(!shares(rotary->q_norm, 0, 1, hd * vs) && !shares(rotary->k_norm, 0, 1, hd * vs), "out overlaps a norm's weight");
  Q8_REQUIRE(!shares(rotary->position, 0, 1, (int64_t)r.rows * 4), "out overlaps position");
  Q8_REQUIRE(!rotary->rotated || !shares(rotary->freq, 0, 1, rotary->rotated * 4), "out overlaps freq");
  if (!r.rows) return DEFER_GPU_OK;
  const hipStream_t s = (hipStream_t)stream;
  if (!r.sequences || !r.most_rows)
    return clear ? launch(k_zero_rows, r.rows, 256, 0, s, out, out_stride, nq, type) : DEFER_GPU_OK;
  AppendArgs a{};
  a.p = p;
  a.r = r;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.qs = q_stride;
  a.ks = k_stride;
  a.vs = v_stride;
  a.os = out_stride;
  a.position = rotary->position;
  a.freq = rotary->freq;
  a.qn = rotary->q_norm;
  a.kn = rotary->k_norm;
  a.eps = (double)rotary->eps;
  a.factor = (double)rotary->factor;
  a.hd = hd;
  a.nh = q_heads;
  a.half = rotary->rotated / 2;
  a.interleaved = rotary->interleaved != 0;
  // Heads of a workgroup: 16 of its lanes take a row's head, so that a full run of queries takes
  // it 4 rounds and one of the cache's heads 2 (keys, values); fewer rows take more heads, so
  // that the lanes have work. Where those would be more workgroups than the chip holds at once
  // (4 on a CU), each takes twice as many heads and forms the rows' angles for all of them:
  // 2000 rows of 32 + 8 heads of 128 in 21.6 us rather than 25 (4 times as many: 23), but 11 x 33
  // normed rows of 24 + 4 heads of 96, too few for that, in 11.2 rather than 8.9.
  const uint32_t most = std::min(r.most_rows, (uint32_t)KV_RUN);
  auto power = [&](uint32_t n, uint32_t heads) {  // the largest one up to n, no more than heads need
    uint32_t s = 0;
    while ((2u << s) <= n && (1u << s) < heads) ++s;
    return s;
  };
  uint64_t blocks = 0;
  for (uint32_t items = most >= 8 ? 64 : 16, twice = 0; twice < 2; ++twice, items *= 2) {
    a.q_shift = power(items / most, q_heads);
    a.kv_shift = power(items / 4 / most, p.heads);
    a.kv_chunks = (p.heads + (1u << a.kv_shift) - 1) >> a.kv_shift;
    a.chunks = a.kv_chunks + ((q_heads + (1u << a.q_shift) - 1) >> a.q_shift);
    blocks = (uint64_t)r.sequences * kv_runs(r.most_rows) * a.chunks;
    if (blocks <= 1024) break;
  }
  if (clear && r.row_start) blocks += std::min(blocks, (uint64_t)256);  // for the rows of no sequence
  Q8_REQUIRE(blocks <= MAX_THREADS / 256, "too many rows for one call");
  const bool vec = hd % 8 == 0 && (a.interleaved ? a.half % 4 == 0 : a.half % 8 == 0) &&
                   ((uintptr_t)a.qn | (uintptr_t)a.kn | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)(q_stride * vs) |
                    (uintptr_t)(k_stride * vs) | (uintptr_t)(v_stride * vs) | (uintptr_t)(out_stride * vs)) % 16 == 0;
  const size_t lds = (size_t)most * angles_of(a.half, a.interleaved) * sizeof(double2) + ((size_t)most * KV_ROW << a.kv_shift);
  const uint32_t nb = (uint32_t)blocks;
  return type == DEFER_GPU_F32    ? append_launch<float>(a, nb, lds, vec, s)
         : type == DEFER_GPU_BF16 ? append_launch<__bf16>(a, nb, lds, vec, s)
                                  : append_launch<_Float16>(a, nb, lds, vec, s);
}

extern "C" int defer_gpu_q8_kv_keep(const defer_gpu_q8_pages* pages, const defer_gpu_q8_rows* rows, const int32_t* keep,
                                    const int32_t* kept, int32_t* kv_len_out, void* stream) {
  Pages p;
  Rows r;
  const int rc = check_pages(pages, rows, &p, &r);
  if (rc) return rc;
  Q8_REQUIRE(r.most_rows <= MAX_TREE, "%u rows of a sequence: at most %u", r.most_rows, MAX_TREE);
  if (!r.sequences) return DEFER_GPU_OK;
  Q8_REQUIRE(r.kv_len && kept && kv_len_out, "null argument");
  Q8_REQUIRE(r.rows == 0 || keep, "keep is null");
  Q8_REQUIRE(r.row_start || r.rows == r.sequences, "%u rows of %u sequences without row_start", r.rows, r.sequences);
  Q8_REQUIRE(aligned_to(keep, 4) && aligned_to(kept, 4) && aligned_to(kv_len_out, 4), "an array is not aligned to its type");
  const int64_t n = (int64_t)r.sequences * 4;
  auto apart = [&](const void* in, int64_t bytes) {
    return in == nullptr || (const char*)kv_len_out + n <= (const char*)in || (const char*)in + bytes <= (const char*)kv_len_out;
  };
  Q8_REQUIRE(apart(r.kv_len, n) && apart(kept, n) && apart(r.row_start, n + 4) && apart(keep, (int64_t)r.rows * 4),
             "kv_len_out overlaps an input");
  const uint64_t blocks = (uint64_t)r.sequences * p.heads;
  Q8_REQUIRE(blocks <= MAX_THREADS / 256, "too many sequences for one call");
  const KeepArgs a{p, r, keep, kept, kv_len_out, pages->head_dim};
  return launch(k_keep, (uint32_t)blocks, 256, 0, (hipStream_t)stream, a);
}

extern "C" size_t defer_gpu_q8_log_probs_workspace(uint32_t rows, uint32_t n, uint32_t top) {
  if (rows > MAX_THREADS / WAVE || n > MAX_SCORE || top > MAX_TOP) return 0;
  return (size_t)rows * score_chunks(n) * (sizeof(ScorePart) + (top ? SCORE_GROUPS * sizeof(uint32_t) : 0));
}

extern "C" int defer_gpu_q8_log_probs(uint32_t type, const void* x, int64_t x_stride, uint32_t rows, uint32_t n,
                                      const int32_t* target, float scale, uint32_t top, float* log_p, float* entropy,
                                      int32_t* rank, int32_t* top_index, float* top_log_p, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const int rc = check_rows_values(type, x, x_stride, rows, n, "logits");
  if (rc) return rc;
  Q8_REQUIRE(n <= MAX_SCORE, "%u logits: at most %u", n, MAX_SCORE);
  Q8_REQUIRE(top <= MAX_TOP && top <= n, "the %u best of %u: at most %u", top, n, MAX_TOP);
  Q8_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "scale %g", (double)scale);
  Q8_REQUIRE(rows == 0 || (log_p && entropy && rank && (top == 0 || (top_index && top_log_p))), "null output");
  Q8_REQUIRE(aligned_to(target, 4) && aligned_to(log_p, 4) && aligned_to(entropy, 4) && aligned_to(rank, 4) &&
                 aligned_to(top_index, 4) && aligned_to(top_log_p, 4),
             "an array is not aligned to its type");
  Q8_REQUIRE((uint64_t)rows * score_chunks(n) <= MAX_THREADS / SCORE_THREADS * SCORE_WAVES, "too many rows for one call");
  if (!rows) return DEFER_GPU_OK;
  const size_t need = defer_gpu_q8_log_probs_workspace(rows, n, top);
  Q8_REQUIRE(workspace && workspace_bytes >= need, "log_probs needs a workspace of %zu bytes, got %zu", need,
             workspace ? workspace_bytes : (size_t)0);
  Q8_REQUIRE(aligned16(workspace), "workspace is not 16-byte aligned");
  ScoreArgs a{x, x_stride, target, rows, n, top, score_chunks(n), scale, log_p, entropy, top_log_p, rank, top_index,
              static_cast<ScorePart*>(workspace), nullptr};
  a.maxima = reinterpret_cast<uint32_t*>(a.part + (size_t)rows * a.chunks);
  const bool vec = ((uintptr_t)x | (uintptr_t)(x_stride * (int64_t)value_size(type))) % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  return type == DEFER_GPU_F32    ? score_launch<float>(a, vec, s)
         : type == DEFER_GPU_BF16 ? score_launch<__bf16>(a, vec, s)
                                  : score_launch<_Float16>(a, vec, s);
}
