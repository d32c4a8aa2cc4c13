// q8_attn.h -- what the attention over the 8-bit cache and that of a tree of drafts
// have in common: the arithmetic of a block of positions, which gives both the same bits.
#pragma once

#include "q8_common.h"

namespace q8 {

namespace {

struct AttnArgs {
  Pages p;
  Rows r;
  const void* q;
  void* out;
  int64_t qs, os;
  uint32_t type, nh, group, hd, tiles, units;
  uint32_t per_wave;  // units a wave takes (SPLIT)
  bool q_vec;  // a head's 16 values are 16-byte loads
  bool clear;  // zeros for the rows of no sequence
  int64_t most_len;
  float scale2;  // scale * log2(e)
  const uint8_t* hidden;
  int64_t hs;
  uint32_t hidden_len;
  float* part;  // [rows][nh][units][2 + dp]: maximum, sum, accumulators
  const int32_t* parent;  // [rows], of rows that are nodes of trees
};

// Four signed base-256 digits of x, one a byte: x = sum of byte_i 256^i.
__device__ __forceinline__ uint32_t digits(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }
// ... and back, from sums of products of each digit with codes.
__device__ __forceinline__ float undigit(v4i d) {
  return fmaf((float)((d[3] << 8) + d[2]), 65536.0f, (float)((d[1] << 8) + d[0]));
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A running softmax: maximum (as an exponent of 2), sum, accumulators. The
// next part (m, l, acc) joins it with the weights x and y.
__device__ __forceinline__ void join_weights(float& M, float m, float* x, float* y) {
  const float mn = fmaxf(M, m), m0 = mn == -INFINITY ? 0.0f : mn;
  *x = exp2_of(M - m0);
  *y = exp2_of(m - m0);
  M = mn;
}

constexpr int P_ROW = 80;  // bytes of a digit row of 64 probabilities in LDS: rows of four heads on other banks

// A pair's query from q0 on (16 lanes' worth: four lanes of each of four pairs hold
// the four digits of 16 KC values), as its digits times the sign of the scale;
// returns its factor: for digit sums times 2^-45, or negative, for the sums as
// they are.
template <int KC>
__device__ __forceinline__ float query_digits(const AttnArgs& a, int64_t q0, bool ok, v4i* aq) {
  const uint32_t lane = threadIdx.x % WAVE, n16 = lane % 16, quad = lane / 16;
  float x[KC][16], top = 0.0f, bad = 0.0f;
#pragma unroll
  for (int kk = 0; kk < KC; ++kk) {
    const uint32_t d0 = kk * 64 + quad * 16;
    if (a.q_vec) {
      const int64_t at = q0 + (d0 < a.hd ? d0 : 0);
      if (a.type == DEFER_GPU_F32) {
        const v4f* p = reinterpret_cast<const v4f*>(static_cast<const float*>(a.q) + at);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[kk][e] = p[e / 4][e % 4];
      } else {
        typedef uint16_t v8h __attribute__((ext_vector_type(8)));
        const v8h* p = reinterpret_cast<const v8h*>(static_cast<const uint16_t*>(a.q) + at);
        const bool bf = a.type == DEFER_GPU_BF16;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint16_t h = p[e / 8][e % 8];
          x[kk][e] = bf ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) x[kk][e] = ok && d0 < a.hd ? x[kk][e] : 0.0f;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[kk][e] = ok && d0 + e < a.hd ? load_value(a.q, q0 + d0 + e, a.type) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      top = fmaxf(top, fabsf(x[kk][e]));
      bad = fmaf(x[kk][e], 0.0f, bad);
    }
  }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  bad += __shfl_xor(bad, 16);
  bad += __shfl_xor(bad, 32);
  const bool tiny = top > 0.0f && top < 0x1p-64f;
  if (__builtin_expect(__any(tiny), 0)) {
    const float lift = tiny ? 0x1p80f : 1.0f;
    top *= lift;
#pragma unroll
    for (int kk = 0; kk < KC; ++kk)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[kk][e] *= lift;
  }
  int ex = 0;  // top < 2^ex
  (void)frexpf(top, &ex);
  ex = top > 0.0f ? ex : 0;
  const float up = isnan(bad) ? 0.0f : a.scale2 < 0.0f ? -ldexpf(1.0f, 30 - ex) : ldexpf(1.0f, 30 - ex);
  const int unit = (tiny ? ex - 80 : ex) - 30;  // of the digit sums
  const float s = isnan(bad) ? __builtin_nanf("") : (ex > 64 ? -ldexpf(1.0f, unit) : ldexpf(1.0f, unit + 45)) * fabsf(a.scale2);
  const uint32_t dg = n16 % 4, sel = dg | (4 + dg) << 8;
#pragma unroll
  for (int kk = 0; kk < KC; ++kk)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = digits(to_int(x[kk][4 * w + e] * up));
      aq[kk][w] = (int)perm(perm(y[3], y[2], sel), perm(y[1], y[0], sel), 0x05040100u);
    }
  return s;
}

// A lane's scores s of the four positions that it sees, with their value scales:
// the digits y of their probabilities, the running maximum m and sum l, the weights xw
// of what came before and be of this block. vbad: what makes the sum NaN (WHOLE: every
// position is seen).
template <bool WHOLE>
__device__ __forceinline__ void block_weights(const float* s, const bool* see, const v4f& vs, float vbad, float sq, float& m, float& l,
                                              float* xw, float* be, uint32_t* y) {
  float w[4];
  const float top = row_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
  const bool none = !WHOLE && top == -INFINITY;
  const float m0 = none ? 0.0f : top * sq;
  const bool sharp = fabsf(m0) > 0x1p26f;
  const float before = sharp ? top : 0.0f, behind = sharp ? 0.0f : m0;
  float lp = vbad;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float p = exp2_of(fmaf(s[j] - before, sq, -behind));
    if (!WHOLE) {
      p = see[j] ? p : 0.0f;
      lp += see[j] ? fmaf(vs[j], 0.0f, p) : 0.0f;
      w[j] = see[j] ? p * vs[j] : 0.0f;
    } else {
      lp += p;
      w[j] = p * vs[j];
    }
  }
  int ex = 0;
  (void)frexpf(row_max(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))), &ex);
  ex = max(ex, -96);
  const float up = ldexpf(1.0f, 30 - ex);
  float yw;
  join_weights(m, none ? -INFINITY : m0, xw, &yw);
  *be = yw * ldexpf(1.0f, ex - 30);
  l = fmaf(lp, yw, l * *xw);
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = digits(to_int(w[j] * up));
}

inline AttnArgs attn_args(const Pages& p, const Rows& r, const Attention& in, void* workspace) {
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
  a.most_len = in.most_len;
  a.scale2 = in.scale * 1.44269504088896340736f;
  a.hidden = in.hidden;
  a.hs = in.hidden_stride;
  a.hidden_len = in.hidden_len;
  a.part = static_cast<float*>(workspace);
  a.clear = in.clear && r.row_start;
  const size_t vs = in.type == DEFER_GPU_F32 ? 4 : 2;
  a.q_vec = in.head_dim % 16 == 0 && ((uintptr_t)in.q | (uintptr_t)(in.q_stride * (int64_t)vs)) % 16 == 0;
  a.parent = in.parent;
  return a;
}

}  // namespace

}  // namespace q8
