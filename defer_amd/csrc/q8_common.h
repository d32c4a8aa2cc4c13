// q8_common.h -- what the translation units of the 8-bit operators share: value
// types, reductions, rows to codes, where the cache's codes are, launches, and
// the checks of the C entry points.
#pragma once

#include "q8.h"

#include <math.h>

namespace q8 {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int WAVE = 64;
constexpr uint32_t MAX_THREADS = 0xffffffffu;  // of a launch in one dimension
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
// (Written out: the compiler moves each lane's value, quiets it, then takes the
// maximum: three instructions a step. A lane reads another's register two wait
// states after it was written.)
__device__ __forceinline__ float row_max(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:4 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:2 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_ror:1 row_mask:0xf bank_mask:0xf\n\ts_nop 1"
      : "+v"(v));
#endif
  return v;
}
// Towards zero; what is not a number is 0, what is out of range the nearest.
__device__ __forceinline__ int to_int(float v) {
  int i = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_cvt_i32_f32 %0, %1" : "=v"(i) : "v"(v));
#endif
  return i;
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
// The code of x, of 64 bits, at a scale s of 32: rint(x / s) with ties to even. The
// code times s is exact in 64 bits and, but for code 0, within a factor of two
// of x, so what it leaves of x is exact, too, and says where the product with
// 1 / s is on the wrong side of a half (a division takes three times the
// instructions). `scale` is 0 or NaN for a row of zeros.
struct Coder {
  double s, r;
  __device__ __forceinline__ explicit Coder(float scale) : s(scale > 0.0f ? (double)scale : 0.0), r(s > 0.0 ? 1.0 / s : 0.0) {}
  __device__ __forceinline__ int operator()(double v) const {
    const double x = s > 0.0 ? v : 0.0;
    int c = (int)rint(x * r);
    const double left = fma(-(double)c, s, x), over = 2.0 * fabs(left) - s;
    if (over > 0.0 || (over == 0.0 && (c & 1))) c += left > 0.0 ? 1 : -1;
    return c;
  }
};

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

// Runs that rows of neighbouring positions may lie in.
Q8_HD uint32_t kv_runs(uint32_t rows) { return (rows + 14) / 16 + 1; }
constexpr int KV_ROW = 256 + 8;  // bytes of a token's codes in LDS
constexpr int KV_RUN = 16;       // positions a workgroup takes: a quarter of a page

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
// 4 x 4 bytes, rows to columns.
__device__ __forceinline__ void transpose4(const uint32_t* in, uint32_t* out) {
  const uint32_t l01 = perm(in[1], in[0], 0x05010400u), l23 = perm(in[3], in[2], 0x05010400u);
  const uint32_t h01 = perm(in[1], in[0], 0x07030602u), h23 = perm(in[3], in[2], 0x07030602u);
  out[0] = perm(l23, l01, 0x05040100u);
  out[1] = perm(l23, l01, 0x07060302u);
  out[2] = perm(h23, h01, 0x05040100u);
  out[3] = perm(h23, h01, 0x07060302u);
}

// 8 values of a row from d on, zeros from hd on; vec: 16-byte loads.
__device__ __forceinline__ void load8(const void* p, int64_t i0, uint32_t d, uint32_t hd, uint32_t type, bool vec, float* y) {
  if (vec && d < hd) {
    if (type == DEFER_GPU_F32) {
      const v4f* q = reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i0 + d);
      const v4f a = q[0], b = q[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = a[e];
        y[4 + e] = b[e];
      }
    } else {
      const v4i w = *reinterpret_cast<const v4i*>(static_cast<const uint16_t*>(p) + i0 + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t h = (uint16_t)((uint32_t)w[e / 2] >> (16 * (e % 2)));
        y[e] = type == DEFER_GPU_BF16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
      }
    }
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e) y[e] = d + e < hd ? load_value(p, i0 + d + e, type) : 0.0f;
}
__device__ __forceinline__ void store8(void* p, int64_t i0, uint32_t d, uint32_t hd, uint32_t type, bool vec, const float* y) {
  if (vec && d < hd) {
    if (type == DEFER_GPU_F32) {
      v4f* q = reinterpret_cast<v4f*>(static_cast<float*>(p) + i0 + d);
      q[0] = v4f{y[0], y[1], y[2], y[3]};
      q[1] = v4f{y[4], y[5], y[6], y[7]};
    } else {
      v4i w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t lo = type == DEFER_GPU_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y[2 * e]) : __builtin_bit_cast(uint16_t, (_Float16)y[2 * e]);
        const uint16_t hi = type == DEFER_GPU_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)y[2 * e + 1]) : __builtin_bit_cast(uint16_t, (_Float16)y[2 * e + 1]);
        w[e] = (int)((uint32_t)lo | (uint32_t)hi << 16);
      }
      *reinterpret_cast<v4i*>(static_cast<uint16_t*>(p) + i0 + d) = w;
    }
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 8; ++e)
    if (d + e < hd) store_value(p, i0 + d + e, type, y[e]);
}

// ------------------------------------------------------------- launches

// Zeros for the rows of a call without sequences.
__global__ __launch_bounds__(256) void k_zero_rows(void* out, int64_t stride, uint32_t n, uint32_t type) {
  for (uint32_t i = threadIdx.x; i < n; i += 256) store_value(out, (int64_t)blockIdx.x * stride + i, type, 0.0f);
}

// (The launch's own status: the runtime's last error may be that of an earlier
// call of the program's, and stays there for it.)
template <class A>
struct Same {
  typedef A type;
};
template <class... A>
int launch(void (*kernel)(A...), dim3 grid, dim3 block, size_t lds, hipStream_t s, typename Same<A>::type... args) {
  void* p[] = {&args...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, p, lds, s);
  return e == hipSuccess ? DEFER_GPU_OK : defer_gpu_fail_(DEFER_GPU_E_HIP, "launch: %s", hipGetErrorString(e));
}

// ------------------------------------------------------------- checks

#define Q8_REQUIRE(cond, ...)                                              \
  do {                                                                     \
    if (!(cond)) return defer_gpu_fail_(DEFER_GPU_E_INVALID, __VA_ARGS__); \
  } while (0)

inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline size_t value_size(uint32_t type) { return type == DEFER_GPU_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

inline int check_rows_values(uint32_t type, const void* x, int64_t stride, uint32_t rows, uint32_t n, const char* what) {
  Q8_REQUIRE(type <= DEFER_GPU_F16, "value type %u", type);
  Q8_REQUIRE(n >= 1 && n <= 0x7fffffffu && rows <= MAX_THREADS / 1024, "%s: %u rows of %u values", what, rows, n);
  Q8_REQUIRE(rows == 0 || x, "%s is null", what);
  Q8_REQUIRE(rows <= 1 || stride >= (int64_t)n, "%s: rows of %u values %lld apart", what, n, (long long)stride);
  Q8_REQUIRE(aligned_to(x, value_size(type)), "%s is not aligned to its type", what);
  return DEFER_GPU_OK;
}

inline int check_pages(const defer_gpu_q8_pages* p, const defer_gpu_q8_rows* r, Pages* pages, Rows* rows) {
  Q8_REQUIRE(p && r, "null argument");
  Q8_REQUIRE(p->head_dim >= 1 && p->head_dim <= MAX_HEAD_DIM, "head_dim %u: 1 to %u", p->head_dim, MAX_HEAD_DIM);
  Q8_REQUIRE(p->heads >= 1 && p->heads <= 65535, "%u cache heads", p->heads);
  Q8_REQUIRE(p->pages <= 0x7fffffffu && p->table_width <= 0x7fffffffu / PAGE, "%u pages, %u a sequence", p->pages,
             p->table_width);
  Q8_REQUIRE(r->rows <= MAX_THREADS / 1024 && r->sequences <= MAX_THREADS / 1024, "%u rows of %u sequences", r->rows, r->sequences);
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
  Q8_REQUIRE(((uint64_t)r->sequences + 1) * p->heads * kv_runs(r->most_rows) <= MAX_THREADS / 256,
             "too many rows for one call");
  return DEFER_GPU_OK;
}

inline int check_heads(const defer_gpu_q8_pages* p, uint32_t q_heads, uint32_t most_len) {
  Q8_REQUIRE(q_heads >= 1 && q_heads <= 65535 && q_heads % p->heads == 0, "%u query heads on %u cache heads", q_heads,
             p->heads);
  Q8_REQUIRE(most_len <= 0x7fffffffu, "most_len %u", most_len);
  return DEFER_GPU_OK;
}

}  // namespace

}  // namespace q8
