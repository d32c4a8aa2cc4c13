// q8_tree.hip -- the attention of rows that are nodes of a tree of drafted tokens,
// over the 8-bit cache: the bits of each row are those that k_attn (q8.hip) has
// for its path alone.
#include "q8_attn.h"

#include <algorithm>

namespace q8 {

namespace {

constexpr int TREE_WAVES = 4;                 // of a workgroup: tiles that share a block's codes
constexpr int PATH_LDS = 3 * 4 * PAGE * 4;    // bytes: four pairs' scores, value scales and marks by position
constexpr int path_lds(int R) { return R * (16 * P_ROW + PATH_LDS); }
static_assert(16 * P_ROW <= 2 * 4 * PAGE * 4, "probabilities take the place of scores and value scales");

// A sequence's drafted rows as a tree, a row each lane: the rows that are its
// own or above it. A parent that is no earlier row is none: the row hangs on the
// history. Each step doubles how far up a row has looked.
struct Tree {
  uint64_t path;
  // the lane's row's parent
  __device__ __forceinline__ static int up(const int32_t* parent, const Span& sp) {
    const int lane = threadIdx.x % WAVE;
    return lane < sp.n ? parent[sp.start + lane] : -1;
  }
  __device__ __forceinline__ explicit Tree(int up) {
    const int lane = threadIdx.x % WAVE;
    up = up < lane ? up : -1;
    path = 1ull << lane;
    while (__any(up >= 0)) {
      const int from = max(up, 0), above = __shfl(up, from);
      const uint64_t more = __shfl((unsigned long long)path, from);
      if (up >= 0) {
        path |= more;
        up = above;
      }
    }
  }
  // how many rows are above the lane's own
  __device__ __forceinline__ int depth() const { return __popcll(path) - 1; }
  // the position of row j, which is as far behind the history as the row is deep; -1: it has
  // none. (By all lanes.)
  __device__ __forceinline__ int64_t pos(const Span& sp, uint32_t j) const {
    const int64_t history = (int64_t)sp.len - sp.n, d = __shfl(depth(), (int)j);
    return history < 0 || j >= MAX_TREE ? -1 : history + d;
  }
};

// A block's codes in LDS, as 16-byte chunks. Key 4 n + j is row 16 j + n there,
// and a row's chunks are turned by n (or by n / 2, where two rows are not 256 bytes
// apart), the chunks of a value's row by half its number: so that the 16
// lanes that read the same chunk of 16 rows read different banks.
template <int KC>
struct Stage {
  static constexpr int DP = 64 * KC, CHUNKS = DP / 16;
  static constexpr int SCALES = 2 * PAGE * DP, BYTES = SCALES + 2 * PAGE * 4;  // behind the codes the scales
  __device__ __forceinline__ static uint32_t turn(uint32_t n) { return CHUNKS % 8 == 0 ? n : n / 2; }
  __device__ __forceinline__ static uint32_t key_at(uint32_t n, int j, uint32_t c) {
    return (16 * j + n) * DP + (c + turn(n)) % CHUNKS * 16;
  }
  __device__ __forceinline__ static uint32_t value_at(uint32_t n, int t, uint32_t quad) {
    return PAGE * DP + (16 * t + n) * PAGE + ((quad + n / 2) & 3) * 16;
  }
  // where lane `lane` of copy i (of 4 KC each for keys and values) has its chunk from
  __device__ __forceinline__ static uint32_t key_from(uint32_t i, uint32_t lane) {
    const uint32_t l = 64 * i + lane, row = l / CHUNKS, n = row % 16, j = row / 16;
    const uint32_t c = (l % CHUNKS + 2 * CHUNKS - turn(n) % CHUNKS) % CHUNKS;
    return (4 * n + j) * DP + c * 16;
  }
  __device__ __forceinline__ static uint32_t value_from(uint32_t i, uint32_t lane) {
    const uint32_t l = 64 * i + lane, row = l / 4, n = row % 16;
    return row * PAGE + ((l - n / 2) & 3) * 16;
  }
};

// A workgroup's four waves take a tile each, of R times four (row, query head)
// pairs of one sequence and cache head, and go through its blocks of 64 positions
// together: a block's codes come to LDS once for all four, the next ones while
// this one is worked on. The arithmetic of a block is k_attn's.
//
// Blocks before the history's end are the same for every row. Behind it a row's
// positions are those of the path from there down to itself, as if the
// path were all there is: the scores of the nodes' own places go through LDS to
// the path's positions, the probabilities back from there. Sums over a block's
// positions of digits times codes are exact, so that the places' order changes
// nothing.
//
// SPLIT: a workgroup takes per_wave units, left in the workspace for k_tree_join.
//
// 7 x 25 rows over 6000 positions, 32 heads on 8 of 128: 165 us, of which the digits' products
// are 34 at the matrix cores' rate and the codes 15 (154 without copying them); bound by the chain of a
// block, 1.7 us: 188 vector and 16 matrix instructions, about 0.4 us of issue, and the waits between
// them (copies, three passes through LDS), which one or two waves a SIMD do not cover (392 workgroups on
// 256 CUs). 32 x 12 rows over 384, 32 heads on 8 of 64, some places hidden: 23 us, three workgroups a
// CU that each go through seven blocks (26 with each lane reading its four places' marks when it
// needs them). 7 rows at 203, 9 heads on 3 of 64: 9.2, a chain of reads and four blocks one after the other. With each wave loading the codes of its own tile, as k_attn does,
// the first two took 541 and 59 us; three blocks in LDS instead of two gave nothing, for one workgroup
// less a CU.
template <int KC, int R, bool SPLIT>
__global__ __launch_bounds__(64 * TREE_WAVES, KC == 1 ? 3 : KC == 2 ? 2 : 1) void k_tree(AttnArgs a) {
  constexpr int DT = 4 * KC, DP = 64 * KC;
  typedef Stage<KC> St;
  extern __shared__ __align__(16) uint8_t lds[];  // two blocks' codes, then each wave's probabilities and path
  const uint32_t lane = threadIdx.x % WAVE, n16 = lane % 16, quad = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  uint8_t* const pl = lds + 2 * St::BYTES + wave * path_lds(R);

  const uint32_t shs = a.r.sequences * a.p.heads, chunks = SPLIT ? (a.units + a.per_wave - 1) / a.per_wave : 1;
  const uint32_t sh = blockIdx.x % shs, item = blockIdx.x / shs, seq = sh / a.p.heads, g = sh % a.p.heads;
  const uint32_t tile = item / chunks * TREE_WAVES + wave;
  if (a.clear && blockIdx.x == gridDim.x - 1) {
    // rows of no sequence lie before the first span and behind the last
    const int64_t lo = span_of(a.r.row_start, a.r.kv_len, 0, a.r.rows).start;
    const int64_t hi = max(lo, min((int64_t)a.r.row_start[a.r.sequences], (int64_t)a.r.rows));
    for (int64_t i = wave; i < lo + ((int64_t)a.r.rows - hi); i += TREE_WAVES) {
      const int64_t row = i < lo ? i : hi + (i - lo);
      for (uint32_t d = lane; d < a.nh * a.hd; d += WAVE) store_value(a.out, row * a.os + d, a.type, 0.0f);
    }
  }
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  const int rows = min(sp.n, (int)a.r.most_rows);  // (at most MAX_TREE)
  if (__builtin_expect(sp.n > rows, 0) && a.clear && item == 0)  // rows behind the most are as rows of no sequence
    for (int j = rows + (int)wave; j < sp.n; j += TREE_WAVES)
      for (uint32_t d = lane; d < a.group * a.hd; d += WAVE)
        store_value(a.out, (int64_t)(sp.start + j) * a.os + (int64_t)g * a.group * a.hd + d, a.type, 0.0f);
  if (rows <= 0 || item / chunks * TREE_WAVES * 4 * R >= (uint32_t)rows * a.group) return;
  const int32_t* table = a.p.table + (size_t)seq * a.p.width;
  const uint8_t* hid = a.hidden ? a.hidden + (int64_t)seq * a.hs : nullptr;
  const int history = (int)max((int64_t)sp.len - sp.n, (int64_t)-1), first_path = history / PAGE;
  const uint32_t pair0 = tile * 4 * R;

  // copies of a block's codes: this wave's KC of keys and KC of values
  const size_t page_codes = (size_t)PAGE * DP;
  uint32_t kf[KC], vf[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    kf[i] = St::key_from(wave * KC + i, lane);
    vf[i] = St::value_from(wave * KC + i, lane);
  }
  // (the first two waves' first copy is of 64 scales)
  auto copy = [&](int page, int buf) {
    if (wave < 2) {
      const float* const from = (wave ? a.p.value_scale : a.p.key_scale) + ((size_t)page * a.p.heads + g) * PAGE;
      const auto sr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, PAGE * 4, 0x00020000);
      uint8_t* const to = lds + buf * St::BYTES + St::SCALES + wave * PAGE * 4;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (__attribute__((address_space(3))) void*)to, 4, (int)lane * 4, 0, 0, 0);
    }
    const size_t at = ((size_t)page * a.p.heads + g) * page_codes;
    const auto kr = __builtin_amdgcn_make_buffer_rsrc(a.p.keys + at, 0, (int)page_codes, 0x00020000);
    const auto vr = __builtin_amdgcn_make_buffer_rsrc(a.p.values + at, 0, (int)page_codes, 0x00020000);
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      uint8_t* const to = lds + buf * St::BYTES + (wave * KC + i) * 1024;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (__attribute__((address_space(3))) void*)to, 16, (int)kf[i], 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (__attribute__((address_space(3))) void*)(to + page_codes), 16, (int)vf[i], 0, 0, 0);
    }
  };
  // pages of 64 blocks at a time, one a lane
  int window = -1, window_page = -1;
  auto page_at = [&](int block) {
    if (block / WAVE != window) {
      window = block / WAVE;
      window_page = page_of(table, a.p.width, a.p.pages, (int64_t)window * WAVE + lane);
    }
    return __builtin_amdgcn_readlane(window_page, block % WAVE);
  };
  // All copies have arrived, and every wave is done with what was in the place of the next ones.
  auto meet = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // What the first block waits for goes out before all else: rows' parents, its page, its codes, the queries.
  const int up = Tree::up(a.parent, sp);
  const int ul_first = unit_len(max(min((int64_t)history, a.most_len - 1), (int64_t)0)), u_first = SPLIT ? (int)(item % chunks * a.per_wave) : 0;
  const int page_first = history < 0 ? -1 : page_at(u_first * (ul_first / PAGE));
  if (page_first >= 0) copy(page_first, 0);
  v4i aq[R][KC];
  float sq[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t pr = pair0 + 4 * r + n16 / 4, j = pr / a.group;
    const bool ok = j < (uint32_t)rows;
    const int64_t q0 = (int64_t)(sp.start + (ok ? j : 0)) * a.qs + (int64_t)(g * a.group + pr % a.group) * a.hd;
    sq[r] = __shfl(query_digits<KC>(a, q0, ok, aq[r]), (int)quad * 4);
  }

  const Tree tree(up);
  const int depth = tree.depth();

  // the whole sequence's last position, and each pair's (-1: none)
  int deepest = (int)lane < rows ? depth : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) deepest = max(deepest, __shfl_xor(deepest, o));
  const int last = history < 0 ? -1 : __builtin_amdgcn_readfirstlane((int)min((int64_t)history + deepest, a.most_len - 1));
  int pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t j = (pair0 + 4 * r + quad) / a.group;
    const int64_t at = tree.pos(sp, j);
    pos[r] = j < (uint32_t)rows && at >= 0 ? (int)min(at, a.most_len - 1) : -1;
  }

  // Rows whose positions lie on both sides of a multiple of 8,192 have units of
  // different lengths: one length after the other.
  const int ul_last = unit_len(max(last, 0));
  for (int ul = ul_first; ul <= ul_last; ul += UNIT) {
    int ps[R], pmax = -1, pmin = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ps[r] = pos[r] >= 0 && unit_len(pos[r]) == ul ? pos[r] : -1;
      pmax = max(pmax, ps[r]);
      pmin = min(pmin, ps[r] < 0 ? 0x7fffffff : ps[r]);
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

    // Scores of a tile and the keys at `codes`: pair quad, keys 4 n16 + j.
    auto scores = [&](const v4i (*k)[KC], int r, const v4f& kp, float* x) {
      const float unit = sq[r] < 0.0f ? 1.0f : 0x1p-45f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v4i d = {0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KC; ++kk) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[r][kk], k[j][kk], d, 0, 0, 0);
        x[j] = undigit(d) * unit * kp[j];
      }
    };
    auto keys = [&](const uint8_t* codes, v4i (*k)[KC]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int kk = 0; kk < KC; ++kk) k[j][kk] = *reinterpret_cast<const v4i*>(codes + St::key_at(n16, j, 4 * kk + quad));
    };
    auto fence = [] {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };

    // A block of the history, its hidden places. WHOLE: every row sees all of it.
    auto block = [&](auto whole, int b, uint64_t hide, const uint8_t* codes) {
      constexpr bool WHOLE = decltype(whole)::value;
      const int tb = b * PAGE + 4 * n16;
      const uint32_t hides = (uint32_t)(hide >> (4 * n16));
      const v4f ks = *reinterpret_cast<const v4f*>(codes + St::SCALES + 16 * n16);
      const v4f vs = *reinterpret_cast<const v4f*>(codes + St::SCALES + PAGE * 4 + 16 * n16);
      float vbad = 0.0f;
      if (WHOLE) vbad = fmaf(vs[0], 0.0f, vs[1] * 0.0f) + fmaf(vs[2], 0.0f, vs[3] * 0.0f);
      v4i k[4][KC], v[DT];
      keys(codes, k);
      float xw[R], be[R], x[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r) scores(k, r, ks, x[r]);
#pragma unroll
      for (int t = 0; t < DT; ++t) v[t] = *reinterpret_cast<const v4i*>(codes + St::value_at(n16, t, quad));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float* const s = x[r];
        bool see[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          see[j] = WHOLE || (tb + j <= ps[r] && !(hides >> j & 1));
          s[j] = see[j] ? s[j] : -INFINITY;
        }
        uint32_t y[4], by_digit[4];
        block_weights<WHOLE>(s, see, vs, vbad, fabsf(sq[r]), m[r], l[r], &xw[r], &be[r], y);
        uint32_t* pw = reinterpret_cast<uint32_t*>(pl + (16 * r + 4 * quad) * P_ROW) + n16;
        transpose4(y, by_digit);
#pragma unroll
        for (int i = 0; i < 4; ++i) pw[i * P_ROW / 4] = by_digit[i];
      }
      fence();
      v4i pa[R];
#pragma unroll
      for (int r = 0; r < R; ++r) pa[r] = *reinterpret_cast<const v4i*>(pl + (16 * r + n16) * P_ROW + quad * 16);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const v4i zero = {0, 0, 0, 0};
          const v4i o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa[r], v[t], zero, 0, 0, 0);
          acc[r][t] = fmaf(undigit(o), be[r], acc[r][t] * xw[r]);
        }
      }
      fence();
    };

    // A block of a path's positions, around the history's end or behind it. The nodes
    // on it are in this place's page or the next (a tree has no more than 64 rows), whose
    // hidden places are given. all: no place is hidden or without a page.
    auto path_block = [&](int b, int page, int page_behind, uint64_t hide, uint64_t hide_behind, bool all, const uint8_t* codes) {
      float* const sl = reinterpret_cast<float*>(pl + R * 16 * P_ROW) + quad * PAGE;  // this quad's pair, of R
      constexpr int EACH = 4 * PAGE, VALUE = EACH, MARK = 2 * EACH, OF_R = 3 * EACH;
      uint32_t* const ml = reinterpret_cast<uint32_t*>(sl + MARK);
      if (!all) {
#pragma unroll
        for (int r = 0; r < R; ++r) *reinterpret_cast<v4i*>(ml + r * OF_R + 4 * n16) = v4i{0, 0, 0, 0};
        fence();
      }
      const size_t behind = ((size_t)max(page_behind, 0) * a.p.heads + g) * page_codes;
      uint32_t at[2] = {0, 0}, seen[2] = {0, 0};  // of a place's nodes: the position within the block; of each r, a bit
#pragma unroll
      for (int pb = 0; pb < 2; ++pb) {
        if ((pb ? page_behind : page) < 0) continue;
        v4i k[4][KC];
        v4f kp, vp;
        if (pb) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int kk = 0; kk < KC; ++kk)
              k[j][kk] = *reinterpret_cast<const v4i*>(a.p.keys + behind + (4 * n16 + j) * DP + quad * 16 + kk * 64);
          const size_t hp = ((size_t)page_behind * a.p.heads + g) * PAGE + 4 * n16;
          kp = *reinterpret_cast<const v4f*>(a.p.key_scale + hp);
          vp = *reinterpret_cast<const v4f*>(a.p.value_scale + hp);
        } else {
          keys(codes, k);
          kp = *reinterpret_cast<const v4f*>(codes + St::SCALES + 16 * n16);
          vp = *reinterpret_cast<const v4f*>(codes + St::SCALES + PAGE * 4 + 16 * n16);
        }
        const int node0 = (b + pb) * PAGE + 4 * (int)n16 - history;  // the lane's first place's
        uint32_t on = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int node = node0 + j, t = node + history, d = __shfl(depth, node & (WAVE - 1));
          const int to = (node < 0 ? t : history + d) - b * PAGE;
          const bool is = node < rows && to >= 0 && to < PAGE && !((pb ? hide_behind : hide) >> (4 * n16 + j) & 1);
          at[pb] |= (uint32_t)(to & (PAGE - 1)) << (8 * j);
          on |= (uint32_t)is << j;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint64_t path = __shfl((unsigned long long)tree.path, (int)((pair0 + 4 * r + quad) / a.group) & (WAVE - 1));
          // the nodes among the lane's places that are on the pair's path; places before them are on every one
          const uint32_t mine = node0 >= 0 ? (uint32_t)(path >> (node0 & (WAVE - 1))) & 15
                                           : ((uint32_t)(path << (-node0 & 3)) & 15) | (node0 > -4 ? (1u << -node0) - 1 : 15);
          float x[4];
          scores(k, r, kp, x);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int to = at[pb] >> (8 * j) & 255;
            const bool see = (on & mine) >> j & 1 && b * PAGE + to <= ps[r];
            seen[pb] |= (uint32_t)see << (4 * r + j);
            if (see) {
              sl[r * OF_R + to] = x[j];
              sl[r * OF_R + VALUE + to] = vp[j];
              if (!all) ml[r * OF_R + to] = 1;
            }
          }
        }
      }
      fence();
      float xw[R], be[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const v4f sv = *reinterpret_cast<const v4f*>(sl + r * OF_R + 4 * n16);
        const v4f vv = *reinterpret_cast<const v4f*>(sl + r * OF_R + VALUE + 4 * n16);
        float s[4];
        bool see[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) see[j] = b * PAGE + 4 * (int)n16 + j <= ps[r];
        if (!all) {
          const v4i mv = *reinterpret_cast<const v4i*>(ml + r * OF_R + 4 * n16);
#pragma unroll
          for (int j = 0; j < 4; ++j) see[j] = mv[j] != 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = see[j] ? sv[j] : -INFINITY;
        uint32_t y[4];
        block_weights<false>(s, see, vv, 0.0f, fabsf(sq[r]), m[r], l[r], &xw[r], &be[r], y);
        *reinterpret_cast<v4i*>(ml + r * OF_R + 4 * n16) = v4i{(int)y[0], (int)y[1], (int)y[2], (int)y[3]};
      }
      fence();
      // back to the places: the second page's probabilities where the scores were
      uint8_t* const pb_lds = pl + R * 16 * P_ROW;
#pragma unroll
      for (int pb = 0; pb < 2; ++pb) {
        if ((pb ? page_behind : page) < 0) continue;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint32_t p[4], by_digit[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t y = ml[r * OF_R + (at[pb] >> (8 * j) & 255)];
            p[j] = seen[pb] >> (4 * r + j) & 1 ? y : 0;
          }
          transpose4(p, by_digit);
          uint32_t* pw = reinterpret_cast<uint32_t*>((pb ? pb_lds + r * PATH_LDS : pl + 16 * r * P_ROW) + 4 * quad * P_ROW) + n16;
#pragma unroll
          for (int i = 0; i < 4; ++i) pw[i * P_ROW / 4] = by_digit[i];
        }
      }
      fence();
      v4i pa[R], pn[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        pa[r] = pn[r] = v4i{0, 0, 0, 0};
        if (page >= 0) pa[r] = *reinterpret_cast<const v4i*>(pl + (16 * r + n16) * P_ROW + quad * 16);
        if (page_behind >= 0) pn[r] = *reinterpret_cast<const v4i*>(pb_lds + r * PATH_LDS + n16 * P_ROW + quad * 16);
      }
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        v4i v = {0, 0, 0, 0}, vn = {0, 0, 0, 0};
        if (page >= 0) v = *reinterpret_cast<const v4i*>(codes + St::value_at(n16, t, quad));
        if (page_behind >= 0) vn = *reinterpret_cast<const v4i*>(a.p.values + behind + (16 * t + n16) * PAGE + quad * 16);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          v4i o = {0, 0, 0, 0};
          if (page >= 0) o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa[r], v, o, 0, 0, 0);
          if (page_behind >= 0) o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pn[r], vn, o, 0, 0, 0);
          acc[r][t] = fmaf(undigit(o), be[r], acc[r][t] * xw[r]);
        }
      }
      fence();
    };

    const int bpu = ul / PAGE, all_blocks = last / PAGE + (last >= 0);
    int u = u_first;
    const int blocks = SPLIT ? min(all_blocks, (u + (int)a.per_wave) * bpu) : all_blocks;
    const int last_place = (history + rows - 1) / PAGE;  // the last row's page
    // whether a block's place is hidden, one a lane: on its way with the block before
    auto hidden_at = [&](int b) -> uint32_t {
      const int64_t t = (int64_t)b * PAGE + lane;
      return hid && t < a.hidden_len ? hid[t] : 0;
    };
    int b = u * bpu, page = b < blocks ? page_at(b) : -1;
    uint32_t hidden = hidden_at(b);
    if (ul != ul_first) {
      meet();  // every wave is done with the codes of the rows before
      if (page >= 0) copy(page, 0);
    }
    for (int buf = 0; b < blocks; ++b, buf ^= 1) {
      meet();
      const int next = b + 1 < blocks ? page_at(b + 1) : -1;
      if (next >= 0) copy(next, buf ^ 1);
      const uint32_t hidden_next = hidden_at(b + 1);
      const uint8_t* const codes = lds + buf * St::BYTES;
      if (b * PAGE <= pmax) {
        const uint64_t hide = __ballot(hidden != 0);
        if (b >= first_path) {
          const int behind = b < last_place ? (b + 1 < blocks ? next : page_at(b + 1)) : -1;
          const uint64_t hide_behind = b < last_place ? __ballot(hidden_next != 0) : 0;
          path_block(b, page, behind, hide, hide_behind, !(hide | hide_behind) && page >= 0 && (behind >= 0 || b >= last_place), codes);
        } else if (page >= 0) {
          if (!hide && b * PAGE + PAGE - 1 <= pmin)
            block(std::true_type(), b, hide, codes);
          else
            block(std::false_type(), b, hide, codes);
        }
      }
      if (b + 1 == blocks || (b + 1) % bpu == 0) {  // the unit ends
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float lu = row_sum(l[r]);
          if (!SPLIT) {
            float x, y;
            join_weights(M[r], m[r], &x, &y);
#pragma unroll
            for (int t = 0; t < DT; ++t) A[r][t] = fmaf(acc[r][t], y, A[r][t] * x);
            L[r] = fmaf(lu, y, L[r] * x);
          } else if (ps[r] >= 0 && u < unit_count(ps[r])) {
            const uint32_t pr = pair0 + 4 * r + quad;
            float* o = a.part + (((size_t)(sp.start + pr / a.group) * a.nh + g * a.group + pr % a.group) * a.units + u) * (2 + DP);
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
        ++u;
      }
      page = next;
      hidden = hidden_next;
    }
    if (!SPLIT) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // a pair without a position is written in the first pass
        const uint32_t pr = pair0 + 4 * r + quad, j = pr / a.group;
        if (j >= (uint32_t)rows || !(ps[r] >= 0 || (pos[r] < 0 && ul == ul_first))) continue;
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
  __builtin_amdgcn_s_waitcnt(0x0f70);  // nothing may still be on its way into LDS at the end
}

// Joins a row's units in order, as k_attn_join: one workgroup of dp lanes per row of a
// sequence and head. What a row leaves is read before it is known how many units it has: the
// chain of reads bounds it, 5 to 6 us (8 rows of 32 heads over 8000).
__global__ __launch_bounds__(256) void k_tree_join(AttnArgs a) {
  const uint32_t h = blockIdx.x % a.nh, j = blockIdx.x / a.nh % a.r.most_rows, seq = blockIdx.x / a.nh / a.r.most_rows;
  const Span sp = span_of(a.r.row_start, a.r.kv_len, seq, a.r.rows);
  if (j >= (uint32_t)sp.n) return;
  const uint32_t row = sp.start + j, d = threadIdx.x, dp = a.p.dp, lane = threadIdx.x % WAVE;
  const int up = Tree::up(a.parent, sp);
  const float* p = a.part + ((size_t)row * a.nh + h) * a.units * (2 + dp);
  static_assert(MAX_UNITS <= WAVE, "a unit for each lane");
  const float ml = lane < a.units ? p[lane * (2 + dp)] : 0.0f, ll = lane < a.units ? p[lane * (2 + dp) + 1] : 0.0f;
  float M = -INFINITY, L = 0.0f, A = 0.0f;
  constexpr int AT_ONCE = 32;
  float acc[AT_ONCE];
#pragma unroll
  for (int e = 0; e < AT_ONCE; ++e) acc[e] = e < (int)a.units ? p[e * (2 + dp) + 2 + d] : 0.0f;
  const Tree tree(up);
  const int n = unit_count(min(tree.pos(sp, j), a.most_len - 1));
  for (int u0 = 0; u0 < n; u0 += AT_ONCE) {
    if (u0) {
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) acc[e] = u0 + e < n ? p[(u0 + e) * (2 + dp) + 2 + d] : 0.0f;
    }
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

// How a call's pairs are dealt.
struct TreePlan {
  bool split;
  uint32_t R, groups, units, per_wave;  // groups: workgroups of a sequence and cache head
  size_t lds, workspace;
};
TreePlan plan_of(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t dp, uint32_t most_len) {
  const uint32_t pairs = r.most_rows * (heads / kv_heads);
  TreePlan p;
  auto groups_of = [&](uint32_t R) { return (pairs + 4 * TREE_WAVES * R - 1) / (4 * TREE_WAVES * R); };
  auto all_of = [&](uint32_t R) { return (uint64_t)r.sequences * kv_heads * groups_of(R); };
  // Two tiles a wave share what it reads from LDS, where there are waves enough
  // without (us with one and two, 8B rows: 32 x 48 of 2000 301 and 277, 64 x 16 of 1000 118 and
  // 110, but 16 x 33 of 3000, 1,152 workgroups, 190 and 205).
  p.R = dp <= 128 && all_of(1) >= 2048 ? 2 : 1;
  p.groups = groups_of(p.R);
  p.units = (uint32_t)most_units(most_len);
  // Fewer workgroups than CUs: a row's units are dealt to about three a CU (us in one
  // piece and dealt: 8 8B rows of 8000 132 and 26, 64 360M rows of 3500 55 and 24, 3 x 30 1B
  // rows of 1500 33 and 27; 7 135M rows of 203, two units, 9.0 and 10.6; 7 x 25 8B rows
  // of 6000, 392 workgroups, 162 and 179).
  const size_t partials = (size_t)r.rows * heads * p.units * (2 + dp) * sizeof(float);
  p.split = p.units >= 4 && all_of(p.R) < 256 && partials <= ((size_t)128 << 20);
  p.per_wave = p.split ? (uint32_t)std::max<uint64_t>(1, all_of(p.R) * p.units / 768) : 1;
  p.workspace = p.split ? partials : 0;
  p.lds = 2 * (2 * PAGE * dp + 2 * PAGE * 4) + TREE_WAVES * path_lds(p.R);
  return p;
}

template <int R, bool SPLIT>
int tree_launch(const AttnArgs& a, uint32_t blocks, size_t lds, hipStream_t s) {
  const uint32_t threads = WAVE * TREE_WAVES;
  switch (a.p.dp / 64) {
    case 1: return launch(k_tree<1, R, SPLIT>, blocks, threads, lds, s, a);
    case 2: return launch(k_tree<2, R, SPLIT>, blocks, threads, lds, s, a);
    case 3: if constexpr (R == 1) return launch(k_tree<3, R, SPLIT>, blocks, threads, lds, s, a); break;
    case 4: if constexpr (R == 1) return launch(k_tree<4, R, SPLIT>, blocks, threads, lds, s, a); break;
  }
  return defer_gpu_fail_(DEFER_GPU_E_INVALID, "no attention kernel for head_dim %u", a.hd);
}

}  // namespace

size_t tree_attention_workspace(const Rows& r, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t most_len) {
  if (!r.rows || !r.sequences || !r.most_rows || r.most_rows > MAX_TREE) return 0;
  return plan_of(r, heads, kv_heads, padded(head_dim), most_len).workspace;
}

int tree_attention(const Pages& p, const Rows& r, const Attention& in, void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (!r.rows) return DEFER_GPU_OK;
  if (!r.sequences || !r.most_rows)
    return in.clear ? launch(k_zero_rows, r.rows, 256, 0, s, in.out, in.out_stride, in.heads * in.head_dim, in.type) : DEFER_GPU_OK;
  const TreePlan pl = plan_of(r, in.heads, p.heads, p.dp, in.most_len);
  if (pl.workspace && (!workspace || workspace_bytes < pl.workspace))
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "attention needs a workspace of %zu bytes, got %zu", pl.workspace,
                           workspace ? workspace_bytes : (size_t)0);
  AttnArgs a = attn_args(p, r, in, workspace);
  a.units = pl.units;
  a.per_wave = pl.per_wave;
  const uint32_t chunks = pl.split ? (pl.units + pl.per_wave - 1) / pl.per_wave : 1;
  const uint64_t blocks = (uint64_t)pl.groups * chunks * r.sequences * p.heads;
  if (blocks > MAX_THREADS / (WAVE * TREE_WAVES) || (pl.split && (uint64_t)r.sequences * r.most_rows * in.heads > MAX_THREADS / p.dp))
    return defer_gpu_fail_(DEFER_GPU_E_INVALID, "too many rows for one call");
  const uint32_t nb = (uint32_t)blocks;
  if (!pl.split) return pl.R == 1 ? tree_launch<1, false>(a, nb, pl.lds, s) : tree_launch<2, false>(a, nb, pl.lds, s);
  const int rc = tree_launch<1, true>(a, nb, pl.lds, s);  // (two tiles a wave are for many workgroups)
  return rc ? rc : launch(k_tree_join, r.sequences * r.most_rows * in.heads, p.dp, 0, s, a);
}

}  // namespace q8
