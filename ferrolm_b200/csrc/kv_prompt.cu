// Attention of many rows of a sequence (a prompt, or a piece of one) over blocks of a key/value cache.
//
// Every row has a list of blocks of its own, and neighbours have many of them in common.  A CTA has 32 queries for each of its
// four warps (8 rows of a group of 4 heads, say), goes once over the union of their lists in ascending order, 64 rows of the
// cache at a time, and a warp passes over pieces of 16 rows that none of its own rows has.  With one 128-row tile for the CTA,
// as a tcgen05 product wants it, every row of the tile would pay for the blocks of all others; the warps' own tiles of
// mma.sync, at a quarter of the rate, pay for those of eight rows.  Bound by these products and, where lists have little in
// common, by the copies.
//
// S = Q K^T with 16 queries to a tile, whose weights are the operand of O = P V as they stand in registers.  32 rows of keys share
// a read of the queries.  A maximum that grows by less than a factor of 2 (fp16) or 256 (bf16) is left as it was: the weights
// stay within their type, and the sums need not be scaled as often.  Values that are not finite would reach rows that do not
// see them as 0 * inf: stages that hold some are worked on without them, and they are added where they are seen.
#include <climits>

#include "kv.cuh"

namespace fv {

namespace {

enum { KV_PROMPT_THREADS = 128, KV_PROMPT_WARPS = 4, KV_PROMPT_COLS = 32 };

template <int KIND, int D>
struct Tile {
  static constexpr int BYTES = KIND == FV_KV_SAME ? 2 : 1, ROW = D * BYTES;
  static constexpr int PITCH = ROW + 16;  // an odd number of 16 bytes: eight rows lie in different banks
  static constexpr int ROWS = 64;         // of the cache, in a stage
  static constexpr int STAGE = 2 * ROWS * PITCH + (KIND == FV_KV_SAME ? 0 : 2 * ROWS * 4) + 16;  // keys, values, scales, positions
  static constexpr int STAGES = KIND == FV_KV_SAME ? 2 : 3;
  static constexpr int Q_PITCH = 2 * D + 16;
  static constexpr int Q = KV_PROMPT_WARPS * KV_PROMPT_COLS * Q_PITCH;
  static constexpr int SMEM = Q + STAGES * STAGE;  // and the bits of the union behind it
};

__device__ __forceinline__ void ldmatrix(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}

// 0x7F80 or 0x7C00 in both halves: the exponent of what is not finite
template <class T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {  // zeros in the halves that are not finite
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
  return w & ~__vcmpeq2(w & e, e);
}
// x + 0 * w in both halves: NaN from the first that is not finite on
template <class T>
__device__ __forceinline__ uint32_t watch(uint32_t x, uint32_t w) {
  uint32_t y;
  if constexpr (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(w), "r"(0u), "r"(x));
  else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(w), "r"(0u), "r"(x));
  return y;
}

template <class T, int KIND, int D>
__global__ void __launch_bounds__(KV_PROMPT_THREADS, 2) kv_prompt_kernel(KvAttend a, KvBatch m, int tiles) {
  using S = Tile<KIND, D>;
  using M = typename std::conditional<KIND == FV_KV_SAME, T, __half>::type;
  constexpr int COLS = KV_PROMPT_COLS, W = KV_PROMPT_WARPS;  // columns: a row and a query head
  constexpr float ONE = std::is_same<M, __half>::value ? 14.f : 0.f;  // log2 of what stands for a weight of 1
  constexpr float GROWN = std::is_same<M, __half>::value ? 1.f : 8.f;   // log2 of what a maximum may lag behind by
  unsigned char* const ring = dyn_smem() + S::Q;
  uint32_t* const bits = reinterpret_cast<uint32_t*>(dyn_smem() + S::SMEM);
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;

  // which rows of which sequence
  const int tw = a.group <= COLS ? COLS / a.group : 1, tc = tw * W;  // rows of a warp and of the CTA
  const int head = blockIdx.y / tiles, first = (blockIdx.y % tiles) * COLS;
  const int cols = tiles > 1 ? min(COLS, a.group - first) : tw * a.group;  // of a warp
  const int per = tiles > 1 ? COLS : a.group;                             // columns of a row
  const int item = int(gridDim.x - 1 - blockIdx.x);                        // the rows that see most come first
  const int b = m.cu ? kv_find(m, item, tc, 1) : min(item, m.nseq - 1);
  const int r0 = m.cu_at(b), r1 = max(m.cu_at(b + 1), r0);
  const int row0 = m.cu ? r0 + (item - (r0 / tc + b)) * tc : r0, rows = min(tc, r1 - row0);
  if (row0 < r0 || rows <= 0 || (!m.cu && item >= m.nseq)) return;
  const int pos_cta = __ldg(m.lens + b) - r1 + row0, last = pos_cta + rows - 1;  // positions of the first and the last row
  const int blocks = min(m.table_width, last < 0 ? 0 : (last >> m.page_shift) + 1);
  const int row = row0 + warp * tw, mine = min(tw, max(0, rows - warp * tw)), pos = pos_cta + warp * tw;
  const unsigned everyone = mine == 32 ? ~0u : (1u << mine) - 1u;

  // the union of the lists
  if (a.blocks) {
    for (int i = threadIdx.x; i < (blocks + 31) / 32; i += KV_PROMPT_THREADS) bits[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < rows * a.k; i += KV_PROMPT_THREADS) {
      const int r = i / a.k, e = __ldg(a.blocks + (size_t(row0 + r) * a.heads + head) * a.k + (i - r * a.k));
      if (e >= 0 && e < blocks) atomicOr(bits + (e >> 5), 1u << (e & 31));
    }
  }
  // the queries, a column each: in 8 bits as fp16 times a power of two, and in the order in which the codes come
  unsigned char* const sq = dyn_smem() + warp * (COLS * S::Q_PITCH);
  float by[2][2];  // of a lane's columns: 16 x + 8 i + g
  {
    float f[COLS / 4];  // of column 4 i + lane / 8, by the eight lanes that have it
#pragma unroll
    for (int i = 0; i < COLS / 4; ++i) {
      const int c = 4 * i + (lane >> 3), tok = c / per, h = first + c - tok * per;
      const bool on = tok < mine && c < cols && h < a.group;
      const unsigned char* src = a.q + size_t(row + (on ? tok : 0)) * a.q_row + size_t(head * a.group + (on ? h : 0)) * a.q_head;
      uint4 w[(D / 8 + 7) / 8];
      float most = 0.f;
#pragma unroll
      for (int x = 0; x < (D / 8 + 7) / 8; ++x) {
        const int p = (lane & 7) + 8 * x;
        w[x] = make_uint4(0, 0, 0, 0);
        if (on && p < D / 8) w[x] = __ldg(reinterpret_cast<const uint4*>(src) + p);
        if constexpr (!std::is_same<M, T>::value) {
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const float2 y = Pair<T>::to_float(reinterpret_cast<const uint32_t*>(&w[x])[z]);
            most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));
          }
        }
      }
      f[i] = 1.f;
      if constexpr (!std::is_same<M, T>::value) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(FV_FULL, most, o));
        f[i] = half_factor(most);
      }
#pragma unroll
      for (int x = 0; x < (D / 8 + 7) / 8; ++x) {
        const int p = (lane & 7) + 8 * x;
        if (p >= D / 8) continue;
        if constexpr (KIND == FV_KV_SAME) {
          *reinterpret_cast<uint4*>(sq + c * S::Q_PITCH + p * 16) = w[x];
        } else {
          // components 4 t .. 4 t + 3 of 16 stand at 2 t, 2 t + 1, 8 + 2 t, 8 + 2 t + 1; these 8 are the first or second half
          uint32_t* to = reinterpret_cast<uint32_t*>(sq + c * S::Q_PITCH + (p >> 1) * 32);
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            uint32_t y = reinterpret_cast<const uint32_t*>(&w[x])[z];
            if constexpr (!std::is_same<M, T>::value) {
              const float2 v = Pair<T>::to_float(y);
              y = Pair<M>::from_float(v.x * f[i], v.y * f[i]);
            }
            to[(p & 1) * 2 + (z >> 1) + (z & 1) * 4] = y;
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // column 4 j + lane / 8 of f[j]
        const float lo = __shfl_sync(FV_FULL, f[4 * x + 2 * i], (g & 3) * 8), hi = __shfl_sync(FV_FULL, f[4 * x + 2 * i + 1], (g & 3) * 8);
        by[x][i] = a.scale / (g < 4 ? lo : hi);
      }
  }
  int row_of[2][2];  // of a lane's columns; 31, which no warp has with a column to spare, for none
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 16 * x + 8 * i + g;
      row_of[x][i] = c < cols && c / per < mine ? c / per : 31;
    }
  __syncthreads();

  // the walk over the pieces of the union: block `at`, whose page is `page`, piece `sub`; the block after it is known already
  int at = -1, page = -1, sub = 0, after = -1, after_page = -1;
  auto look = [&]() {  // the next block with a page
    at = after, page = after_page, sub = 0;
    if (after >= blocks) return;
    ++after;
    if (a.blocks) {
      int w = after >> 5;
      uint32_t x = after < blocks ? bits[w] & (~0u << (after & 31)) : 0u;
      while (x == 0u && ++w < (blocks + 31) / 32) x = bits[w];
      after = x ? w * 32 + __ffs(int(x)) - 1 : blocks;
    }
    after_page = m.page(b, after < blocks ? after : -1);
  };
  const int pieces = 1 << (m.page_shift - 4);
  auto fill = [&](int stage) {
    unsigned char* s = ring + stage * S::STAGE;
    const uint32_t to = uint32_t(__cvta_generic_to_shared(s));
    int* where = reinterpret_cast<int*>(s + S::STAGE - 16);
    for (int p = 0; p < 4; ++p) {
      while (at < blocks && (page < 0 || sub == pieces || (at << m.page_shift) + sub * 16 > last)) look();
      const int start = at < blocks ? (at << m.page_shift) + sub * 16 : -1;
      if (threadIdx.x == 0) where[p] = start;
      if (start < 0) continue;
      const size_t from = ((size_t(page) * a.heads + head) << m.page_shift) + sub * 16;
      ++sub;
#pragma unroll
      for (int i = 0; i < (S::ROW + KV_PROMPT_THREADS - 1) / KV_PROMPT_THREADS; ++i) {
        const int u = threadIdx.x + i * KV_PROMPT_THREADS, r = u / (S::ROW / 16), x = (u - r * (S::ROW / 16)) * 16, bytes = start + r <= last ? 16 : 0;
        if (S::ROW % KV_PROMPT_THREADS && u >= S::ROW) break;
        const uint32_t dst = to + (16 * p + r) * S::PITCH + x;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(a.kp + from * S::ROW + u * 16), "r"(bytes));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + S::ROWS * S::PITCH), "l"(a.vp + from * S::ROW + u * 16), "r"(bytes));
      }
      if constexpr (KIND != FV_KV_SAME) {
        if (threadIdx.x < 32) {
          const int r = threadIdx.x & 15, bytes = start + r <= last ? 4 : 0;
          const float* src = (threadIdx.x < 16 ? a.k_scale : a.v_scale) + from + r;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 2 * S::ROWS * S::PITCH + ((threadIdx.x >> 4) * S::ROWS + 16 * p + r) * 4), "l"(src), "r"(bytes));
        }
      }
    }
    asm volatile("cp.async.commit_group;");
  };
  look();  // `after` becomes the first block
  look();
#pragma unroll 1
  for (int i = 0; i < S::STAGES - 1; ++i) fill(i);

  // a lane has the list of one of its warp's rows: the entry that is next, and the one behind it on its way
  const int32_t* const list = a.blocks ? a.blocks + (size_t(row + (lane < mine ? lane : 0)) * a.heads + head) * a.k : nullptr;
  int entry = -1, ahead = a.blocks && lane < mine ? __ldg(list) : 0, index = 0;

  float o[2][D / 8][4], top[2][2], l[2][2];  // tiles of 16 columns; of 8 components
  int unit = 0;  // 8 bits: values stand for multiples of 2^(unit - 126)
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    top[x][0] = top[x][1] = -INFINITY, l[x][0] = l[x][1] = 0.f;
#pragma unroll
    for (int u = 0; u < D / 8; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[x][u][i] = 0.f;
  }
  const int r8 = lane & 7, second = lane >> 3 & 1, third = lane >> 4;  // which row of which of four 8 x 8 tiles a lane points at
  const uint32_t q_at = uint32_t(__cvta_generic_to_shared(sq)) + (r8 + second * 8) * S::Q_PITCH + third * 16;

  // 32 rows of the cache, in two pieces that begin at start[0] and start[1] and are seen by who[0] and who[1]; ALL: by every row of
  // the warp, whole.  ODD: some of their values are not finite.
  auto take = [&](const unsigned char* s, int pair, const int* start, const unsigned* who, auto all_of, auto odd_of) {
    constexpr bool ALL = decltype(all_of)::value, ODD = decltype(odd_of)::value;
    const uint32_t keys = uint32_t(__cvta_generic_to_shared(s)) + 32 * pair * S::PITCH, values = keys + S::ROWS * S::PITCH;
    [[maybe_unused]] const float* const scales = reinterpret_cast<const float*>(s + 2 * S::ROWS * S::PITCH) + 32 * pair;
    float sc[2][4][4] = {};  // tiles of columns; of 8 rows of the cache
    if constexpr (KIND == FV_KV_SAME) {
      const uint32_t k_at = keys + (r8 + third * 8) * S::PITCH + second * 16;
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        uint32_t q[2][4], k[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) ldmatrix(q[x], q_at + x * 16 * S::Q_PITCH + st * 32), ldmatrix(k[x], k_at + x * 16 * S::PITCH + st * 32);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) mma_16<M>(sc[x][j], q[x][0], q[x][1], q[x][2], q[x][3], k[j >> 1][(j & 1) * 2], k[j >> 1][(j & 1) * 2 + 1]);
      }
    } else {
      const uint32_t k_at = keys + (r8 + second * 8) * S::PITCH + third * 16;
#pragma unroll
      for (int st = 0; st < D / 32; ++st) {
        uint32_t c[2][4];  // 16 rows each: rows 0-7 and 8-15 of 16 components, then of the next 16
#pragma unroll
        for (int h = 0; h < 2; ++h) ldmatrix(c[h], k_at + h * 16 * S::PITCH + st * 32);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t q[2][4], k[4][2];
#pragma unroll
          for (int x = 0; x < 2; ++x) ldmatrix(q[x], q_at + x * 16 * S::Q_PITCH + (2 * st + z) * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j) codes_to_half<KIND>(c[j >> 1][2 * z + (j & 1)], k[j][0], k[j][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) mma_16<M>(sc[x][j], q[x][0], q[x][1], q[x][2], q[x][3], k[j][0], k[j][1]);
        }
      }
    }
    [[maybe_unused]] float vs[4][2];  // of a lane's rows of the cache: 8 j + 2 t + i
    float grown = 1.f;
    if constexpr (KIND != FV_KV_SAME) {
      float most = 0.f;  // leaves NaN out: it reaches the sums through its weight
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * t);
        float2 v = *reinterpret_cast<const float2*>(scales + S::ROWS + 8 * j + 2 * t);
        if (!ALL && start[j >> 1] < 0) v = make_float2(0.f, 0.f);
        most = fmaxf(most, fmaxf(v.x, v.y));
        vs[j][0] = v.x, vs[j][1] = v.y;
#pragma unroll
        for (int x = 0; x < 2; ++x) sc[x][j][0] *= ks.x, sc[x][j][1] *= ks.y, sc[x][j][2] *= ks.x, sc[x][j][3] *= ks.y;
      }
      const int e = max(unit, int(__reduce_max_sync(FV_FULL, __float_as_uint(most)) >> 23));
      grown = __uint_as_float(uint32_t(max(127 + unit - e, 0)) << 23);
      unit = e;
      const float down = __uint_as_float(uint32_t(max(253 - e, 1)) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) vs[j][0] *= down, vs[j][1] *= down;
    }
    bool moved = grown != 1.f;
    float to[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool seen = ALL || (who[j >> 1] >> row_of[x][i] & 1u);
          const int ahead = pos + row_of[x][i] - start[j >> 1] - 8 * (j & 1) - 2 * t;  // rows of the cache up to the column's own
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            float& v = sc[x][j][2 * i + z];
            v *= by[x][i];
            if (!ALL && !(seen && z <= ahead)) v = -INFINITY;
            y = fmaxf(y, v);
          }
        }
        to[x][i] = y;
        moved = moved || y > top[x][i] + GROWN;  // -inf + GROWN is -inf
      }
    if (__any_sync(FV_FULL, moved)) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y = fmaxf(top[x][i], to[x][i]);
          y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 1));
          y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 2));
          const float by_l = y > top[x][i] ? exp2_of(top[x][i] - y) : 1.f, by_o = by_l * grown;
          top[x][i] = y;
          l[x][i] *= by_l;
#pragma unroll
          for (int u = 0; u < D / 8; ++u) o[x][u][2 * i] *= by_o, o[x][u][2 * i + 1] *= by_o;
        }
    }
    // weights, rounded to 16 bits: tiles of 16 columns by 16 rows of the cache
    uint32_t p[2][2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float off = top[x][i] == -INFINITY ? 0.f : ONE - top[x][i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            y[z] = exp2_of(sc[x][j][2 * i + z] + off);
            l[x][i] += y[z];
            if constexpr (KIND != FV_KV_SAME) y[z] = y[z] != 0.f ? y[z] * vs[j][z] : 0.f;
            if constexpr (ODD) sc[x][j][2 * i + z] = y[z];
          }
          p[x][j >> 1][i + 2 * (j & 1)] = Pair<M>::from_float(y[0], y[1]);
        }
      }
    if constexpr (KIND == FV_KV_SAME) {
      const uint32_t v_at = values + (r8 + second * 8) * S::PITCH + third * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!ALL && start[h] < 0) continue;  // its place holds anything
#pragma unroll
        for (int u = 0; u < D / 8; u += 2) {
          uint32_t v[4];
          ldmatrix_t(v, v_at + h * 16 * S::PITCH + u * 16);
          if constexpr (ODD) {
#pragma unroll
            for (int z = 0; z < 4; ++z) v[z] = finite_only<T>(v[z]);
          }
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int x = 0; x < 2; ++x) mma_16<M>(o[x][u + z], p[x][h][0], p[x][h][1], p[x][h][2], p[x][h][3], v[2 * z], v[2 * z + 1]);
        }
        if constexpr (ODD) {  // what was left out, to the columns that have a weight for it
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {
            const T* vr = reinterpret_cast<const T*>(s + (S::ROWS + 32 * pair + 16 * h + j) * S::PITCH);
            float w[2][2];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float y = 0.f;  // tile j / 8 of the piece, lane j / 2 % 4, number j % 2
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  const float here = __shfl_sync(FV_FULL, sc[x][2 * h + (z >> 1)][2 * i + (z & 1)], (lane & ~3) + (j >> 1 & 3));
                  if ((j >> 3) == (z >> 1) && (j & 1) == (z & 1)) y = here;
                }
                w[x][i] = y;
              }
#pragma unroll
            for (int u = 0; u < D / 8; ++u)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const float v = float(vr[8 * u + 2 * t + z]);
                if (kv_finite(v)) continue;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (w[x][i] != 0.f) o[x][u][2 * i + z] += w[x][i] * v;
              }
          }
        }
      }
    } else {
      const uint32_t v_at = values + (r8 + second * 8) * S::PITCH + third * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!ALL && start[h] < 0) continue;
#pragma unroll
        for (int u = 0; u < D / 8; u += 4) {
          uint32_t c[4];  // rows 0-7 and 8-15 of 16 components, then of the next 16
          ldmatrix_t(c, v_at + h * 16 * S::PITCH + u * 8);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            uint32_t v[2][2];  // the even and the odd components of 16, of two neighbouring rows each
#pragma unroll
            for (int i = 0; i < 2; ++i) codes_to_half<KIND>(__byte_perm(c[2 * z + i], 0, 0x3120), v[0][i], v[1][i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int x = 0; x < 2; ++x) mma_16<M>(o[x][u + 2 * z + i], p[x][h][0], p[x][h][1], p[x][h][2], p[x][h][3], v[i][0], v[i][1]);
          }
        }
      }
    }
  };

#pragma unroll 1
  for (int stage = 0;; stage = stage + 1 == S::STAGES ? 0 : stage + 1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2));
    unsigned char* const s = ring + stage * S::STAGE;
    int odd = 0;
    if constexpr (KIND == FV_KV_SAME) {  // each thread looks at what it has copied
      uint32_t found = 0u;
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < (S::ROW + KV_PROMPT_THREADS - 1) / KV_PROMPT_THREADS; ++i) {
          const int u = threadIdx.x + i * KV_PROMPT_THREADS, r = u / (S::ROW / 16), x = (u - r * (S::ROW / 16)) * 16;
          if (S::ROW % KV_PROMPT_THREADS && u >= S::ROW) break;
          const uint4 v = *reinterpret_cast<const uint4*>(s + (S::ROWS + 16 * p + r) * S::PITCH + x);
          found = watch<T>(watch<T>(watch<T>(watch<T>(found, v.x), v.y), v.z), v.w);
        }
      odd = __syncthreads_or(found != 0u);  // 0 * w is 0 or -0, and 0 + -0 is 0
    } else {
      __syncthreads();
    }
    const int* const where = reinterpret_cast<const int*>(s + S::STAGE - 16);
    if (where[0] < 0) break;  // the union is done
    fill(stage == 0 ? S::STAGES - 1 : stage - 1);  // the stage that everybody has left
#pragma unroll 1
    for (int pair = 0; pair < 2; ++pair) {
      int start[2];
      unsigned who[2];  // the warp's rows that see the piece
      bool all = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        start[h] = where[2 * pair + h];
        bool sees = lane < mine && start[h] >= 0 && start[h] <= pos + lane;
        if (a.blocks) {
          const int block = start[h] >= 0 ? start[h] >> m.page_shift : -1;
          while (lane < mine && entry < block) {  // entries that are blocks, each above all before it; blocks: none is left
            const int e = ahead;
            ++index;
            ahead = index < a.k ? __ldg(list + index) : 0;
            if (index > a.k) entry = INT_MAX;
            else if (e > entry && e < blocks && (e << m.page_shift) <= pos + lane) entry = e;
          }
          sees = sees && entry == block;
        }
        who[h] = __ballot_sync(FV_FULL, sees);
        all = all && who[h] == everyone && start[h] + 15 <= pos;
      }
      if ((who[0] | who[1]) == 0u) continue;
      using Yes = std::true_type;
      using No = std::false_type;
      if (KIND == FV_KV_SAME && odd) take(s, pair, start, who, No(), std::integral_constant<bool, KIND == FV_KV_SAME>());
      else if (all) take(s, pair, start, who, Yes(), No());
      else take(s, pair, start, who, No(), No());
    }
  }
  asm volatile("cp.async.wait_all;");

  // results: through the place of the warp's own queries, to be written in whole rows
  const float f = KIND != FV_KV_SAME ? __uint_as_float(uint32_t(min(unit + 1, 254)) << 23) : 1.f;
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y = l[x][i];
      y += __shfl_xor_sync(FV_FULL, y, 1);
      y += __shfl_xor_sync(FV_FULL, y, 2);
      const int c = 16 * x + 8 * i + g, tok = c / per;
      const float down = y == 0.f ? 0.f : f / y;
      uint32_t* to = reinterpret_cast<uint32_t*>(sq + c * S::Q_PITCH);
#pragma unroll
      for (int u = 0; u < D / 8; u += 2) {
        float v[4] = {o[x][u][2 * i], o[x][u][2 * i + 1], o[x][u + 1][2 * i], o[x][u + 1][2 * i + 1]};
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = y == 0.f ? 0.f : v[z] * down;
        if constexpr (KIND == FV_KV_SAME) {
          to[4 * u + t] = Pair<T>::from_float(v[0], v[1]), to[4 * u + 4 + t] = Pair<T>::from_float(v[2], v[3]);
        } else {  // components 4 t, 4 t + 2, 4 t + 1, 4 t + 3 of 16
          *reinterpret_cast<uint2*>(to + 4 * u + 2 * t) = make_uint2(Pair<T>::from_float(v[0], v[2]), Pair<T>::from_float(v[1], v[3]));
        }
      }
      if (a.lse && t == 0 && c < cols && tok < mine)
        a.lse[size_t(row + tok) * a.heads * a.group + size_t(head) * a.group + first + c - tok * per] =
            y == 0.f ? -INFINITY : (top[x][i] - ONE + log2f(y)) * 0.693147180559945309f;
    }
  __syncwarp();
  for (int i = lane; i < COLS * (D / 8); i += 32) {
    const int c = i / (D / 8), x = i - c * (D / 8), tok = c / per;
    if (c < cols && tok < mine)
      *reinterpret_cast<uint4*>(a.out + ((size_t(row + tok) * a.heads * a.group + size_t(head) * a.group + first + c - tok * per) * D + x * 8) * 2) =
          *reinterpret_cast<const uint4*>(sq + c * S::Q_PITCH + x * 16);
  }
}

template <class T, int KIND, int D>
int prompt_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a) {
  using S = Tile<KIND, D>;
  const int tiles = (a.group + KV_PROMPT_COLS - 1) / KV_PROMPT_COLS, tc = KV_PROMPT_WARPS * (a.group <= KV_PROMPT_COLS ? KV_PROMPT_COLS / a.group : 1);
  const size_t items = b->cu ? b->rows / tc + b->nseq : b->nseq, smem = S::SMEM + (b->table_width + 31) / 32 * 4;
  if (size_t(kv->heads) * tiles > 65535) return fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: more than 65535 tiles of query heads");
  FV_TRY((kv_allow_smem<kv_prompt_kernel<T, KIND, D>>(kv->device, smem)));
  kv_prompt_kernel<T, KIND, D><<<dim3(unsigned(items), unsigned(kv->heads * tiles)), KV_PROMPT_THREADS, smem, s>>>(a, kv_batch(kv, b), tiles);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // namespace

int kv_prompt_attend(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a) { FV_KV_DISPATCH(kv, prompt_of, kv, s, b, a); }

}  // namespace fv
