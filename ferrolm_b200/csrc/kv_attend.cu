// Attention of single rows (tokens) over blocks of a key/value cache, and the entry point of both kinds of attention.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale q . k_j - max),  lse = log of the sum
//
// One row has as many queries to a key head as its group has heads, so a key is read for a few products only: the bytes of the
// blocks bound it.  A CTA, or a cluster of up to 8 where there are few rows, works on one row and key head; its warps take 16
// rows of a block at a time, each with a running maximum and sum of its own, straight from memory into the operands of matrix
// products: no shared memory, no barrier and no other warp stands between a warp and its loads.  They are joined at the end,
// within a cluster through its shared memory.
//
// The products are S^T = K Q^T and O^T = V^T P^T, so that 8 queries fill a tile that would have 16 the other way round.  Sums
// over components may go in any order, so lane t of four holds neighbouring components where the product would have it
// hold some of each 16: loads are 16 bytes.  V's rows arrive a lane each and are paired by byte permutations, P^T comes from S^T by a
// transposition in registers.
//
// In 8 bits the codes are exact in fp16; a key's scale multiplies its score, a value's its weight, relative to the largest
// power of two of a scale so far.  Weights are rounded to 16 bits for the second product: fp16 with 2^14 for 1, so that none
// above 2^-28 loses bits, or two bf16 numbers (a weight and what its rounding left), which is as good; the loads leave the time.
#include <climits>

#include <cooperative_groups.h>

#include "kv.cuh"

namespace fv {

namespace {

namespace cg = cooperative_groups;

enum { KV_TOKEN_WARPS = 4 };

// bytes that lie next to one another, N registers of them
template <int N>
__device__ __forceinline__ void load_words(uint32_t* to, const void* from) {
  if constexpr (N == 4) {
    const uint4 x = __ldg(static_cast<const uint4*>(from));
    to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = __ldg(static_cast<const uint2*>(from));
    to[0] = x.x, to[1] = x.y;
  } else {
    to[0] = __ldg(static_cast<const uint32_t*>(from));
  }
}

// Where a lane's components lie.  Keys: step s of 16 components takes four neighbouring ones from lane t of four.  Values:
// lane g of eight has dim / 8 components, in pieces of 16, 8 or 4 bytes.
template <int KIND, int D>
struct Layout {
  static constexpr int BYTES = KIND == FV_KV_SAME ? 2 : 1;
  static constexpr int KEY_WORDS = KIND != FV_KV_SAME && D == 96 ? 2 : 4;  // of one load
  static constexpr int KEY_LOADS = D * BYTES / 4 / (4 * KEY_WORDS);        // for a row, by each of 4 lanes
  static constexpr int PER_LOAD = 4 * KEY_WORDS / BYTES;                   // components
  static __device__ __forceinline__ int key_at(int step, int t) {          // first of the four
    constexpr int steps = PER_LOAD / 4;
    return (step / steps) * (4 * PER_LOAD) + t * PER_LOAD + (step % steps) * 4;
  }
  static constexpr int VALUE_WORDS = D * BYTES / 32;
  static constexpr int FIRST = KIND == FV_KV_SAME ? 8 : D == 128 ? 16 : 8;  // components of the first piece
  static constexpr int REST = D / 8 - FIRST;                               // and of the second: 0, 4 or 8
  static __device__ __forceinline__ int value_at(int e, int g) {
    return e < FIRST ? g * FIRST + e : 8 * FIRST + g * REST + (e - FIRST);
  }
  static __device__ __forceinline__ void load_value(uint32_t* to, const unsigned char* row, int g) {
    constexpr int w = FIRST * BYTES / 4;
    load_words<w>(to, row + g * FIRST * BYTES);
    if constexpr (REST > 0) load_words<REST * BYTES / 4>(to + w, row + (8 * FIRST + g * REST) * BYTES);
  }
};

// 16 rows of one block as a warp holds them: lane (g, t) has keys g and g + 8 and values 2t, 2t + 1, 2t + 8, 2t + 9
template <int KIND, int D>
struct Rows {
  using L = Layout<KIND, D>;
  uint32_t k[2][L::KEY_LOADS * L::KEY_WORDS];
  uint32_t v[4][L::VALUE_WORDS];
  float ks[2], vs[2];
  int visible;  // of the 16; 0: nothing was loaded

  __device__ __forceinline__ void load(const KvAttend& a, int page, int head, int page_shift, int slot, int seen, int g, int t) {
    visible = min(seen, 16);
    if (visible <= 0) return;
    const size_t at = ((size_t(page) * a.heads + head) << page_shift) + slot;
    const unsigned char* kr = a.kp + (at + g) * (D * L::BYTES);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < L::KEY_LOADS; ++c)
        load_words<L::KEY_WORDS>(&k[i][c * L::KEY_WORDS], kr + i * 8 * (D * L::BYTES) + (c * 4 + t) * (4 * L::KEY_WORDS));
#pragma unroll
    for (int i = 0; i < 4; ++i) L::load_value(v[i], a.vp + (at + 2 * t + (i & 1) + (i & 2) * 4) * (D * L::BYTES), g);
    if constexpr (KIND != FV_KV_SAME) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ks[i] = __ldg(a.k_scale + at + g + 8 * i), vs[i] = __ldg(a.v_scale + at + g + 8 * i);
    }
    if (visible < 16) {  // rows that are not there may hold anything: zeros in their place
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * t + (i & 1) + (i & 2) * 4 >= visible) {
#pragma unroll
          for (int w = 0; w < L::VALUE_WORDS; ++w) v[i][w] = 0u;
        }
      if constexpr (KIND != FV_KV_SAME) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (g + 8 * i >= visible) vs[i] = 0.f;
      }
    }
  }
};

// A warp's share of a row's attention: NT tiles of 8 queries.  A lane's queries are 8 x + 2 t and the next one.
template <class T, int KIND, int D, int NT>
struct Share {
  using M = typename std::conditional<KIND == FV_KV_SAME, T, __half>::type;
  using L = Layout<KIND, D>;
  static constexpr bool TWO = std::is_same<M, __nv_bfloat16>::value;
  static constexpr float ONE = TWO ? 0.f : 14.f;  // log2 of what stands for a weight of 1
  uint32_t q[D / 16][NT][2];
  float by[NT][2];  // scale of a lane's queries
  float o[D / 16][NT][4], m[NT][2], l[NT][2];
  int unit;  // 8 bits: values stand for multiples of 2^(unit - 126)

  __device__ __forceinline__ void begin(const KvAttend& a, int row, int head, int first, int g, int t) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int h = first + 8 * x + g;
      const bool on = h < a.group;
      const unsigned char* src = a.q + size_t(row) * a.q_row + size_t(head * a.group + (on ? h : 0)) * a.q_head;
      uint32_t w[D / 16][2];
      float most = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        w[s][0] = w[s][1] = 0u;
        if (on) load_words<2>(w[s], src + 2 * L::key_at(s, t));
        if constexpr (!std::is_same<M, T>::value) {
          const float2 u = Pair<T>::to_float(w[s][0]), v = Pair<T>::to_float(w[s][1]);
          most = fmaxf(most, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(v.x), fabsf(v.y))));
        }
      }
      float f = 1.f;
      if constexpr (!std::is_same<M, T>::value) {
        most = fmaxf(most, __shfl_xor_sync(FV_FULL, most, 1));
        most = fmaxf(most, __shfl_xor_sync(FV_FULL, most, 2));
        f = half_factor(most);
      }
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (std::is_same<M, T>::value) {
            q[s][x][i] = w[s][i];
          } else {
            const float2 u = Pair<T>::to_float(w[s][i]);
            q[s][x][i] = Pair<M>::from_float(u.x * f, u.y * f);
          }
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) by[x][i] = a.scale / __shfl_sync(FV_FULL, f, (2 * t + i) * 4);
    }
#pragma unroll
    for (int x = 0; x < NT; ++x) m[x][0] = m[x][1] = -INFINITY, l[x][0] = l[x][1] = 0.f;
#pragma unroll
    for (int u = 0; u < D / 16; ++u)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[u][x][i] = 0.f;
    unit = 0;
  }

  __device__ __forceinline__ void take(const Rows<KIND, D>& r, int g) {
    if (r.visible <= 0) return;
    float s[NT][4] = {};
#pragma unroll
    for (int st = 0; st < D / 16; ++st) {
      uint32_t a[4];
      if constexpr (KIND == FV_KV_SAME) {
        a[0] = r.k[0][2 * st], a[1] = r.k[1][2 * st], a[2] = r.k[0][2 * st + 1], a[3] = r.k[1][2 * st + 1];
      } else {
        codes_to_half<KIND>(r.k[0][st], a[0], a[2]);
        codes_to_half<KIND>(r.k[1][st], a[1], a[3]);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) mma_16<M>(s[x], a[0], a[1], a[2], a[3], q[st][x][0], q[st][x][1]);
    }
    float vs[2] = {1.f, 1.f}, grown = 1.f;
    if constexpr (KIND != FV_KV_SAME) {
      const float most = fmaxf(fmaxf(r.vs[0], r.vs[1]), 0.f);  // leaves NaN out: it reaches the sums through its weight
      const int e = max(unit, int(__reduce_max_sync(FV_FULL, __float_as_uint(most)) >> 23));
      grown = __uint_as_float(uint32_t(max(127 + unit - e, 0)) << 23);
      unit = e;
      const float down = __uint_as_float(uint32_t(max(253 - e, 1)) << 23);
      vs[0] = r.vs[0] * down, vs[1] = r.vs[1] * down;
    }
    bool moved = grown != 1.f;
    float to[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y = s[x][i] * by[x][i & 1];
        if constexpr (KIND != FV_KV_SAME) y *= r.ks[i >> 1];
        s[x][i] = g + (i & 2) * 4 < r.visible ? y : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = fmaxf(s[x][i], s[x][i + 2]);
        y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 4));
        y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 8));
        y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 16));
        to[x][i] = fmaxf(m[x][i], y);
        moved = moved || to[x][i] > m[x][i];
      }
    }
    if (__any_sync(FV_FULL, moved)) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float by_l = to[x][i] > m[x][i] ? exp2_of(m[x][i] - to[x][i]) : 1.f, by_o = by_l * grown;
          m[x][i] = to[x][i];
          l[x][i] *= by_l;
#pragma unroll
          for (int u = 0; u < D / 16; ++u) o[u][x][i] *= by_o, o[u][x][i + 2] *= by_o;
        }
    }
    uint32_t b[NT][2], rest[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = exp2_of(s[x][i] - (m[x][i & 1] == -INFINITY ? 0.f : m[x][i & 1]) + ONE);
        l[x][i & 1] += p[i];
        if constexpr (KIND != FV_KV_SAME) p[i] = p[i] != 0.f ? p[i] * vs[i >> 1] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = Pair<M>::from_float(p[2 * i], p[2 * i + 1]);
        b[x][i] = transposed(w);
        if constexpr (TWO) {
          const float2 f = Pair<M>::to_float(w);
          rest[x][i] = transposed(Pair<M>::from_float(p[2 * i] - f.x, p[2 * i + 1] - f.y));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < D / 16; ++u) {
      uint32_t a[4];
      if constexpr (KIND == FV_KV_SAME) {
        a[0] = __byte_perm(r.v[0][u], r.v[1][u], 0x5410), a[1] = __byte_perm(r.v[0][u], r.v[1][u], 0x7632);
        a[2] = __byte_perm(r.v[2][u], r.v[3][u], 0x5410), a[3] = __byte_perm(r.v[2][u], r.v[3][u], 0x7632);
      } else {
        const int sel = u & 1 ? 0x7362 : 0x5140;  // components 2u and 2u + 1 of two rows
        codes_to_half<KIND>(__byte_perm(r.v[0][u / 2], r.v[1][u / 2], sel), a[0], a[1]);
        codes_to_half<KIND>(__byte_perm(r.v[2][u / 2], r.v[3][u / 2], sel), a[2], a[3]);
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        mma_16<M>(o[u][x], a[0], a[1], a[2], a[3], b[x][0], b[x][1]);
        if constexpr (TWO) mma_16<M>(o[u][x], a[0], a[1], a[2], a[3], rest[x][0], rest[x][1]);
      }
    }
  }

  // The share to shared memory: [8 NT][D] sums, then maxima and sums of weights.
  __device__ __forceinline__ void store(float* so, float* sm, float* sl, int g, int t) {
    const float f = KIND != FV_KV_SAME ? __uint_as_float(uint32_t(min(unit + 1, 254)) << 23) : 1.f;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = l[x][i];
        y += __shfl_xor_sync(FV_FULL, y, 4);
        y += __shfl_xor_sync(FV_FULL, y, 8);
        y += __shfl_xor_sync(FV_FULL, y, 16);
        const int col = 8 * x + 2 * t + i;
        if (g == 0) sm[col] = m[x][i], sl[col] = y;
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
          so[col * D + L::value_at(2 * u, g)] = o[u][x][i] * f;
          so[col * D + L::value_at(2 * u + 1, g)] = o[u][x][i + 2] * f;
        }
      }
  }
};

// Of n shares the weights with which they join, the common maximum and the sum.
template <int N>
__device__ __forceinline__ float join(const float* m, const float* l, float* w, float& total) {
  float most = m[0];
#pragma unroll
  for (int i = 1; i < N; ++i) most = fmaxf(most, m[i]);
  const float from = most == -INFINITY ? 0.f : most;
  total = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = exp2_of(m[i] - from);
    total = __fmaf_rn(w[i], l[i], total);
  }
  return most;
}

template <class T>
__device__ __forceinline__ T rounded(float x) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <class T, int KIND, int D, int NT>
__global__ void __launch_bounds__(32 * KV_TOKEN_WARPS) kv_token_kernel(KvAttend a, KvBatch m, int splits, int tiles) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT;
  float* s_o = reinterpret_cast<float*>(dyn_smem());  // [W][COLS][D]
  float* s_m = s_o + W * COLS * D;                    // [W + 1][COLS], the last for the CTA
  float* s_l = s_m + (W + 1) * COLS;
  int2* s_list = reinterpret_cast<int2*>(s_l + (W + 1) * COLS);  // (block, page) of the row's list
  __shared__ int s_n;
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int row = blockIdx.x / splits, rank = blockIdx.x % splits;
  const int head = blockIdx.y / tiles, first = (blockIdx.y % tiles) * COLS;
  const int b = m.cu ? kv_find(m, row, 1, 0) : row;
  if (row < m.cu_at(b) || row >= m.cu_at(b + 1)) return;  // the same for a whole cluster
  const int pos = __ldg(m.lens + b) - max(m.cu_at(b + 1), row + 1) + row;
  const int last = pos < 0 ? -1 : pos >> m.page_shift;
  int n = min(last + 1, m.table_width);
  Share<T, KIND, D, NT> share;
  share.begin(a, row, head, first, g, t);
  if (a.blocks) {
    if (warp == 0) {  // entries that are blocks the row can see, each above all before it
      const int32_t* list = a.blocks + (size_t(row) * a.heads + head) * a.k;
      int most = -1, count = 0;
      for (int i0 = 0; i0 < a.k; i0 += 32) {
        const int e = i0 + lane < a.k ? __ldg(list + i0 + lane) : -1;
        const bool in = e >= 0 && e < n;
        int up = in ? e : -1;  // largest up to this lane
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(FV_FULL, up, o);
          if (lane >= o) up = max(up, y);
        }
        const int before = __shfl_up_sync(FV_FULL, up, 1);
        const int page = in && e > max(most, lane ? before : -1) ? m.page(b, e) : -1;
        const unsigned has = __ballot_sync(FV_FULL, page >= 0);
        if (page >= 0) s_list[count + __popc(has & ((1u << lane) - 1u))] = make_int2(e, page);
        count += __popc(has);
        most = max(most, __shfl_sync(FV_FULL, up, 31));
      }
      if (lane == 0) s_n = count;
    }
    __syncthreads();
    n = s_n;
  }
  const int per_shift = m.page_shift - 4, chunks = n << per_shift, step = splits * W;
  auto load = [&](Rows<KIND, D>& r, int c) {
    r.visible = 0;
    if (c >= chunks) return;
    const int i = c >> per_shift, slot = (c & ((1 << per_shift) - 1)) << 4;
    const int2 at = a.blocks ? s_list[i] : make_int2(i, m.page(b, i));
    if (at.y >= 0) r.load(a, at.y, head, m.page_shift, slot, pos - ((at.x << m.page_shift) + slot) + 1, g, t);
  };
  Rows<KIND, D> x, y;  // while the rows of one are worked on, those of the other are on their way
  load(x, rank * W + warp);
  for (int c = rank * W + warp; c < chunks; c += 2 * step) {
    load(y, c + step);
    share.take(x, g);
    load(x, c + 2 * step);
    share.take(y, g);
  }
  share.store(s_o + warp * COLS * D, s_m + warp * COLS, s_l + warp * COLS, g, t);
  __syncthreads();
  // the warps' shares to one, in the place of the first
  for (int col = warp; col < COLS; col += W) {
    float mm[W], ll[W], w[W], total;
#pragma unroll
    for (int i = 0; i < W; ++i) mm[i] = s_m[i * COLS + col], ll[i] = s_l[i * COLS + col];
    const float most = join<W>(mm, ll, w, total);
    for (int d = lane; d < D; d += 32) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) sum = __fmaf_rn(w[i], s_o[(i * COLS + col) * D + d], sum);
      s_o[col * D + d] = sum;
    }
    if (lane == 0) s_m[W * COLS + col] = most, s_l[W * COLS + col] = total;
  }
  const float* const s_most = s_m + W * COLS;
  const float* const s_total = s_l + W * COLS;
  cg::cluster_group cluster = cg::this_cluster();
  if (splits > 1) cluster.sync();
  else __syncthreads();
  for (int col = warp + rank * W; col < COLS; col += W * splits) {
    const int h = first + col;
    if (h >= a.group) break;
    float mine = -INFINITY, sum_l = 0.f;  // lane i has those of CTA i
    if (lane < splits) {
      const int at = splits > 1 ? lane : 0;
      mine = splits > 1 ? *cluster.map_shared_rank(s_most + col, at) : s_most[col];
      sum_l = splits > 1 ? *cluster.map_shared_rank(s_total + col, at) : s_total[col];
    }
    float most = mine;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(FV_FULL, most, o));
    most = __shfl_sync(FV_FULL, most, 0);
    const float w = exp2_of(mine - (most == -INFINITY ? 0.f : most));
    float total = lane < splits ? w * sum_l : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) total += __shfl_xor_sync(FV_FULL, total, o);
    total = __shfl_sync(FV_FULL, total, 0);
    const size_t query = size_t(row) * a.heads * a.group + size_t(head) * a.group + h;
    const float down = total == 0.f ? 0.f : 1.f / total;
    for (int d = lane; d < D; d += 32) {
      float sum = 0.f;
      for (int i = 0; i < splits; ++i) {
        const float* from = splits > 1 ? cluster.map_shared_rank(s_o + col * D + d, i) : s_o + col * D + d;
        sum = __fmaf_rn(__shfl_sync(FV_FULL, w, i), *from, sum);
      }
      reinterpret_cast<T*>(a.out)[query * D + d] = rounded<T>(total == 0.f ? 0.f : sum * down);
    }
    if (lane == 0 && a.lse)
      a.lse[query] = total == 0.f ? -INFINITY : (most - Share<T, KIND, D, NT>::ONE + log2f(total)) * 0.693147180559945309f;
  }
  if (splits > 1) cluster.sync();  // nobody leaves while its shares are read
}

template <class T, int KIND, int D, int NT>
int token_launch(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT;
  const int tiles = (a.group + COLS - 1) / COLS;
  const size_t tasks = b->rows * size_t(kv->heads) * tiles, chunks = (a.blocks ? size_t(a.k) : b->table_width) * (kv->page_size / 16);
  // CTAs to a row: until the GPU has two for every SM, as long as each warp has two pieces of 16 rows to work on
  int splits = 1;
  while (splits < 8 && tasks * splits < 2 * 148 && chunks >= size_t(4 * W) * splits) splits *= 2;
  if (size_t(kv->heads) * tiles > 65535 || b->rows > size_t(INT_MAX) / 8)
    return fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: more than 65535 tiles of query heads, or rows beyond 2^28");
  const size_t smem = 4 * (size_t(W) * COLS * D + 2 * (W + 1) * COLS) + (a.blocks ? size_t(a.k) * 8 : 0);
  FV_TRY((kv_allow_smem<kv_token_kernel<T, KIND, D, NT>>(kv->device, smem)));
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {unsigned(splits), 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(b->rows * splits), unsigned(kv->heads * tiles));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FV_CUDA(cudaLaunchKernelEx(&cfg, kv_token_kernel<T, KIND, D, NT>, a, kv_batch(kv, b), splits, tiles));
  return FV_OK;
}

template <class T, int KIND, int D>
int token_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a) {
  return a.group <= 8 ? token_launch<T, KIND, D, 1>(kv, s, b, a) : token_launch<T, KIND, D, 2>(kv, s, b, a);
}

}  // namespace

int kv_token_attend(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a) {
  FV_KV_DISPATCH(kv, token_of, kv, s, b, a);
}

}  // namespace fv

extern "C" int fv_kv_attend_dev(const fv_kv* kv, void* stream, const fv_kv_batch* batch, const void* q, size_t q_row, size_t q_head,
                                size_t group, const int32_t* blocks, size_t k, float scale, void* out, float* lse) {
  FV_TRY(fv::kv_check(kv, batch, "fv_kv_attend_dev"));
  if (group == 0 || group > 128) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: group is 1 to 128 query heads to a key head");
  if (blocks && (k == 0 || k > FV_KV_MAX_BLOCKS)) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: k is 1 to 4096 blocks");
  if (!(scale - scale == 0.f)) return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: scale is not finite");
  if (batch->rows == 0 || batch->nseq == 0) return FV_OK;
  if (!q || !out) return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: NULL queries or result");
  if (!fv::kv_aligned(q, 16) || ((q_row | q_head) & 7) || !fv::kv_aligned(out, 16) || !fv::kv_aligned(blocks, 4) || !fv::kv_aligned(lse, 4))
    return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: queries and result begin on 16 bytes, strides are multiples of 8 elements, blocks and lse begin on 4 bytes");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  const fv::KvAttend a{static_cast<const unsigned char*>(q), 2 * q_row, 2 * q_head, int(kv->heads), int(group), blocks, int(blocks ? k : 0),
                       scale * 1.44269504088896341f, static_cast<const unsigned char*>(kv->k), static_cast<const unsigned char*>(kv->v),
                       kv->k_scale, kv->v_scale, static_cast<unsigned char*>(out), lse};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fv::kv_token_attend(kv, s, batch, a);
}
