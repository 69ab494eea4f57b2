// Attention of single rows (tokens) over blocks of a key/value cache, and the entry point of both kinds of attention.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale q . k_j - max),  lse = log of the sum
//
// One row has as many queries to a key head as its group has heads, so a key is read for a few products only: the bytes of the
// blocks bound it.  A warp takes 16 rows of a block at a time, with a running maximum and sum of its own, through stages in shared
// memory that no other warp waits for.  Many rows, and short lists, get a CTA for each key head; the work of few is cut into equal
// parts for all warps that the GPU holds, and joined by a second kernel.
//
// The products are S^T = K Q^T and O^T = V^T P^T, so that 8 queries fill a tile that would have 16 the other way round.  Sums
// over components may go in any order, so lane t of four holds neighbouring components where the product would have it
// hold some of each 16: loads are 16 bytes.  V's rows arrive a lane each and are paired by byte permutations, P^T comes from S^T by a
// transposition in registers.
//
// 64 rows of 64 heads over 48 blocks of int8 (417 MB): 93 us, 4.5 TB/s, 0.69 of the copy rate; 32 whole sequences in bf16 (0.9 GB):
// 162 us, 5.6 TB/s; 12 of 15k rows in e4m3 (271 MB): 57 us, 4.8 TB/s.  A warp's steps from keys to scores to weights depend on one
// another (about 1160 clocks a piece of bf16 when it is alone); in 8 bits the codes' way to fp16 adds to them.  One request's
// 32 blocks take 10.2 us in a graph, most of it dependent loads: the list, the table, the rows, and the shares that are joined.
//
// In 8 bits the codes are exact in fp16; a key's scale multiplies its score, a value's its weight, relative to the largest
// power of two of a scale that the row has seen.  Weights are rounded to 16 bits for the second product: fp16 with 2^14 for 1, so that
// none above 2^-28 loses bits, or two bf16 numbers (a weight and what its rounding left), which is as good; the loads leave the time.
// In 8 bits what is rounded is the weight times its value's relative scale: no bits are lost above 2^-28 of that product, and
// below it up to 2^-38 of the largest scale times the code, so a row whose scale is 2^20 below the largest one seen keeps all
// bits for weights above 2^-8.  bf16 queries become fp16 there, times a power of two that brings the largest component to 2^13: a component
// below 2^-30 of it loses bits, up to 2^-38 of it.  A second number would cost a second product; scores of keys in 8 bits are no better.
#include <climits>

#include "kv.cuh"

namespace fv {

int kv_prompt_attend(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a);  // kv_prompt.cu
bool kv_prompt_fits(const fv_kv_batch* b, size_t group, bool lists, size_t k);

// A CTA works on each task (a row and key head), or the work of all is cut into equal parts for the warps that the GPU holds, whose
// shares are then joined.  Which of them: lengths are on the device, so from the most pieces of 16 rows that a task can have.  Both
// sides, 16 to 1024 tasks of 32 to 768 pieces with caches cold, 8 key heads of 4 queries in dim 128, us by tasks / in parts:
//   whole sequences of 5/16 to 16/16 of the table      lists of blocks: all tasks the same
//   int8, pieces  64         128        384            64         128        384
//   64 tasks      14.5/11.7  23.6/16.1  61.5/26.1      15.2/13.1  24.6/17.7  63.7/33.1
//   248 tasks     20.3/21.5  33.1/30.8  83.6/62.3      21.6/26.1  34.5/39.0  87.1/84.1
//   304 tasks     25.7/25.2  40.4/36.6  99.7/74.7      37.5/34.8  56.4/48.2  143/101
//   512 tasks     34.9/34.3  56.2/51.4  142/114        41.8/44.5  66.2/66.9  178/170
//   1024 tasks    57.1/57.9  92.1/89.2  236/215        70.6/73.7  116/120    346/344
//   bf16
//   64 tasks      15.6/12.7  25.6/17.1  66.4/33.6      16.5/14.5  27.2/20.9  69.1/45.8
//   248 tasks     22.4/25.5  39.7/41.1  106/97.8       28.9/35.4  49.2/56.5  130/139
//   304 tasks     28.8/31.4  48.2/49.7  123/119        49.9/44.9  77.6/67.8  197/169
//   512 tasks     38.9/45.6  69.1/75.4  190/191        53.8/64.8  86.9/105   247/283
// Sequences differ, and a CTA by itself waits for the longest: parts pay from a length on that grows with what is to be joined, and
// sooner in 8 bits, where bytes are not what bounds a task.  So do lists that reach over more than a quarter of the table: sequences that
// are shorter have fewer blocks than k.  Other lists are alike, so tasks go in waves, and parts pay where the places that the
// last wave leaves empty would have taken more pieces than cutting costs, about 32 of a place and one for every 16 tasks; not
// where a wave is full to more than 7/8 (e4m3 loses up to 5% there where int8 gains as much).  In 16 bits with one tile of queries fewer
// CTAs saturate the bytes too: there only what leaves a third of the SMs without one, half of them where rows are 64 long, and a second
// wave full to at most 0.6 in dim 128, where an SM holds two CTAs (of three or four the others cover for those that are gone).
// Over 24 shapes and 4000 such points these lines are 0.5% from the better side on average, within 5% for 96% of them, 21% at worst.
enum { KV_PARTS_TASKS = 1024, KV_PARTS_WARPS = 160 * 16, KV_SMS = 148 };
constexpr int kv_ctas_an_sm(int kind, int dim) { return dim == 64 ? 4 : dim == 96 && kind == FV_KV_SAME ? 3 : 2; }
static bool in_parts(int kind, int dim, int group, bool alike, size_t tasks, size_t pieces) {
  if (tasks == 0 || tasks > KV_PARTS_TASKS) return false;
  if (!alike) return pieces >= (kind != FV_KV_SAME ? 48 + tasks / 16 : 32 + tasks / 2);
  const size_t places = size_t(KV_SMS) * kv_ctas_an_sm(kind, dim), waves = (tasks + places - 1) / places, all = waves * places;
  if ((all - tasks) * pieces < (32 + tasks / 16) * places) return false;
  if (kind != FV_KV_SAME || group > 8) return 8 * tasks <= 7 * all;
  if (waves == 1) return tasks <= size_t(KV_SMS * 2 / 3) * (dim == 64 ? 2 : 1);
  return dim == 128 && 5 * tasks <= 3 * all;
}

namespace {

enum { KV_TOKEN_WARPS = 4 };

// bytes that lie next to one another, N registers of them
template <int N>
__device__ __forceinline__ void load_words(uint32_t* to, const void* from) {
  if constexpr (N == 4) {
    const uint4 x = *static_cast<const uint4*>(from);
    to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *static_cast<const uint2*>(from);
    to[0] = x.x, to[1] = x.y;
  } else {
    to[0] = *static_cast<const uint32_t*>(from);
  }
}

// Pieces of 16 rows of one block on their way through a warp's part of shared memory, and which components a lane takes from
// them.  In 8 bits a warp works on two pieces at a time: on one, it would mostly wait for its own results
// (64 rows of 64 heads over 48 blocks of int8: 98 us with one, 94 with two).
// Keys: step s of 16 components takes four neighbouring ones from lane t of four.  Values: lane g of eight has dim / 8
// components, in pieces of 16, 8 or 4 bytes.  16-byte pieces of a row change places by the row's number, so that the lanes
// that read at the same time read from different banks.
template <int KIND, int D>
struct Stage {
  static constexpr int BYTES = KIND == FV_KV_SAME ? 2 : 1, ROW = D * BYTES;
  static constexpr int KEY_WORDS = KIND != FV_KV_SAME && D == 96 ? 2 : 4;  // of one load
  static constexpr int KEY_LOADS = ROW / 4 / (4 * KEY_WORDS);              // for a row, by each of 4 lanes
  static constexpr int PER_LOAD = 4 * KEY_WORDS / BYTES;                   // components
  static constexpr int VALUE_WORDS = ROW / 32;
  static constexpr int FIRST = KIND == FV_KV_SAME ? 8 : D == 128 ? 16 : 8;  // components of a lane's first piece
  static constexpr int REST = D / 8 - FIRST;                               // and of its second: 0, 4 or 8
  static constexpr int SCALES = KIND == FV_KV_SAME ? 0 : 32 * 4;
  static constexpr int PIECE = 2 * 16 * ROW + SCALES + 16;  // keys, values, scales, how many of the rows are seen
  static constexpr int PIECES = KIND == FV_KV_SAME ? 1 : 2;
  static constexpr int SIZE = PIECES * PIECE;
  static constexpr int LEAST = 4 / PIECES;  // stages worth a share of their own
  static constexpr int DEPTH = 16 * 1024 / SIZE < 3 ? 3 : 16 * 1024 / SIZE > 6 ? 6 : 16 * 1024 / SIZE;

  static __device__ __forceinline__ int key_at(int step, int t) {  // first of the four
    constexpr int steps = PER_LOAD / 4;
    return (step / steps) * (4 * PER_LOAD) + t * PER_LOAD + (step % steps) * 4;
  }
  static __device__ __forceinline__ int value_at(int e, int g) { return e < FIRST ? g * FIRST + e : 8 * FIRST + g * REST + (e - FIRST); }
  // where byte `at` of row r lies
  static __device__ __forceinline__ int key_byte(int r, int at) { return r * ROW + (ROW % 128 == 0 ? at ^ (r & 1) << 6 : at); }
  static __device__ __forceinline__ int value_byte(int r, int at) {
    const int turn = r >> 1 & 3;
    if (ROW % 128 == 0) return r * ROW + (at ^ turn << 5);
    if (ROW == 192) return r * ROW + (at < 128 ? at ^ turn << 5 : at ^ (turn & 1) << 5);
    return r * ROW + at;
  }

  // Starts the copies of 16 rows from `slot` of `page` on, of which `seen` are seen; the others may hold anything: zeros in
  // place of their values.
  static __device__ __forceinline__ void fill(unsigned char* s, const KvAttend& a, int page, int head, int page_shift, int slot, int seen, int lane) {
    if (lane == 0) *reinterpret_cast<int*>(s + 2 * 16 * ROW + SCALES) = min(seen, 16);
    if (seen <= 0) return;
    const size_t at = ((size_t(page) * a.heads + head) << page_shift) + slot;
    const unsigned char *kr = a.kp + at * ROW + lane * 16, *vr = a.vp + at * ROW + lane * 16;
    const uint32_t to = uint32_t(__cvta_generic_to_shared(s));
    // rows that a lane copies at one time are an even number apart: their keys' pieces change places alike
    const uint32_t kt = to + key_byte(lane / (ROW / 16), lane % (ROW / 16) * 16);
    copy_keys<0>(kt, kr);
    if (seen >= 16) copy_values<0, true>(to, vr, lane, seen);
    else copy_values<0, false>(to, vr, lane, seen);
    if constexpr (KIND != FV_KV_SAME) {
      const int r = lane & 15;
      const float* from = (lane < 16 ? a.k_scale : a.v_scale) + at + r;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 2 * 16 * ROW + lane * 4), "l"(from), "r"(r < seen ? 4 : 0));
    }
  }
  template <int I>
  static __device__ __forceinline__ void copy_keys(uint32_t to, const unsigned char* from) {
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%2], 16;" ::"r"(to), "l"(from), "n"(512 * I));
    if constexpr (I + 1 < ROW / 32) copy_keys<I + 1>(to, from);
  }
  template <int I, bool ALL>
  static __device__ __forceinline__ void copy_values(uint32_t to, const unsigned char* from, int lane, int seen) {
    const uint32_t at = to + uint32_t(value_to(lane, I));
    if constexpr (ALL) asm volatile("cp.async.cg.shared.global [%0], [%1+%2], 16;" ::"r"(at), "l"(from), "n"(512 * I));
    else asm volatile("cp.async.cg.shared.global [%0], [%1+%2], 16, %3;" ::"r"(at), "l"(from), "n"(512 * I), "r"((lane + 32 * I) / (ROW / 16) < seen ? 16 : 0));
    if constexpr (I + 1 < ROW / 32) copy_values<I + 1, ALL>(to, from, lane, seen);
  }
  static __device__ __forceinline__ int value_to(int lane, int i) {
    const int u = lane + 32 * i;
    return 16 * ROW + value_byte(u / (ROW / 16), u % (ROW / 16) * 16);
  }
  static __device__ __forceinline__ int seen(const unsigned char* s) { return *reinterpret_cast<const int*>(s + 2 * 16 * ROW + SCALES); }
};

// A warp's share of a row's attention: NT tiles of 8 queries.  A lane's queries are 8 x + 2 t and the next one.
template <class T, int KIND, int D, int NT>
struct Share {
  using M = typename std::conditional<KIND == FV_KV_SAME, T, __half>::type;
  using L = Stage<KIND, D>;
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

  __device__ __forceinline__ void take(const unsigned char* stage, int g, int t) {
    constexpr int P = L::PIECES;
    int visible[P], any = 0;
#pragma unroll
    for (int h = 0; h < P; ++h) visible[h] = L::seen(stage + h * L::PIECE), any = max(any, visible[h]);
    if (any <= 0) return;
    float s[P][NT][4];
#pragma unroll
    for (int h = 0; h < P; ++h) {
      const unsigned char* keys = stage + h * L::PIECE;
      float part[2][NT][4] = {};  // two sums, for a product not to wait for the one before it
#pragma unroll
      for (int c = 0; c < L::KEY_LOADS; ++c) {
        uint32_t k[2][L::KEY_WORDS];
#pragma unroll
        for (int i = 0; i < 2; ++i) load_words<L::KEY_WORDS>(k[i], keys + L::key_byte(g + 8 * i, (c * 4 + t) * (4 * L::KEY_WORDS)));
#pragma unroll
        for (int z = 0; z < L::PER_LOAD / 4; ++z) {
          uint32_t a[4];
          if constexpr (KIND == FV_KV_SAME) {
            a[0] = k[0][2 * z], a[1] = k[1][2 * z], a[2] = k[0][2 * z + 1], a[3] = k[1][2 * z + 1];
          } else {
            codes_to_half<KIND>(k[0][z], a[0], a[2]);
            codes_to_half<KIND>(k[1][z], a[1], a[3]);
          }
          const int st = c * (L::PER_LOAD / 4) + z;
#pragma unroll
          for (int x = 0; x < NT; ++x) mma_16<M>(part[st & 1][x], a[0], a[1], a[2], a[3], q[st][x][0], q[st][x][1]);
        }
      }
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][x][i] = part[0][x][i] + part[1][x][i];
    }
    float vs[P][2], grown = 1.f;
    if constexpr (KIND != FV_KV_SAME) {
      float most = 0.f;  // leaves NaN out: it reaches the sums through its weight
#pragma unroll
      for (int h = 0; h < P; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // of a piece that is not there the scales are anything
          const float* scales = reinterpret_cast<const float*>(stage + h * L::PIECE + 2 * 16 * L::ROW) + g + 8 * i;
          vs[h][i] = visible[h] > 0 ? scales[16] : 0.f;
          const float ks = scales[0];
          most = fmaxf(most, vs[h][i]);
#pragma unroll
          for (int x = 0; x < NT; ++x) s[h][x][2 * i] *= ks, s[h][x][2 * i + 1] *= ks;
        }
      const int e = max(unit, int(__reduce_max_sync(FV_FULL, __float_as_uint(most)) >> 23));
      grown = __uint_as_float(uint32_t(max(127 + unit - e, 0)) << 23);
      unit = e;
      const float down = __uint_as_float(uint32_t(max(253 - e, 1)) << 23);
#pragma unroll
      for (int h = 0; h < P; ++h) vs[h][0] *= down, vs[h][1] *= down;
    }
    bool moved = grown != 1.f;
    float to[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int h = 0; h < P; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][x][i] = g + (i & 2) * 4 < visible[h] ? s[h][x][i] * by[x][i & 1] : -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        to[x][i] = fmaxf(s[0][x][i], s[0][x][i + 2]);
        if constexpr (P > 1) to[x][i] = fmaxf(to[x][i], fmaxf(s[P - 1][x][i], s[P - 1][x][i + 2]));
        moved = moved || to[x][i] > m[x][i];
      }
    }
    if (__any_sync(FV_FULL, moved)) {  // seldom, after the first pieces
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y = fmaxf(m[x][i], to[x][i]);
          y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 4));
          y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 8));
          y = fmaxf(y, __shfl_xor_sync(FV_FULL, y, 16));
          const float by_l = y > m[x][i] ? exp2_of(m[x][i] - y) : 1.f, by_o = by_l * grown;
          m[x][i] = y;
          l[x][i] *= by_l;
#pragma unroll
          for (int u = 0; u < D / 16; ++u) o[u][x][i] *= by_o, o[u][x][i + 2] *= by_o;
        }
    }
    uint32_t b[P][NT][2], rest[P][NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int h = 0; h < P; ++h) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = exp2_of(s[h][x][i] - (m[x][i & 1] == -INFINITY ? 0.f : m[x][i & 1]) + ONE);
          l[x][i & 1] += p[i];
          if constexpr (KIND != FV_KV_SAME) p[i] = p[i] != 0.f ? p[i] * vs[h][i >> 1] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w = Pair<M>::from_float(p[2 * i], p[2 * i + 1]);
          b[h][x][i] = transposed(w);
          if constexpr (TWO) {
            const float2 f = Pair<M>::to_float(w);
            rest[h][x][i] = transposed(Pair<M>::from_float(p[2 * i] - f.x, p[2 * i + 1] - f.y));
          }
        }
      }
#pragma unroll
    for (int h = 0; h < P; ++h) {
      if (P > 1 && visible[h] <= 0) continue;  // its values are anything
      const unsigned char* values = stage + h * L::PIECE + 16 * L::ROW;
      uint32_t v[4][L::VALUE_WORDS];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 2 * t + (i & 1) + (i & 2) * 4;
        constexpr int w = L::FIRST * L::BYTES / 4;
        load_words<w>(v[i], values + L::value_byte(r, g * L::FIRST * L::BYTES));
        if constexpr (L::REST > 0) load_words<L::REST * L::BYTES / 4>(v[i] + w, values + L::value_byte(r, (8 * L::FIRST + g * L::REST) * L::BYTES));
      }
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        uint32_t a[4];
        if constexpr (KIND == FV_KV_SAME) {
          a[0] = __byte_perm(v[0][u], v[1][u], 0x5410), a[1] = __byte_perm(v[0][u], v[1][u], 0x7632);
          a[2] = __byte_perm(v[2][u], v[3][u], 0x5410), a[3] = __byte_perm(v[2][u], v[3][u], 0x7632);
        } else {
          const int sel = u & 1 ? 0x7362 : 0x5140;  // components 2u and 2u + 1 of two rows
          codes_to_half<KIND>(__byte_perm(v[0][u / 2], v[1][u / 2], sel), a[0], a[1]);
          codes_to_half<KIND>(__byte_perm(v[2][u / 2], v[3][u / 2], sel), a[2], a[3]);
        }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          mma_16<M>(o[u][x], a[0], a[1], a[2], a[3], b[h][x][0], b[h][x][1]);
          if constexpr (TWO) mma_16<M>(o[u][x], a[0], a[1], a[2], a[3], rest[h][x][0], rest[h][x][1]);
        }
      }
    }
  }

  // The share as it lies in registers: for every two components u and tile x a float4 of each lane, then the maxima and the sums
  // of weights of the 8 NT queries.  A value's unit is multiplied in.
  static constexpr int FLOATS = 8 * NT * (D + 2);
  __device__ __forceinline__ void store(float* to, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const float f = KIND != FV_KV_SAME ? __uint_as_float(uint32_t(min(unit + 1, 254)) << 23) : 1.f;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
        reinterpret_cast<float4*>(to)[(u * NT + x) * 32 + lane] = make_float4(o[u][x][0] * f, o[u][x][1] * f, o[u][x][2] * f, o[u][x][3] * f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = l[x][i];
        y += __shfl_xor_sync(FV_FULL, y, 4);
        y += __shfl_xor_sync(FV_FULL, y, 8);
        y += __shfl_xor_sync(FV_FULL, y, 16);
        if (g == 0) to[8 * NT * D + 8 * x + 2 * t + i] = m[x][i], to[8 * NT * (D + 1) + 8 * x + 2 * t + i] = y;
      }
    }
  }
};

template <class T>
__device__ __forceinline__ uint32_t rounded2(float x, float y) { return Pair<T>::from_float(x, y); }

// Joins the shares of a CTA's W warps and writes the queries' results in 16 U components of D from `u0` on.  A share: U * NT * 32
// float4, the maxima and sums of weights behind them, FLOATS in all.
template <class T, int KIND, int D, int NT, int W, int U>
__device__ __forceinline__ void finish(const float* s, const KvAttend& a, int row, int head, int first, int u0, int warp, int lane) {
  using H = Share<T, KIND, D, NT>;
  constexpr int SUMS = 128 * U * NT, FLOATS = SUMS + 16 * NT;
  const int g = lane >> 2, t = lane & 3;
  float w[W][NT][2], down[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = 8 * x + 2 * t + i, h = first + col;
      float m[W], most = -INFINITY, total = 0.f;
#pragma unroll
      for (int z = 0; z < W; ++z) m[z] = s[z * FLOATS + SUMS + col], most = fmaxf(most, m[z]);
#pragma unroll
      for (int z = 0; z < W; ++z) {
        w[z][x][i] = exp2_of(m[z] - (most == -INFINITY ? 0.f : most));
        total = __fmaf_rn(w[z][x][i], s[z * FLOATS + SUMS + 8 * NT + col], total);
      }
      down[x][i] = total == 0.f ? 0.f : 1.f / total;
      if (a.lse && warp == 0 && u0 == 0 && g == 0 && h < a.group)
        a.lse[(size_t(row) * a.heads + head) * a.group + h] = total == 0.f ? -INFINITY : (most - H::ONE + log2f(total)) * 0.693147180559945309f;
    }
#pragma unroll
  for (int j = 0; j < U * NT; ++j) {
    if (j % W != warp) continue;
    const int u = u0 + j / NT, x = j % NT, h = first + 8 * x + 2 * t;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int z = 0; z < W; ++z) {
      const float4 y = reinterpret_cast<const float4*>(s + z * FLOATS)[j * 32 + lane];
      sum.x = __fmaf_rn(w[z][x][0], y.x, sum.x), sum.y = __fmaf_rn(w[z][x][1], y.y, sum.y);
      sum.z = __fmaf_rn(w[z][x][0], y.z, sum.z), sum.w = __fmaf_rn(w[z][x][1], y.w, sum.w);
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (((size_t(row) * a.heads + head) * a.group + h) * D + H::L::value_at(2 * u, g)) * 2);
    if (h < a.group) out[0] = down[x][0] == 0.f ? 0u : rounded2<T>(sum.x * down[x][0], sum.z * down[x][0]);
    if (h + 1 < a.group) out[D / 2] = down[x][1] == 0.f ? 0u : rounded2<T>(sum.y * down[x][1], sum.w * down[x][1]);
  }
}

// Where a row of the call stands.
struct Place {
  int b, pos;  // b < 0: in no sequence
};
__device__ __forceinline__ Place place_of(const KvBatch& m, int row) {  // whole warps call it
  const int b = m.cu ? kv_find(m, row, 1, 0) : row;
  if (row < m.cu_at(b) || row >= m.cu_at(b + 1)) return {-1, -1};
  return {b, m.len(b) - max(m.cu_at(b + 1), row + 1) + row};
}

// The pieces of one row and key head, 16 rows each, and where they lie: lane i has block and page of the i-th of 32 of the row's
// blocks, from `base` on.
struct Pieces {
  int b, pos, head, count, base, most, block, page;
  const int32_t* list;

  // of `row` and key head `head`
  __device__ __forceinline__ void begin(const KvAttend& a, const KvBatch& m, int row, int head_of) {
    const Place p = place_of(m, row);
    b = p.b, pos = p.pos, head = head_of;
    list = a.blocks ? a.blocks + (size_t(row) * a.heads + head_of) * a.k : nullptr;
    base = -32, most = -1;
  }
  __device__ __forceinline__ void look(const KvAttend& a, const KvBatch& m, int entry) {
    const int n = pos < 0 ? 0 : min((pos >> m.page_shift) + 1, m.table_width), lane = lane_id();
    const int to = entry & ~31;
    if (list) {  // entries that are blocks the row can see, each above all before it
      for (int from = base + 32; ; from += 32) {
        const int e = from + lane < a.k ? __ldg(list + from + lane) : -1;
        const bool in = e >= 0 && e < n;
        int up = in ? e : -1;  // largest up to this lane
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(FV_FULL, up, o);
          if (lane >= o) up = max(up, y);
        }
        const int before = __shfl_up_sync(FV_FULL, up, 1);
        block = e;
        page = from == to && in && e > max(most, lane ? before : -1) ? m.page(b, e) : -1;
        most = max(most, __shfl_sync(FV_FULL, up, 31));
        if (from == to) break;
      }
    } else {
      block = to + lane;
      page = block < n ? m.page(b, block) : -1;
    }
    base = to;
  }
  template <class S>
  __device__ __forceinline__ void fill(unsigned char* stage, const KvAttend& a, const KvBatch& m, int c) {
    const int per = m.page_shift - 4, i = c >> per, slot = (c & ((1 << per) - 1)) << 4;
    if (i >= base + 32) look(a, m, i);
    const int at = __shfl_sync(FV_FULL, block, i & 31), p = __shfl_sync(FV_FULL, page, i & 31);
    S::fill(stage, a, p, head, m.page_shift, slot, p >= 0 ? pos - ((at << m.page_shift) + slot) + 1 : 0, lane_id());
  }
};

// Pieces of a row: those of its list, or all up to its own position.
__device__ __forceinline__ int pieces_of(const KvAttend& a, const KvBatch& m, int pos) {
  if (pos < 0) return 0;
  return a.blocks ? a.k << (m.page_shift - 4) : min((pos >> 4) + 1, m.table_width << (m.page_shift - 4));
}

// A CTA for one row and key head; its warps take turns at the pieces.
template <class T, int KIND, int D, int NT>
__global__ void __launch_bounds__(32 * KV_TOKEN_WARPS) kv_token_kernel(KvAttend a, KvBatch m, int tiles) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT;
  using S = Stage<KIND, D>;
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  unsigned char* ring = dyn_smem() + warp * (S::DEPTH * S::SIZE);  // a warp's stages; later the shares
  const int row = blockIdx.x, head = blockIdx.y / tiles, first = (blockIdx.y % tiles) * COLS;
  Pieces pieces;
  pieces.begin(a, m, row, head);
  if (pieces.b < 0) return;
  const int n = pieces_of(a, m, pieces.pos), step = W * S::PIECES;
  int next = warp * S::PIECES, at = 0;
  auto fill = [&](int to) {
    if (next < n) {
#pragma unroll
      for (int h = 0; h < S::PIECES; ++h) pieces.fill<S>(ring + to * S::SIZE + h * S::PIECE, a, m, next + h);
    }
    next += step;
    asm volatile("cp.async.commit_group;");
  };
#pragma unroll 1
  for (int i = 0; i < S::DEPTH; ++i) fill(i);
  Share<T, KIND, D, NT> share;
  share.begin(a, row, head, first, g, t);
#pragma unroll 1
  for (int c = warp * S::PIECES; c < n; c += step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::DEPTH - 1));
    __syncwarp();
    share.take(ring + at * S::SIZE, g, t);
    __syncwarp();
    fill(at);
    at = at + 1 == S::DEPTH ? 0 : at + 1;
  }
  asm volatile("cp.async.wait_all;");
  __syncthreads();  // the stages become the shares' place
  float* s = reinterpret_cast<float*>(dyn_smem());
  share.store(s + warp * Share<T, KIND, D, NT>::FLOATS, lane);
  __syncthreads();
  finish<T, KIND, D, NT, W, D / 16>(s, a, row, head, first, 0, warp, lane);
}

// Or: all the pieces of all rows and heads (tasks), in units of a stage, are cut into equal parts, one for each warp that
// the GPU holds, whatever the lengths.  A warp leaves its share of each task that it meets in `part`: that of warp w of task t at
// number w + t, since along the units one of the two grows.  A second kernel joins them.
struct Parts {
  int rows, tasks_a_row, least, warps;  // least: units a warp takes at least
  float* part;
};


// Units before each row to s[0 .. rows], by a CTA of 128 threads.
template <class S>
__device__ __forceinline__ void units_before(const KvAttend& a, const KvBatch& m, int rows, int* s, int* s_warp) {
  const int warp = threadIdx.x >> 5, lane = lane_id();
  int sum = 0;
  for (int r0 = 0; r0 < rows; r0 += 128) {
    const int r = r0 + threadIdx.x;
    int pos = -1;
    if (m.cu) {  // kv_find works for one row of a warp: a thread looks for its own by halves
      int lo = 0, n = m.nseq;
      while (n > 1) {
        const int h = n / 2;
        if (m.cu_at(lo + h) <= r) lo += h, n -= h;
        else n = h;
      }
      if (r < rows && r >= m.cu_at(lo) && r < m.cu_at(lo + 1)) pos = m.len(lo) - max(m.cu_at(lo + 1), r + 1) + r;
    } else if (r < rows) {
      pos = m.len(r) - 1;
    }
    int x = (pieces_of(a, m, pos) + S::PIECES - 1) / S::PIECES;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(FV_FULL, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int before = sum;
    for (int w = 0; w < 4; ++w) {
      if (w < warp) before += s_warp[w];
      sum += s_warp[w];
    }
    if (r < rows) s[r + 1] = before + x;
    __syncthreads();
  }
  if (threadIdx.x == 0) s[0] = 0;
  __syncthreads();
}

// Units that a warp takes: its part of all, but no fewer than are worth a share of its own, and so many that the sequences'
// lengths on average leave no more than 256 shares of a task to join.
__device__ __forceinline__ int units_a_warp(const Parts& p, int all) {
  const long long total = (long long)(all) * p.tasks_a_row;
  return max(max(p.least, all / (256 * p.rows)), int((total + p.warps - 1) / p.warps));
}

template <class T, int KIND, int D, int NT>
__global__ void __launch_bounds__(32 * KV_TOKEN_WARPS) kv_parts_kernel(KvAttend a, KvBatch m, Parts p, int tiles, int before_at) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT;
  using S = Stage<KIND, D>;
  using H = Share<T, KIND, D, NT>;
  __shared__ int s_warp[W];
  int* before = reinterpret_cast<int*>(dyn_smem() + before_at);
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  unsigned char* ring = dyn_smem() + warp * (S::DEPTH * S::SIZE);
  asm volatile("griddepcontrol.launch_dependents;");  // the kernel that joins may come and wait
  units_before<S>(a, m, p.rows, before, s_warp);
  const long long total = (long long)(before[p.rows]) * p.tasks_a_row;
  const int mine = units_a_warp(p, before[p.rows]), w = blockIdx.x * W + warp;
  const long long begin = (long long)(w) * mine;
  if (begin >= total) return;
  const int n = int(min((long long)(mine), total - begin));
  // a place among the units
  struct Cursor {
    int row, task, unit, units;  // task and unit of the row's
    __device__ __forceinline__ bool step(const int* before, int tasks) {  // whether another task begins
      if (++unit < units) return false;
      unit = 0;
      if (++task == tasks) {
        task = 0;
        do ++row;
        while (before[row + 1] == before[row]);
        units = before[row + 1] - before[row];
      }
      return true;
    }
  };
  Cursor in;
  {
    int lo = 0, c = p.rows;
    while (c > 1) {  // the last row that begins at or before the warp's first unit
      const int h = c / 2;
      if ((long long)(before[lo + h]) * p.tasks_a_row <= begin) lo += h, c -= h;
      else c = h;
    }
    const int rest = int(begin - (long long)(before[lo]) * p.tasks_a_row), units = before[lo + 1] - before[lo];
    in = {lo, rest / units, rest % units, units};
  }
  Cursor out = in;
  Pieces pieces;
  pieces.begin(a, m, in.row, in.task / tiles);
  int filled = 0;
  auto fill = [&](int to) {
    if (filled < n) {
#pragma unroll
      for (int h = 0; h < S::PIECES; ++h) pieces.fill<S>(ring + to * S::SIZE + h * S::PIECE, a, m, in.unit * S::PIECES + h);
      if (++filled < n && in.step(before, p.tasks_a_row)) pieces.begin(a, m, in.row, in.task / tiles);
    }
    asm volatile("cp.async.commit_group;");
  };
#pragma unroll 1
  for (int i = 0; i < S::DEPTH; ++i) fill(i);
  H share;
  share.begin(a, out.row, out.task / tiles, out.task % tiles * COLS, g, t);
  int at = 0;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::DEPTH - 1));
    __syncwarp();
    share.take(ring + at * S::SIZE, g, t);
    __syncwarp();
    fill(at);
    at = at + 1 == S::DEPTH ? 0 : at + 1;
    const size_t number = size_t(w) + size_t(out.row) * p.tasks_a_row + out.task;
    const bool last = i + 1 == n, other = !last && out.step(before, p.tasks_a_row);
    if (last || other) share.store(p.part + number * H::FLOATS, lane);
    if (other) share.begin(a, out.row, out.task / tiles, out.task % tiles * COLS, g, t);
  }
}

// A CTA joins 32 of the components of a task; a warp takes four of its shares at a time.
template <class T, int KIND, int D, int NT>
__global__ void __launch_bounds__(32 * KV_TOKEN_WARPS) kv_join_kernel(KvAttend a, KvBatch m, Parts p, int tiles) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT, U = 2, FLOATS = 128 * U * NT + 16 * NT, AT_ONCE = 4;
  using H = Share<T, KIND, D, NT>;
  __shared__ int s_warp[W];
  __shared__ __align__(16) float s[W * FLOATS];
  int* before = reinterpret_cast<int*>(dyn_smem());
  const int warp = threadIdx.x >> 5, lane = lane_id(), t = lane & 3;
  const int row = blockIdx.x, task = blockIdx.y, u0 = blockIdx.z * U;
  units_before<Stage<KIND, D>>(a, m, p.rows, before, s_warp);
  const bool none = place_of(m, row).b < 0;
  const int mine = units_a_warp(p, before[p.rows]), units = before[row + 1] - before[row];
  const long long begin = (long long)(before[row]) * p.tasks_a_row + (long long)(task) * units;
  const int w0 = int(begin / mine), w1 = units ? int((begin + units - 1) / mine) : w0 - 1;  // the warps that met the task
  const float* const part = p.part + (size_t(row) * p.tasks_a_row + task) * H::FLOATS;
  // For the shares.  Every CTA waits, whether it has some or not: what the stream holds next starts when these are done, and must
  // not start before the kernel that leaves the shares is.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (none) return;
  float4 o[U][NT];
  float most[NT][2], total[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    most[x][0] = most[x][1] = -INFINITY, total[x][0] = total[x][1] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) o[u][x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int w = w0 + warp; w <= w1; w += W * AT_ONCE) {
    float4 y[AT_ONCE][U][NT];
    float ms[AT_ONCE][NT][2], ls[AT_ONCE][NT][2];
#pragma unroll
    for (int z = 0; z < AT_ONCE; ++z) {
      const bool on = w + z * W <= w1;
      const float* from = part + size_t(on ? w + z * W : w) * H::FLOATS;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int u = 0; u < U; ++u) y[z][u][x] = reinterpret_cast<const float4*>(from)[((u0 + u) * NT + x) * 32 + lane];
        const float2 m2 = *reinterpret_cast<const float2*>(from + COLS * D + 8 * x + 2 * t), l2 = *reinterpret_cast<const float2*>(from + COLS * (D + 1) + 8 * x + 2 * t);
        ms[z][x][0] = on ? m2.x : -INFINITY, ms[z][x][1] = on ? m2.y : -INFINITY;
        ls[z][x][0] = on ? l2.x : 0.f, ls[z][x][1] = on ? l2.y : 0.f;
      }
    }
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float was[2], is[AT_ONCE][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = most[x][i];
#pragma unroll
        for (int z = 0; z < AT_ONCE; ++z) top = fmaxf(top, ms[z][x][i]);
        const float of = top == -INFINITY ? 0.f : top;
        was[i] = exp2_of(most[x][i] - of);
        most[x][i] = top;
        total[x][i] *= was[i];
#pragma unroll
        for (int z = 0; z < AT_ONCE; ++z) is[z][i] = exp2_of(ms[z][x][i] - of), total[x][i] = __fmaf_rn(ls[z][x][i], is[z][i], total[x][i]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float4& sum = o[u][x];
        sum.x *= was[0], sum.y *= was[1], sum.z *= was[0], sum.w *= was[1];
#pragma unroll
        for (int z = 0; z < AT_ONCE; ++z) {
          if (w + z * W > w1) continue;  // a share read twice has the weight 0, and may not be finite
          sum.x = __fmaf_rn(y[z][u][x].x, is[z][0], sum.x), sum.y = __fmaf_rn(y[z][u][x].y, is[z][1], sum.y);
          sum.z = __fmaf_rn(y[z][u][x].z, is[z][0], sum.z), sum.w = __fmaf_rn(y[z][u][x].w, is[z][1], sum.w);
        }
      }
    }
  }
  float* to = s + warp * FLOATS;
#pragma unroll
  for (int x = 0; x < NT; ++x) {
#pragma unroll
    for (int u = 0; u < U; ++u) reinterpret_cast<float4*>(to)[(u * NT + x) * 32 + lane] = o[u][x];
    if (lane < 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) to[128 * U * NT + 8 * x + 2 * t + i] = most[x][i], to[128 * U * NT + 8 * NT + 8 * x + 2 * t + i] = total[x][i];
    }
  }
  __syncthreads();
  finish<T, KIND, D, NT, W, U>(s, a, row, task / tiles, task % tiles * COLS, u0, warp, lane);
}

// Warps that the GPU holds of kv_parts_kernel, looked up once for each device.
template <class T, int KIND, int D, int NT>
int parts_warps(int device, size_t smem, int* warps) {
  static std::atomic<int> known[64];
  int n = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    int sms = 0, ctas = 0;
    FV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    FV_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kv_parts_kernel<T, KIND, D, NT>, 32 * KV_TOKEN_WARPS, smem));
    n = sms * (ctas > 0 ? ctas : 1) * KV_TOKEN_WARPS;
    if (device < 64) known[device].store(n, std::memory_order_relaxed);
  }
  *warps = n;
  return FV_OK;
}

template <class T, int KIND, int D, int NT>
int token_launch(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a, void* work, size_t work_bytes) {
  constexpr int W = KV_TOKEN_WARPS, COLS = 8 * NT;
  using S = Stage<KIND, D>;
  using H = Share<T, KIND, D, NT>;
  const int tiles = (a.group + COLS - 1) / COLS;
  const size_t tasks_a_row = size_t(kv->heads) * tiles, tasks = b->rows * tasks_a_row;
  if (tasks_a_row > 65535) return fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: more than 65535 tiles of query heads");
  const size_t ring = size_t(W) * S::DEPTH * S::SIZE, shares = size_t(W) * H::FLOATS * 4;
  const KvBatch m = kv_batch(kv, b);
  const size_t pieces = (a.blocks ? size_t(a.k) : b->table_width) * (kv->page_size / 16);  // of a task, at most
  const bool alike = a.blocks && size_t(a.k) * 4 <= b->table_width;
  static_assert(228 * 1024 / (W * S::DEPTH * S::SIZE + 1024) == kv_ctas_an_sm(KIND, D), "the rule counts the CTAs that an SM holds");
  if (work && in_parts(KIND, D, a.group, alike, tasks, pieces) && pieces * tasks <= size_t(1) << 30) {
    const size_t smem = ring + 4 * (b->rows + 1), most = ring + 4 * (KV_PARTS_TASKS + 1);
    Parts p{int(b->rows), int(tasks_a_row), S::LEAST, 0, static_cast<float*>(work)};
    FV_TRY((kv_allow_smem<kv_parts_kernel<T, KIND, D, NT>>(kv->device, most)));
    FV_TRY((parts_warps<T, KIND, D, NT>(kv->device, ring + 1024, &p.warps)));
    const size_t room = work_bytes / (4 * size_t(H::FLOATS));  // shares that `work` holds
    if (room <= tasks + W) return fail(FV_ERR_ARG, "fv_kv_attend_dev: work is smaller than fv_kv_attend_work says");
    if (size_t(p.warps) > room - tasks) p.warps = int((room - tasks) / W * W);
    kv_parts_kernel<T, KIND, D, NT><<<unsigned(p.warps / W), 32 * W, smem, s>>>(a, m, p, tiles, int(ring));
    FV_CUDA(cudaGetLastError());
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // it starts while the last parts are worked on, and waits for them
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(b->rows), unsigned(tasks_a_row), D / 32);
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = 4 * (b->rows + 1);
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FV_CUDA(cudaLaunchKernelEx(&cfg, kv_join_kernel<T, KIND, D, NT>, a, m, p, tiles));
    return FV_OK;
  }
  const size_t smem = ring > shares ? ring : shares;
  FV_TRY((kv_allow_smem<kv_token_kernel<T, KIND, D, NT>>(kv->device, smem)));
  kv_token_kernel<T, KIND, D, NT><<<dim3(unsigned(b->rows), unsigned(tasks_a_row)), 32 * W, smem, s>>>(a, m, tiles);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

template <class T, int KIND, int D>
int token_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a, void* work, size_t work_bytes) {
  return a.group <= 8 ? token_launch<T, KIND, D, 1>(kv, s, b, a, work, work_bytes) : token_launch<T, KIND, D, 2>(kv, s, b, a, work, work_bytes);
}

}  // namespace

// Several rows of a sequence on average, and room for the union of their lists.
static bool is_prompt(const fv_kv_batch* b, size_t group, bool lists, size_t k) {
  return b->rows > 4 * b->nseq && kv_prompt_fits(b, group, lists, k);
}

int kv_token_attend(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvAttend& a, void* work, size_t work_bytes) {
  FV_KV_DISPATCH(kv, token_of, kv, s, b, a, work, work_bytes);
}

}  // namespace fv

extern "C" size_t fv_kv_attend_work(const fv_kv* kv, const fv_kv_batch* batch, size_t group) {
  if (!kv || !batch || group == 0 || group > 128 || batch->rows > fv::KV_PARTS_TASKS) return 0;
  if (fv::is_prompt(batch, group, false, 0)) return 0;  // with lists too: a shorter union fits where the whole table does
  const size_t cols = group <= 8 ? 8 : 16, tasks = batch->rows * kv->heads * ((group + cols - 1) / cols), pieces = batch->table_width * (kv->page_size / 16);
  const bool parts = fv::in_parts(kv->kind, int(kv->dim), int(group), false, tasks, pieces) || fv::in_parts(kv->kind, int(kv->dim), int(group), true, tasks, pieces);
  return parts ? (tasks + fv::KV_PARTS_WARPS) * cols * (kv->dim + 2) * 4 : 0;
}

extern "C" int fv_kv_attend_dev(const fv_kv* kv, void* stream, const fv_kv_batch* batch, const void* q, size_t q_row, size_t q_head,
                                size_t group, const int32_t* blocks, size_t k, float scale, void* out, float* lse, void* work, size_t work_bytes) {
  FV_TRY(fv::kv_check(kv, batch, "fv_kv_attend_dev"));
  if (group == 0 || group > 128) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: group is 1 to 128 query heads to a key head");
  if (blocks && (k == 0 || k > FV_KV_MAX_BLOCKS)) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_attend_dev: k is 1 to 4096 blocks");
  if (!(scale - scale == 0.f)) return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: scale is not finite");
  if (batch->rows == 0 || batch->nseq == 0) return FV_OK;
  if (!q || !out) return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: NULL queries or result");
  if (!fv::kv_aligned(q, 16) || ((q_row | q_head) & 7) || !fv::kv_aligned(out, 16) || !fv::kv_aligned(blocks, 4) || !fv::kv_aligned(lse, 4) || !fv::kv_aligned(work, 16))
    return fv::fail(FV_ERR_ARG, "fv_kv_attend_dev: queries, result and work begin on 16 bytes, strides are multiples of 8 elements, blocks and lse begin on 4 bytes");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  const fv::KvAttend a{static_cast<const unsigned char*>(q), 2 * q_row, 2 * q_head, int(kv->heads), int(group), blocks, int(blocks ? k : 0),
                       scale * 1.44269504088896341f, static_cast<const unsigned char*>(kv->k), static_cast<const unsigned char*>(kv->v),
                       kv->k_scale, kv->v_scale, static_cast<unsigned char*>(out), lse};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv->pages && fv::is_prompt(batch, group, blocks != nullptr, k)) return fv::kv_prompt_attend(kv, s, batch, a);
  return fv::kv_token_attend(kv, s, batch, a, work, work_bytes);
}
