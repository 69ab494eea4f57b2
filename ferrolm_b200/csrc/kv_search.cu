// The blocks of a key/value cache that promise a query the largest inner products.
//
// With lo <= key <= hi componentwise, q . key <= max(q,0) . hi + min(q,0) . lo for every key of a block, and the sum of that
// over the query heads g of a key head is p . hi + n . lo with p = sum_g max(q_g,0), n = sum_g min(q_g,0): one product of
// 2 dim components, however many heads share the keys.  All of it is done in whole numbers: queries to -127..127 with one
// scale for the group, their sums again, the bounds as add left them; a product of 2 * 128 such terms is exact in 32 bits and
// in a float.  A block's score is that number times the scale of its bounds, rounded once, so the choice does not depend on
// the order of any sum: the same blocks come out whichever way the work is cut.
//
//   codes of q      whole(127 q / max |q|),                  max over the group
//   p, n            sums of the positive and negative codes, then whole(127 p / max(|p|, |n|))
//   score           float(p . hi + n . lo) * bound_scale
//   result          the first `first` blocks, the last `recent` up to the query's own, then the largest scores (the lower
//                   block of equals) up to k in all, in ascending order, -1 behind the last; of more than k forced ones the lowest
//
// The bounds are 2 dim + 4 bytes for a block, so a token's search is a few dependent loads long (the table, the bounds, then the
// threshold): 8.2 us in a graph for one request over 2032 blocks of 8 heads, 4.2 MB, in clusters of 8, and 11.3 us for 48 requests; a
// call's steps on the host make that 10.5 (28.7 without clusters) and 12.3.  A prompt's search is bound by what each row does
// besides its products: 89 us for 3.2k rows of 8 heads over up to 512 blocks, about 2400 instructions a warp for a row and head.
//
// The score is no bound itself: queries, their sums and bounds are rounded to nearest, with one scale for a group's queries, so
// that a head below 1/254 of the largest one counts as nothing, and a block's score may miss the unrounded one by about half a
// step of each (tests/test_gpu_kv_scores.py works it out).  Of the blocks that are not forced 97 to 99 in 100 are the same as
// without any rounding, on keys with channels that stand out.
#include <climits>

#include <cooperative_groups.h>

#include "kv.cuh"

namespace fv {
namespace {

struct KvSearch {
  const unsigned char* q;
  size_t q_row, q_head;  // bytes
  int heads, group, k, first, recent;
  const int8_t* codes;
  const float* scale;
  int32_t* out;
};

enum { KV_SEARCH_THREADS = 256, KV_SEARCH_WARPS = 8, KV_SEARCH_LIST = 128, KV_SEARCH_WIDTH = 50000 };

// The 2 D codes of one row's group of queries to dst, by a warp: lanes 0 .. D/4-1 have 4 components each.
template <class T, int D>
__device__ __forceinline__ void query_codes(const KvSearch& a, int row, int head, int8_t* dst) {
  const int lane = lane_id();
  const bool on = lane < D / 4;
  const unsigned char* src = a.q + size_t(row) * a.q_row + size_t(head) * a.group * a.q_head + lane * 8;
  auto load = [&](int g, float* x) {
    uint2 w = make_uint2(0, 0);
    if (on) w = __ldg(reinterpret_cast<const uint2*>(src + size_t(g) * a.q_head));
    const float2 u = Pair<T>::to_float(w.x), v = Pair<T>::to_float(w.y);
    x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = kv_finite(x[i]) ? x[i] : 0.f;
  };
  float most = 0.f, x[4];
  for (int g = 0; g < a.group; ++g) {
    load(g, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(x[i]));
  }
  most = __uint_as_float(__reduce_max_sync(FV_FULL, __float_as_uint(most)));  // none is negative: ordered like whole numbers
  const float down = kv_down(most), den = most > 0.f ? most * down : 1.f, up = 127.f * down, inv = __fdiv_rn(1.f, den);
  int p[4] = {}, n[4] = {};
  for (int g = 0; g < a.group; ++g) {
    load(g, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = kv_whole(x[i] * up, den, inv);
      p[i] += max(c, 0), n[i] += max(-c, 0);
    }
  }
  int top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(p[i], n[i]));
  top = __reduce_max_sync(FV_FULL, top);
  const float by = float(max(top, 1)), inv2 = __fdiv_rn(1.f, by);  // at most 127 * 128, 14 bits
  uint32_t wp = 0, wn = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    wp |= (uint32_t(kv_whole(127.f * float(p[i]), by, inv2)) & 0xFFu) << (8 * i);
    wn |= (uint32_t(kv_whole(-127.f * float(n[i]), by, inv2)) & 0xFFu) << (8 * i);
  }
  if (on) {
    reinterpret_cast<uint32_t*>(dst)[lane] = wn;          // with the lower bounds
    reinterpret_cast<uint32_t*>(dst + D)[lane] = wp;      // with the upper ones
  }
}

// c += a b: 16 blocks by 32 components by 8 rows, whole numbers
__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The largest `k` of n keys in shared memory, 0 standing for none, to out in ascending order.  TEAM warps work on one row: a
// warp, or the whole block (then every thread calls it).  HELD keys a thread stay in registers (0: they are read again each time).
// The threshold is found bit by bit between the largest key and the smallest of the threads' own largest ones, from which on there
// are at least as many keys as threads, and, for a warp, among those keys alone.
template <int TEAM, int HELD>
__device__ __forceinline__ void choose(const uint32_t* keys, int n, int k, int32_t* out, int* s_team, uint2* s_list) {
  const int lane = lane_id(), me = TEAM > 1 ? int(threadIdx.x) : lane, warp = TEAM > 1 ? int(threadIdx.x >> 5) : 0;
  constexpr int STEP = 32 * TEAM;
  uint32_t held[HELD > 0 ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = me + i * STEP < n ? keys[me + i * STEP] : 0u;
  }
  auto each = [&](auto&& f) {
    if constexpr (HELD > 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) f(held[i]);
    } else {
      for (int i = me; i < n; i += STEP) f(keys[i]);
    }
  };
  int phase = 0;
  auto total = [&](unsigned x) {  // over the team
    x = __reduce_add_sync(FV_FULL, x);
    if constexpr (TEAM > 1) {
      if (lane == 0) s_team[phase * TEAM + warp] = int(x);
      __syncthreads();
      x = 0;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) x += unsigned(s_team[phase * TEAM + w]);
      phase ^= 1;
    }
    return x;
  };
  auto largest = [&](uint32_t x) {
    x = __reduce_max_sync(FV_FULL, x);
    if constexpr (TEAM > 1) {
      if (lane == 0) s_team[phase * TEAM + warp] = int(x);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TEAM; ++w) x = max(x, uint32_t(s_team[phase * TEAM + w]));
      phase ^= 1;
    }
    return x;
  };
  unsigned counts = 0;  // candidates, and forced ones times 2^16: there are at most KV_SEARCH_WIDTH of either, so neither leaves its half
  static_assert(KV_SEARCH_WIDTH < 1 << 16, "two counts share a word");
  uint32_t hi = 0, second = 0;  // a thread's two largest keys that are not forced
  each([&](uint32_t x) {
    counts += (x != 0u ? 1u : 0u) + (x == 0xFFFFFFFFu ? 1u << 16 : 0u);
    const uint32_t y = x == 0xFFFFFFFFu ? 0u : x;
    second = max(second, min(hi, y)), hi = max(hi, y);
  });
  counts = total(counts);
  const int there = int(counts & 0xFFFFu), forced = int(counts >> 16);
  const unsigned before = (1u << lane) - 1u;
  auto bisect = [&](uint32_t lo, uint32_t up, auto&& over, uint32_t& t) {  // the least t with at most k keys from it on, or the k-th key
    const uint32_t differ = up ^ lo;
    int bit = differ ? 31 - __clz(int(differ)) : -1;
    t = bit < 0 ? up : up & ~((2u << bit) - 1u);
    for (; bit >= 0; --bit) {
      const uint32_t c = t | 1u << bit;
      int cnt = 0;
      over([&](uint32_t x) { cnt += x >= c; });
      cnt = int(total(unsigned(cnt)));
      if (cnt >= k) t = c;
      if (cnt == k) return true;
    }
    return false;
  };
  uint32_t t = 1u;  // keys from t on are taken
  bool exact = true;  // and there are no more of them than k; else, of those equal to t the first ones
  if (there > k) {
    exact = false;
    if (forced >= k) {
      t = 0xFFFFFFFFu;
    } else {
      // as many keys as threads, or twice as many, are at least as large as this; 0: some thread has none
      const uint32_t least = k <= STEP ? ~largest(~hi) : k <= 2 * STEP ? ~largest(~second) : 0u;
      if constexpr (TEAM == 1) {
        if (least != 0u) {  // those in order to a list of their own: mostly not many more than k
          int count = 0;
          auto file = [&](uint32_t x, int i) {
            const unsigned in = __ballot_sync(FV_FULL, x >= least);
            const int to = count + __popc(in & before);
            if (x >= least && to < KV_SEARCH_LIST) s_list[to] = make_uint2(x, uint32_t(i));
            count += __popc(in);
          };
          if constexpr (HELD > 0) {
#pragma unroll
            for (int i = 0; i < HELD; ++i) file(held[i], 32 * i + lane);
          } else {
            for (int i0 = 0; i0 < n; i0 += 32) file(i0 + lane < n ? keys[i0 + lane] : 0u, i0 + lane);
          }
          if (count <= KV_SEARCH_LIST) {
            __syncwarp();
            uint2 few[KV_SEARCH_LIST / 32];
#pragma unroll
            for (int i = 0; i < KV_SEARCH_LIST / 32; ++i) few[i] = 32 * i + lane < count ? s_list[32 * i + lane] : make_uint2(0u, 0u);
            exact = bisect(least, largest(hi), [&](auto&& f) {
#pragma unroll
              for (int i = 0; i < KV_SEARCH_LIST / 32; ++i) f(few[i].x);
            }, t);
            if (exact) {
              int at = 0;
#pragma unroll
              for (int i = 0; i < KV_SEARCH_LIST / 32; ++i) {
                const unsigned takes = __ballot_sync(FV_FULL, few[i].x >= t);
                if (few[i].x >= t) out[at + __popc(takes & before)] = int(few[i].y);
                at += __popc(takes);
              }
              __syncwarp();
              return;
            }
            __syncwarp();
          } else {
            exact = bisect(least, largest(hi), each, t);
          }
        } else {
          exact = bisect(1u, largest(hi), each, t);
        }
      } else {
        exact = bisect(max(least, 1u), largest(hi), each, t);
      }
    }
  }
  if (TEAM == 1 && exact) {
    int at = 0;
    auto put = [&](uint32_t x, int i) {
      const unsigned takes = __ballot_sync(FV_FULL, x >= t);
      if (x >= t) out[at + __popc(takes & before)] = i;
      at += __popc(takes);
    };
    if constexpr (HELD > 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) put(held[i], 32 * i + lane);
    } else {
      for (int i0 = 0; i0 < n; i0 += 32) put(i0 + lane < n ? keys[i0 + lane] : 0u, i0 + lane);
    }
    for (int i = at + lane; i < k; i += 32) out[i] = -1;
    return;
  }
  // every warp of the team has a stretch of the keys
  const int per = TEAM > 1 ? ((n + TEAM - 1) / TEAM + 31) / 32 * 32 : n;
  const int begin = min(n, warp * per), end = min(n, begin + per);
  int above = 0, equal = 0;
  for (int i = begin + lane; i < end; i += 32) above += keys[i] > t, equal += keys[i] == t;
  above = __reduce_add_sync(FV_FULL, above), equal = __reduce_add_sync(FV_FULL, equal);
  int all_above = above, equal_before = 0, above_before = 0;
  if constexpr (TEAM > 1) {
    __syncthreads();
    if (lane == 0) s_team[warp] = above, s_team[TEAM + warp] = equal;
    __syncthreads();
    all_above = 0;
    for (int w = 0; w < TEAM; ++w) {
      all_above += s_team[w];
      if (w < warp) above_before += s_team[w], equal_before += s_team[TEAM + w];
    }
  }
  const int room = k - all_above;  // for keys equal to t
  int at = above_before + min(equal_before, room), seen = equal_before;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t x = i < end ? keys[i] : 0u;
    const bool eq = i < end && x == t;
    const unsigned eqs = __ballot_sync(FV_FULL, eq);
    const bool take = i < end && (x > t || (eq && seen + __popc(eqs & before) < room));
    const unsigned takes = __ballot_sync(FV_FULL, take);
    if (take) out[at + __popc(takes & before)] = i;
    at += __popc(takes), seen += __popc(eqs);
  }
  if (warp == TEAM - 1)  // its `at` is how many there are
    for (int i = at + lane; i < k; i += 32) out[i] = -1;
}

// The least t with at least k of a warp's keys from it on, and exactly k where that can be; there are more than k, fewer than
// k of them forced.  N keys a lane, 0 for none.
template <int N>
__device__ __forceinline__ uint32_t kth(const uint32_t* keys, int k) {
  uint32_t hi = 0, low = 0;  // largest that is not forced; the largest complement
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (keys[i] != 0xFFFFFFFFu) hi = max(hi, keys[i]);
    if (keys[i] != 0u) low = max(low, ~keys[i]);
  }
  hi = __reduce_max_sync(FV_FULL, hi), low = ~__reduce_max_sync(FV_FULL, low);
  const uint32_t differ = hi ^ low;
  int bit = differ ? 31 - __clz(int(differ)) : -1;
  uint32_t t = bit < 0 ? hi : hi & ~((2u << bit) - 1u);
  for (; bit >= 0; --bit) {
    const uint32_t c = t | 1u << bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) cnt += keys[i] >= c;
    cnt = __reduce_add_sync(FV_FULL, cnt);
    if (cnt >= k) t = c;
    if (cnt == k) break;
  }
  return max(t, 1u);
}

// The same as choose<8, ..> for most searches, with three barriers instead of one for every bit: of the threads' largest keys the
// k-th is a bound that few more than k keys reach; they are filed in order, and a warp finishes.  False: too many reach it, and
// nothing is done.
__device__ __forceinline__ bool choose_few(const uint32_t* keys, int n, int k, int32_t* out, int* s_team, uint32_t* s_tops, uint2* s_list) {
  constexpr int W = KV_SEARCH_WARPS;
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  const int per = ((n + W - 1) / W + 31) / 32 * 32, begin = min(n, warp * per), end = min(n, begin + per);  // a warp's stretch
  if (k > KV_SEARCH_LIST) return false;
  uint32_t top = 0;
  for (int i = begin + lane; i < end; i += 32) top = max(top, keys[i]);
  s_tops[threadIdx.x] = top;
  __syncthreads();
  uint32_t tops[W];
  int there = 0;  // and forced ones times 2^16; every warp finds the bound for itself
#pragma unroll
  for (int i = 0; i < W; ++i) tops[i] = s_tops[32 * i + lane], there += (tops[i] != 0u) + (tops[i] == 0xFFFFFFFFu ? 1 << 16 : 0);
  there = __reduce_add_sync(FV_FULL, there);
  if ((there & 0xFFFF) <= k || (there >> 16) >= k) return false;
  const uint32_t least = kth<W>(tops, k);
  int count = 0;
  for (int i0 = begin; i0 < end; i0 += 32) count += __popc(__ballot_sync(FV_FULL, i0 + lane < end && keys[i0 + lane] >= least));
  if (lane == 0) s_team[warp] = count;
  __syncthreads();
  int at = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) at += s_team[w];
    all += s_team[w];
  }
  if (all > KV_SEARCH_LIST) return false;
  const unsigned before = (1u << lane) - 1u;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const uint32_t x = i0 + lane < end ? keys[i0 + lane] : 0u;
    const unsigned in = __ballot_sync(FV_FULL, x >= least);
    if (x >= least) s_list[at + __popc(in & before)] = make_uint2(x, uint32_t(i0 + lane));
    at += __popc(in);
  }
  __syncthreads();
  if (warp) return true;
  constexpr int N = KV_SEARCH_LIST / 32;
  uint32_t few[N], which[N];
  int forced = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint2 x = 32 * i + lane < all ? s_list[32 * i + lane] : make_uint2(0u, 0u);
    few[i] = x.x, which[i] = x.y;
    forced += x.x == 0xFFFFFFFFu;
  }
  forced = __reduce_add_sync(FV_FULL, forced);
  const uint32_t t = all == k ? 1u : forced >= k ? 0xFFFFFFFFu : kth<N>(few, k);
  int above = 0, from = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) above += few[i] > t, from += few[i] >= t;
  above = __reduce_add_sync(FV_FULL, above), from = __reduce_add_sync(FV_FULL, from);
  const int room = from == k ? k : k - above;  // for keys equal to t: all of them, or the first
  int to = 0, seen = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned eqs = __ballot_sync(FV_FULL, few[i] == t);
    const bool take = few[i] > t || (few[i] == t && seen + __popc(eqs & before) < room);
    const unsigned takes = __ballot_sync(FV_FULL, take);
    if (take) out[to + __popc(takes & before)] = int(which[i]);
    to += __popc(takes), seen += __popc(eqs);
  }
  return true;
}

// TEAM = 8: one row of the call to a CTA (a token), or to a cluster of up to 8 where there are few.  TEAM = 1: 8 * NT consecutive rows of one sequence (a prompt), which share
// what is read of the bounds.  A warp takes 16 blocks at a time straight from memory into the operands of a matrix product:
// the components are a sum, so lane t of four may hold 16 neighbouring ones where the product would have it hold 4 of each 16,
// on both sides.
template <class T, int D, int NT, int TEAM>
__global__ void __launch_bounds__(KV_SEARCH_THREADS, 3) kv_search_kernel(KvSearch a, KvBatch m, int pitch, int splits) {
  constexpr int R = TEAM > 1 ? 1 : 8 * NT, CHUNKS = 2 * D / 64;
  constexpr int SHIFT = R == 1 ? 0 : R == 8 ? 3 : 4;
  __shared__ __align__(16) int8_t s_codes[8 * NT][2 * D + 16];
  __shared__ int s_team[2 * KV_SEARCH_WARPS];
  __shared__ uint2 s_list[TEAM > 1 ? 1 : KV_SEARCH_WARPS][KV_SEARCH_LIST];
  __shared__ uint32_t s_tops[TEAM > 1 ? KV_SEARCH_THREADS : 1];
  uint32_t* const keys = reinterpret_cast<uint32_t*>(dyn_smem());  // [R][pitch]
  const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int rank = TEAM > 1 ? int(blockIdx.x) % splits : 0;
  int b, row, rows;  // the CTA's rows are row .. row + rows - 1
  {
    const int item = TEAM > 1 ? int(blockIdx.x) / splits : int(blockIdx.x);
    b = m.cu ? kv_find(m, item, R, R > 1) : item;
    const int r0 = m.cu_at(b), r1 = max(m.cu_at(b + 1), r0);
    row = R > 1 ? r0 + ((item - ((r0 >> SHIFT) + b)) << SHIFT) : item;
    rows = min(R, r1 - row);
    if (row < r0 || rows <= 0) return;  // the same for a whole cluster
  }
  const int pos0 = m.len(b) - max(m.cu_at(b + 1), row + 1) + row;  // of the first row
  const int n = min(m.table_width, pos0 + rows - 1 < 0 ? 0 : ((pos0 + rows - 1) >> m.page_shift) + 1);
  const int begin = (rank * KV_SEARCH_WARPS + warp) * 16, step = splits * KV_SEARCH_WARPS * 16;
  int ahead[2];  // the pages that are next
#pragma unroll
  for (int i = 0; i < 2; ++i) ahead[i] = begin + g + 8 * i < n ? m.page(b, begin + g + 8 * i) : -1;
  for (int r = warp; r < 8 * NT; r += KV_SEARCH_WARPS) {
    if (r < rows) {
      query_codes<T, D>(a, row + r, head, s_codes[r]);
    } else {
      for (int i = lane; i < 2 * D / 4; i += 32) reinterpret_cast<uint32_t*>(s_codes[r])[i] = 0u;
    }
  }
  if (TEAM > 1 && splits > 1) cooperative_groups::this_cluster().sync();  // also: the first CTA is there to be written to
  else __syncthreads();
  uint4 q[NT][CHUNKS];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) q[x][c] = *reinterpret_cast<const uint4*>(&s_codes[8 * x + g][64 * c + 16 * t]);
  // the keys of a row's cluster come together in its first CTA
  uint32_t* const to = TEAM > 1 && splits > 1 ? cooperative_groups::this_cluster().map_shared_rank(keys, 0) : keys;
  for (int j0 = begin; j0 < n; j0 += step) {
    int acc[NT][4] = {};
    int page[2];
    float scale[2];
    uint4 w[2][CHUNKS];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      page[i] = ahead[i];
      const size_t at = size_t(max(page[i], 0)) * a.heads + head;
      scale[i] = page[i] >= 0 ? __ldg(a.scale + at) : 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        w[i][c] = page[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(a.codes + at * (2 * D) + 64 * c + 16 * t)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) ahead[i] = j0 + step + g + 8 * i < n ? m.page(b, j0 + step + g + 8 * i) : -1;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        mma_s8(acc[x], w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, q[x][c].x, q[x][c].y);
        mma_s8(acc[x], w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, q[x][c].z, q[x][c].w);
      }
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int r = 8 * x + 2 * t + z, last = (pos0 + r) >> m.page_shift;  // negative where the row has no position
        if (r >= R) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = j0 + g + 8 * i;
          // + 0: of the two zeros the one that is not negative
          uint32_t key = order_bits(__fadd_rn(__fmul_rn(float(acc[x][2 * i + z]), scale[i]), 0.f));
          if (j < a.first || j > last - a.recent) key = 0xFFFFFFFFu;
          if (j > last || page[i] < 0) key = 0u;
          if (j < n) to[size_t(r) * pitch + j] = key;
        }
      }
  }
  if constexpr (TEAM > 1) {
    if (splits > 1) {
      cooperative_groups::this_cluster().sync();
      if (rank) return;
    }
  }
  __syncthreads();
  auto pick = [&](int r) {
    const uint32_t* mine = keys + size_t(r) * pitch;
    int32_t* out = a.out + (size_t(row + r) * a.heads + head) * a.k;
    uint2* const list = s_list[TEAM > 1 ? 0 : warp];
    if constexpr (TEAM > 1) {
      if (choose_few(mine, n, a.k, out, s_team, s_tops, list)) return;
      __syncthreads();
    }
    if (n <= 8 * 32 * TEAM) choose<TEAM, 8>(mine, n, a.k, out, s_team, list);
    else if (TEAM == 1 && n <= 16 * 32) choose<TEAM, TEAM == 1 ? 16 : 0>(mine, n, a.k, out, s_team, list);
    else if (TEAM == 1 && n <= 24 * 32) choose<TEAM, TEAM == 1 ? 24 : 0>(mine, n, a.k, out, s_team, list);
    else choose<TEAM, 0>(mine, n, a.k, out, s_team, list);
  };
  if constexpr (TEAM > 1) {
    pick(0);
  } else {
    for (int r = warp; r < rows; r += KV_SEARCH_WARPS) pick(r);
  }
}

int search_pitch(size_t width) { return int((width + 31) / 32 * 32 + 4); }  // 2 * pitch is 8 mod 32: keys go to 32 banks

template <class T, int D, int NT, int TEAM>
int search_launch(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvSearch& a) {
  constexpr int R = TEAM > 1 ? 1 : 8 * NT;
  const int pitch = search_pitch(b->table_width);
  const size_t smem = size_t(R) * pitch * 4, items = R == 1 ? b->rows : b->rows / R + b->nseq;
  FV_TRY((kv_allow_smem<kv_search_kernel<T, D, NT, TEAM>>(kv->device, smem)));
  int splits = 1;  // CTAs to a row: while the GPU has room for more, and each warp has some of the blocks
  while (R == 1 && splits < 8 && items * kv->heads * splits <= 148 && b->table_width > size_t(splits) * KV_SEARCH_WARPS * 16) splits *= 2;
  if (splits > 1) {
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {unsigned(splits), 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(items * splits), kv->heads);
    cfg.blockDim = dim3(KV_SEARCH_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FV_CUDA(cudaLaunchKernelEx(&cfg, kv_search_kernel<T, D, NT, TEAM>, a, kv_batch(kv, b), pitch, splits));
    return FV_OK;
  }
  kv_search_kernel<T, D, NT, TEAM><<<dim3(unsigned(items), kv->heads), KV_SEARCH_THREADS, smem, s>>>(a, kv_batch(kv, b), pitch, 1);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

template <class T, int D>
int search_of(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvSearch& a) {
  // 16 rows of a prompt share a read of the bounds, or 8 where the keys of 16 do not leave room for two CTAs on an SM (32 of them
  // leave room for two where 16 leave it for three: 99 us and 92 for 3.2k rows over 512 blocks); where a sequence brings a few
  // rows, or the table is wide, a CTA works on one row
  const size_t row = size_t(search_pitch(b->table_width)) * 4, most = 100 * 1024;
  if (b->rows <= 4 * b->nseq || 8 * row > 2 * most) return search_launch<T, D, 1, 8>(kv, s, b, a);
  if (16 * row <= most) return search_launch<T, D, 2, 1>(kv, s, b, a);
  return search_launch<T, D, 1, 1>(kv, s, b, a);
}

template <class T>
int search_dim(const fv_kv* kv, cudaStream_t s, const fv_kv_batch* b, const KvSearch& a) {
  if (kv->dim == 64) return search_of<T, 64>(kv, s, b, a);
  if (kv->dim == 96) return search_of<T, 96>(kv, s, b, a);
  return search_of<T, 128>(kv, s, b, a);
}

}  // namespace
}  // namespace fv

extern "C" int fv_kv_search_dev(const fv_kv* kv, void* stream, const fv_kv_batch* batch, const void* q, size_t q_row, size_t q_head,
                                size_t group, size_t k, size_t first, size_t recent, int32_t* out) {
  FV_TRY(fv::kv_check(kv, batch, "fv_kv_search_dev"));
  if (group == 0 || group > 128) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_search_dev: group is 1 to 128 query heads to a key head");
  if (k == 0 || k > FV_KV_MAX_BLOCKS) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_search_dev: k is 1 to 4096 blocks");
  if (batch->table_width > fv::KV_SEARCH_WIDTH)
    return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_search_dev: a table of more than 50000 blocks; use larger pages");
  if (batch->rows == 0 || batch->nseq == 0) return FV_OK;
  if (!q || !out) return fv::fail(FV_ERR_ARG, "fv_kv_search_dev: NULL queries or result");
  if (!fv::kv_aligned(q, 16) || ((q_row | q_head) & 7) || !fv::kv_aligned(out, 4))
    return fv::fail(FV_ERR_ARG, "fv_kv_search_dev: queries begin on 16 bytes, their strides are multiples of 8 elements, and the result begins on 4 bytes");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  const fv::KvSearch a{static_cast<const unsigned char*>(q), 2 * q_row, 2 * q_head, int(kv->heads), int(group), int(k),
                       int(first < INT_MAX / 2 ? first : INT_MAX / 2), int(recent < INT_MAX / 2 ? recent : INT_MAX / 2), kv->bound_codes,
                       kv->bound_scale, out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv->dtype == FV_KV_BF16 ? fv::search_dim<__nv_bfloat16>(kv, s, batch, a) : fv::search_dim<__half>(kv, s, batch, a);
}
