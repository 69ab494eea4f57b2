// Which pages of a cache are in use, and their copies.
//
// 256 sequences of up to 130 blocks among 30,000 pages: forked in 2.2 us, given back in 2.2, given room in 9.4 and their pages copied in 5.8; 25 us of
// a step's 55, whose rest is the host's.  20,000 pages, half of them in use: planned in 13 us, 660 MB moved in 213 (6.2 TB/s).
//
// refs[p] counts the table entries that hold page p; 0: it is free.  fork and free are a pass over the table with an addition for each entry.
// extend and compact have to number things in order (the free pages, the blocks that want one), so each is planned by one CTA whose
// threads meet at its barriers (compact: one to every 32,768 pages), and what is to be copied is copied by all SMs in a second kernel.  Nothing depends on the order of
// atomics: additions commute, and a page's last holder is found by the smallest number.
#include <climits>

#include "kv.cuh"

namespace fv {
namespace {

enum { PAGES_THREADS = 1024, PAGES_WARPS = 32, PAGES_SEQS = 2048, COPY_THREADS = 256, COPY_SLICE = 32 * 1024, COPY_PARTS = 7, COPY_CACHES = 8, PAGES_WINDOW = 32 * 1024 };

struct Pages {
  int32_t* refs;
  int pages, page_shift;
};
struct Table {
  int32_t* at;
  size_t stride;
  int width, nseq;
};

// Sum over the CTA up to this thread, exclusive; *all: over everybody.  s: PAGES_WARPS + 1 ints, in use until the next barrier.
__device__ __forceinline__ int sum_before(int x, int* s, int* all) {
  const int warp = threadIdx.x >> 5, lane = lane_id();
  int up = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FV_FULL, up, o);
    if (lane >= o) up += y;
  }
  if (lane == 31) s[warp] = up;
  __syncthreads();
  const int mine = lane < PAGES_WARPS ? s[lane] : 0;
  int w = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FV_FULL, w, o);
    if (lane >= o) w += y;
  }
  *all = __shfl_sync(FV_FULL, w, 31);
  const int before = __shfl_sync(FV_FULL, w - mine, warp);
  __syncthreads();
  return before + up - x;
}

// The counts of a window of pages in a CTA's registers: a warp has up to 1024 of them in ascending order, a lane four neighbours at a time.  So passes over
// them do not wait for memory again, and the look may be long before.
struct PageWindow {
  enum { AHEAD = PAGES_WINDOW / PAGES_WARPS / 128 };
  int begin, end;  // of the warp's pages
  int4 r[AHEAD];
  __device__ __forceinline__ void look(const Pages& p, int base) {
    const bool wide = (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0;
    const int all = min(p.pages - base, int(PAGES_WINDOW)), share = ((all + PAGES_WARPS - 1) / PAGES_WARPS + 127) & ~127;
    begin = base + int(threadIdx.x >> 5) * share, end = min(begin + share, base + all);
#pragma unroll
    for (int z = 0; z < AHEAD; ++z) {
      const int at = begin + 128 * z + 4 * int(lane_id());
      r[z] = make_int4(-1, -1, -1, -1);  // behind the last page
      if (at >= end) continue;
      if (wide && at + 4 <= p.pages) {
        r[z] = __ldcg(reinterpret_cast<const int4*>(p.refs + at));
      } else {
        r[z].x = __ldcg(p.refs + at);
        if (at + 1 < p.pages) r[z].y = __ldcg(p.refs + at + 1);
        if (at + 2 < p.pages) r[z].z = __ldcg(p.refs + at + 2);
        if (at + 3 < p.pages) r[z].w = __ldcg(p.refs + at + 3);
      }
    }
  }
  // f(first of four pages, their counts) for whole warps, in ascending order, as long as it says so
  template <class F>
  __device__ __forceinline__ void each(const Pages& p, F&& f) const {
#pragma unroll
    for (int z = 0; z < AHEAD; ++z)
      if (begin + 128 * z < end && !f(begin + 128 * z + 4 * int(lane_id()), r[z])) return;
  }
};

// ---------------------------------------------------------------------------------------------
struct Extend {
  const int32_t *lens, *more;
  int32_t* missing;
  int32_t *count, *before, *free, *src, *dst;  // in the caller's work
};

// Entry e of the blocks that rows come to: sequence b's are before[b] .. before[b + 1], from block `first` on.
__device__ __forceinline__ int32_t* entry_at(const Pages& p, const Table& t, const Extend& x, const int* before, int e) {
  int lo = 0, n = t.nseq;
  while (n > 1) {  // the last sequence that begins at or before e
    const int h = n / 2;
    if (before[lo + h] <= e) lo += h, n -= h;
    else n = h;
  }
  const int first = max(__ldg(x.lens + lo), 0) >> p.page_shift;
  return t.at + size_t(lo) * t.stride + first + (e - before[lo]);
}

// What a table entry says while this runs: a page; -1: it wants one; -2 - q: it wants one and a copy of page q.  A thread's first entry is
// in its registers.
__global__ void __launch_bounds__(PAGES_THREADS) pages_extend_kernel(Pages p, Table t, Extend x) {
  __shared__ int s_sum[PAGES_WARPS + 1], s_before[PAGES_SEQS + 1], s_count;
  const int tid = threadIdx.x;
  PageWindow window;
  window.look(p, 0);  // those that are free now: counts that come to nothing below are given back
  int* const before = t.nseq <= PAGES_SEQS ? s_before : x.before;
  if (tid == 0) s_count = 0, before[0] = 0;
  int entries = 0;
  for (int b0 = 0; b0 < t.nseq; b0 += PAGES_THREADS) {
    const int b = b0 + tid;
    int n = 0, all;
    if (b < t.nseq) {
      const int len = max(__ldg(x.lens + b), 0), more = __ldg(x.more + b);
      const long long end = ((long long)(len) + more + (1 << p.page_shift) - 1) >> p.page_shift;
      if (more >= 0) n = max(int(min(end, (long long)(t.width))) - (len >> p.page_shift), 0);
    }
    const int up = sum_before(n, s_sum, &all);
    if (b < t.nseq) before[b + 1] = entries + up + n;
    entries += all;
  }
  __syncthreads();
  int32_t* const at0 = tid < entries ? entry_at(p, t, x, before, tid) : nullptr;
  int q0 = at0 ? __ldcg(at0) : 0;
  auto get = [&](int e) { return e == tid ? q0 : __ldcg(entry_at(p, t, x, before, e)); };
  auto put = [&](int e, int q) {
    if (e == tid) q0 = q;
    else __stcg(entry_at(p, t, x, before, e), q);
  };
  // who wants a page
  bool shared = false;
  int wants = 0, all;
  for (int e = tid; e < entries; e += PAGES_THREADS) {
    const int q = get(e);
    if (unsigned(q) >= unsigned(p.pages)) put(e, -1), ++wants;
    else if (__ldcg(p.refs + q) > 1) put(e, -2 - q), shared = true, ++wants;
  }
  if (__syncthreads_or(shared)) {
    // who holds a page with others gives it up; where nobody is left, refs becomes the smallest number of those who did, far below 0, and
    // that one keeps it
    for (int e = tid; e < entries; e += PAGES_THREADS) {
      const int q = -2 - get(e);
      if (q >= 0) atomicSub(p.refs + q, 1);
    }
    __syncthreads();
    for (int e = tid; e < entries; e += PAGES_THREADS) {
      const int q = -2 - get(e);
      if (q >= 0 && __ldcg(p.refs + q) <= 0) atomicMin(p.refs + q, INT_MIN + e);
    }
    __syncthreads();
    bool keeps0 = false;  // the thread's first entry keeps its page
    for (int e = tid; e < entries; e += PAGES_THREADS) {
      const int q = -2 - get(e);
      if (q >= 0 && __ldcg(p.refs + q) == INT_MIN + e) put(e, q), --wants, keeps0 = keeps0 || e == tid;
    }
    __syncthreads();
    for (int e = tid; e < entries; e += PAGES_THREADS) {
      const int q = get(e);
      if (e == tid ? keeps0 : q >= 0 && __ldcg(p.refs + q) < 0) __stcg(p.refs + q, 1);
    }
  }
  sum_before(wants, s_sum, &all);
  wants = all;
  if (wants) {
    // the free pages, as many as are wanted
    int found = 0;
    for (int base = 0;;) {
      int n = 0;
      window.each(p, [&](int, const int4& r) { return n += (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0), true; });
      int rank = found + sum_before(n, s_sum, &all);  // of a lane: its pages are not neighbours, only the warp's sum counts
      rank = __shfl_sync(FV_FULL, rank, 0);
      found += all;
      if (rank < wants) {
        window.each(p, [&](int at, const int4& r) {
          const int c = (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0);
          int up = c;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FV_FULL, up, o);
            if (int(lane_id()) >= o) up += y;
          }
          int i = rank + up - c;
          if (r.x == 0 && i < wants) x.free[i] = at;
          i += r.x == 0;
          if (r.y == 0 && i < wants) x.free[i] = at + 1;
          i += r.y == 0;
          if (r.z == 0 && i < wants) x.free[i] = at + 2;
          i += r.z == 0;
          if (r.w == 0 && i < wants) x.free[i] = at + 3;
          rank += __shfl_sync(FV_FULL, up, 31);
          return rank < wants;
        });
      }
      if (found >= wants || p.pages - base <= PAGES_WINDOW) break;
      base += PAGES_WINDOW;
      window.look(p, base);
    }
    if (found < wants) {  // nothing is changed
      for (int e = tid; e < entries; e += PAGES_THREADS) {
        const int q = -2 - get(e);
        if (q >= 0) atomicAdd(p.refs + q, 1), put(e, q);
      }
      if (at0) *at0 = q0;
      if (tid == 0) *x.missing = wants - found, *x.count = 0;
      return;
    }
    __syncthreads();
    int given = 0;
    for (int e0 = 0; e0 < entries; e0 += PAGES_THREADS) {
      const int e = e0 + tid, q = e < entries ? get(e) : 0;
      const int i = given + sum_before(q < 0, s_sum, &all);
      given += all;
      if (q < 0) {
        const int page = __ldcg(x.free + i);
        put(e, page);
        p.refs[page] = 1;
        if (q < -1) {
          const int c = atomicAdd(&s_count, 1);
          x.src[c] = -2 - q, x.dst[c] = page;
        }
      }
    }
    __syncthreads();
  }
  if (at0) *at0 = q0;
  if (tid == 0) *x.missing = 0, *x.count = s_count;
}

__global__ void __launch_bounds__(256) pages_fork_kernel(Pages p, Table from, const int32_t* lens, const int32_t* parents, Table to) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= to.width) return;
  for (int i = blockIdx.y; i < to.nseq; i += gridDim.y) {
    const int b = __ldg(parents + i);
    int q = -1;
    if (unsigned(b) < unsigned(from.nseq) && j < from.width) {
      const int len = lens ? max(__ldg(lens + b), 0) : INT_MAX;
      if ((long long)(j) << p.page_shift < len) q = __ldg(from.at + size_t(b) * from.stride + j);
      if (unsigned(q) >= unsigned(p.pages)) q = -1;
    }
    to.at[size_t(i) * to.stride + j] = q;
    if (q >= 0) atomicAdd(p.refs + q, 1);
  }
}

__global__ void __launch_bounds__(256) pages_free_kernel(Pages p, Table t, const int32_t* lens) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= t.width) return;
  for (int b = blockIdx.y; b < t.nseq; b += gridDim.y) {
    const int len = lens ? max(__ldg(lens + b), 0) : 0;
    if ((long long)(j) << p.page_shift < len) continue;
    int32_t* at = t.at + size_t(b) * t.stride + j;
    const int q = *at;
    if (q == -1) continue;
    *at = -1;
    if (unsigned(q) < unsigned(p.pages) && atomicSub(p.refs + q, 1) <= 0) atomicAdd(p.refs + q, 1);  // it was free already
  }
}

__global__ void __launch_bounds__(256) pages_remap_kernel(const int32_t* map, int pages, Table t) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= t.width) return;
  for (int b = blockIdx.y; b < t.nseq; b += gridDim.y) {
    int32_t* at = t.at + size_t(b) * t.stride + j;
    const int q = *at;
    if (unsigned(q) < unsigned(pages)) *at = __ldg(map + q);
  }
}

// Pages in use in each window.
__global__ void __launch_bounds__(PAGES_THREADS) pages_count_kernel(Pages p, int32_t* counts) {
  __shared__ int s_sum[PAGES_WARPS + 1];
  PageWindow window;
  window.look(p, int(blockIdx.x) * PAGES_WINDOW);
  int n = 0, all;
  window.each(p, [&](int, const int4& r) { return n += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0), true; });
  sum_before(n, s_sum, &all);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

// With n pages in use a free one below n is a hole, and one in use from there on moves to the hole of its number.  A CTA lists the holes and movers
// of its window; how many there are before it follows from the windows' counts and, where one lies on both sides of n, a look at that.
__global__ void __launch_bounds__(PAGES_THREADS) pages_compact_kernel(Pages p, const int32_t* counts, int32_t* map, int32_t* used, int32_t* count, int32_t* src, int32_t* dst) {
  __shared__ int s_sum[PAGES_WARPS + 1];
  const int lane = lane_id(), windows = gridDim.x, mine = blockIdx.x;
  PageWindow window;
  window.look(p, mine * PAGES_WINDOW);
  int n = 0, live, all;
  if (windows == 1) {
    window.each(p, [&](int, const int4& r) { return n += (r.x > 0) + (r.y > 0) + (r.z > 0) + (r.w > 0), true; });
  } else {
    for (int i = threadIdx.x; i < windows; i += PAGES_THREADS) n += __ldcg(counts + i);
  }
  sum_before(n, s_sum, &live);
  // holes and movers of the windows before
  int hole = 0, mover = 0, moved = 0;
  if (windows > 1) {
    const int border = live / PAGES_WINDOW;
    int below = 0;  // in use in the border's window, in front of the border
    for (int i = border * PAGES_WINDOW + threadIdx.x; i < live; i += PAGES_THREADS) below += __ldcg(p.refs + i) > 0;
    sum_before(below, s_sum, &below);
    int h = 0, m = 0, t = 0;
    for (int i = threadIdx.x; i < windows; i += PAGES_THREADS) {
      const int c = __ldcg(counts + i);
      const int holes = i < border ? PAGES_WINDOW - c : i == border ? live - border * PAGES_WINDOW - below : 0;
      t += holes;
      if (i < mine) h += holes, m += i < border ? 0 : i == border ? c - below : c;
    }
    sum_before(h, s_sum, &hole);
    sum_before(m, s_sum, &mover);
    sum_before(t, s_sum, &moved);
  }
  int holes = 0, movers = 0;
  window.each(p, [&](int at, const int4& r) {
    const int* c = reinterpret_cast<const int*>(&r);
#pragma unroll
    for (int z = 0; z < 4; ++z) holes += at + z < live && c[z] <= 0, movers += at + z >= live && at + z < p.pages && c[z] > 0;
    return true;
  });
  hole += sum_before(holes, s_sum, &all);
  if (windows == 1) moved = all;
  mover += sum_before(movers, s_sum, &all);
  hole = __shfl_sync(FV_FULL, hole, 0), mover = __shfl_sync(FV_FULL, mover, 0);
  window.each(p, [&](int at, const int4& r) {
    const int* c = reinterpret_cast<const int*>(&r);
    int own = 0;  // a hole, or from `live` on a mover: a lane's four are counted together, 128 pages lie on both sides of `live` at most once
#pragma unroll
    for (int z = 0; z < 4; ++z) own += at + z < live ? c[z] <= 0 : at + z < p.pages && c[z] > 0 ? 1 << 16 : 0;
    int up = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(FV_FULL, up, o);
      if (lane >= o) up += y;
    }
    int h = hole + ((up - own) & 0xFFFF), m = mover + ((up - own) >> 16);
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      if (at + z >= p.pages) continue;
      if (at + z < live && c[z] <= 0) dst[h++] = at + z;
      if (at + z >= live && c[z] > 0) src[m++] = at + z;
      map[at + z] = c[z] > 0 ? at + z : -1;  // those that move are put right as they do
    }
    const int sum = __shfl_sync(FV_FULL, up, 31);
    hole += sum & 0xFFFF, mover += sum >> 16;
    return true;
  });
  if (mine == 0 && threadIdx.x == 0) *used = live, *count = moved;
}

// ---------------------------------------------------------------------------------------------
// Copies of pages: what the caches' buffers hold of a page, one behind the other, in slices of 32 KB; a CTA has 8 loads of 16 bytes a thread
// on their way.  Slices are of the page, not of a buffer, since small pages would be nothing but ends of buffers (16 rows of one head of 64,
// 8000 pages: 79 us by buffers).  5000 pages of 131 KB: 220 us, 6.0 TB/s, 0.92 of the copy rate.
struct CopyPart {
  unsigned char* at;
  unsigned bytes, start;  // of a page; its first 16 bytes among those of the page
};
struct Copy {
  CopyPart wide[COPY_CACHES * COPY_PARTS], narrow[COPY_CACHES * COPY_PARTS];  // in whole 16 bytes, and in 4
  int nwide, nnarrow;
  unsigned pieces, slices;  // of 16 bytes, and of 32 KB of these
  const int32_t *src, *dst, *count;
  long long n;
  unsigned pages;
  int32_t *map, *refs;  // not NULL: the pages move, and take their counts along
};

// SMALL: pages of less than a quarter of a slice (8000 of 4.5 KB: 23.6 us, 34.5 with a CTA to each; of 13.8 KB: slower), of which an item has several, so that every thread has something to copy.
template <bool SMALL>
__global__ void __launch_bounds__(COPY_THREADS) pages_copy_kernel(const __grid_constant__ Copy c) {
  constexpr int AHEAD = COPY_SLICE / 16 / COPY_THREADS;
  const long long pairs = c.count ? min(c.n, (long long)(max(__ldcg(c.count), 0))) : c.n;
  const long long items = SMALL ? (pairs * c.pieces + COPY_SLICE / 16 - 1) / (COPY_SLICE / 16) : pairs * c.slices;
  if (c.map)
    for (long long i = (long long)(blockIdx.x) * COPY_THREADS + threadIdx.x; i < pairs; i += (long long)(gridDim.x) * COPY_THREADS) {
      const int from = __ldcg(c.src + i), to = __ldcg(c.dst + i);
      c.map[from] = to;
      c.refs[to] = __ldcg(c.refs + from);
      c.refs[from] = 0;
    }
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    if constexpr (SMALL) {
      const long long begin = item * (COPY_SLICE / 16), first = begin / c.pieces;
      const unsigned rest = unsigned(begin - first * c.pieces) + threadIdx.x;
      uint4 x[AHEAD];
      unsigned char* out[AHEAD];
#pragma unroll
      for (int z = 0; z < AHEAD; ++z) {
        const unsigned l = rest + z * COPY_THREADS, n = l / c.pieces, i = l - n * c.pieces;
        out[z] = nullptr;
        if (first + n >= pairs) continue;
        const unsigned from = unsigned(__ldcg(c.src + first + n)), to = unsigned(__ldcg(c.dst + first + n));
        if (from >= c.pages || to >= c.pages) continue;
        int part = 0;
        while (part + 1 < c.nwide && i >= c.wide[part + 1].start) ++part;
        const CopyPart& p = c.wide[part];
        const size_t at = size_t(i - p.start) * 16;
        out[z] = p.at + size_t(to) * p.bytes + at;
        x[z] = __ldcs(reinterpret_cast<const uint4*>(p.at + size_t(from) * p.bytes + at));
        if (i < 32) {  // the first threads of a page have its odd ends too
          const unsigned threads = min(c.pieces, 32u);
          for (int e = 0; e < c.nnarrow; ++e) {
            const CopyPart& y = c.narrow[e];
            for (unsigned b = i * 4; b < y.bytes; b += threads * 4)
              *reinterpret_cast<uint32_t*>(y.at + size_t(to) * y.bytes + b) = *reinterpret_cast<const uint32_t*>(y.at + size_t(from) * y.bytes + b);
          }
        }
      }
#pragma unroll
      for (int z = 0; z < AHEAD; ++z)
        if (out[z]) __stcs(reinterpret_cast<uint4*>(out[z]), x[z]);
      continue;
    }
    const long long pair = item / c.slices;
    const unsigned slice = unsigned(item - pair * c.slices);
    const unsigned from = unsigned(__ldcg(c.src + pair)), to = unsigned(__ldcg(c.dst + pair));
    if (from >= c.pages || to >= c.pages) continue;
    const unsigned first = slice * (COPY_SLICE / 16) + threadIdx.x;
    uint4 x[AHEAD];
    auto each = [&](auto&& f) {
      int part = 0;
#pragma unroll
      for (int z = 0; z < AHEAD; ++z) {
        const unsigned i = first + z * COPY_THREADS;
        if (i >= c.pieces) continue;
        while (part + 1 < c.nwide && i >= c.wide[part + 1].start) ++part;
        const CopyPart& p = c.wide[part];
        f(z, p, size_t(i - p.start) * 16);
      }
    };
    each([&](int z, const CopyPart& p, size_t at) { x[z] = __ldcs(reinterpret_cast<const uint4*>(p.at + size_t(from) * p.bytes + at)); });
    each([&](int z, const CopyPart& p, size_t at) { __stcs(reinterpret_cast<uint4*>(p.at + size_t(to) * p.bytes + at), x[z]); });
    if (slice == 0)
      for (int part = 0; part < c.nnarrow; ++part) {
        const CopyPart& p = c.narrow[part];
        for (unsigned i = threadIdx.x * 4; i < p.bytes; i += COPY_THREADS * 4)
          *reinterpret_cast<uint32_t*>(p.at + size_t(to) * p.bytes + i) = *reinterpret_cast<const uint32_t*>(p.at + size_t(from) * p.bytes + i);
      }
  }
}

// The caches have `pages` pages each.
int copy_pages(const fv_kv* const* caches, size_t ncaches, size_t pages, cudaStream_t s, const int32_t* src, const int32_t* dst, size_t n, const int32_t* count,
               int32_t* map, int32_t* refs) {
  if (n == 0 || pages == 0) return FV_OK;
  for (size_t first = 0; first < ncaches || (map && first == 0); first += COPY_CACHES) {
    Copy c = {};
    for (size_t j = first; j < ncaches && j < first + COPY_CACHES; ++j) {
      const fv_kv* kv = caches[j];
      const size_t rows = size_t(kv->heads) * kv->page_size, row = kv_row_bytes(kv), scale = kv_scale_bytes(kv), bounds = size_t(kv->heads) * 2 * kv->dim;
      void* const at[COPY_PARTS] = {kv->k, kv->v, kv->bounds, kv->bound_codes, kv->k_scale, kv->v_scale, kv->bound_scale};
      const size_t bytes[COPY_PARTS] = {rows * row, rows * row, 2 * bounds, bounds, rows * scale, rows * scale, 4 * size_t(kv->heads)};
      for (int i = 0; i < COPY_PARTS; ++i) {
        if (bytes[i] == 0) continue;
        if (bytes[i] >= size_t(1) << 31) return fail(FV_ERR_UNSUPPORTED, "copies of pages: a page of 2 GB or more");
        if (kv_aligned(at[i], 16) && bytes[i] % 16 == 0) {
          c.wide[c.nwide++] = {static_cast<unsigned char*>(at[i]), unsigned(bytes[i]), c.pieces};
          c.pieces += unsigned(bytes[i] / 16);
        } else {
          c.narrow[c.nnarrow++] = {static_cast<unsigned char*>(at[i]), unsigned(bytes[i]), 0};
        }
      }
    }
    c.slices = (c.pieces + COPY_SLICE / 16 - 1) / (COPY_SLICE / 16);
    c.src = src, c.dst = dst, c.count = count, c.n = (long long)(n), c.pages = unsigned(pages);
    if (first == 0) c.map = map, c.refs = refs;
    const size_t items = n * (c.slices ? c.slices : 1), most = 148 * 16;
    const unsigned ctas = unsigned(items < most ? items : most);
    if (c.pieces && c.pieces < COPY_SLICE / 64) pages_copy_kernel<true><<<ctas, COPY_THREADS, 0, s>>>(c);
    else pages_copy_kernel<false><<<ctas, COPY_THREADS, 0, s>>>(c);
    FV_CUDA(cudaGetLastError());
  }
  return FV_OK;
}

int pages_check(const fv_pages* p, const std::string& w) {
  if (!p) return fail(FV_ERR_ARG, w + ": NULL pages");
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
    return fail(FV_ERR_UNSUPPORTED, w + ": page_size is 16, 32, 64 or 128");
  if (p->pages > size_t(INT_MAX) - 2 * PAGES_WINDOW) return fail(FV_ERR_UNSUPPORTED, w + ": pages does not fit 31 bits");
  if (p->device < 0) return fail(FV_ERR_ARG, w + ": device index out of range");
  if (p->pages && !p->refs) return fail(FV_ERR_ARG, w + ": NULL refs");
  if (!kv_aligned(p->refs, 4)) return fail(FV_ERR_ARG, w + ": refs does not begin on 4 bytes");
  return FV_OK;
}
int table_check(const fv_pages* p, const fv_table* t, const std::string& w) {
  if (!t) return fail(FV_ERR_ARG, w + ": NULL table");
  if (t->nseq > size_t(INT_MAX) / 8 || t->width > size_t(1) << 24 || t->stride > size_t(1) << 40) return fail(FV_ERR_UNSUPPORTED, w + ": nseq or width is too large");
  if (t->width > size_t(INT_MAX) / p->page_size) return fail(FV_ERR_UNSUPPORTED, w + ": positions in the table's last block leave 31 bits");
  if (t->nseq && t->width && !t->table) return fail(FV_ERR_ARG, w + ": NULL table");
  if (t->nseq > 1 && t->stride < t->width) return fail(FV_ERR_ARG, w + ": rows of the table overlap");
  if (!kv_aligned(t->table, 4)) return fail(FV_ERR_ARG, w + ": table does not begin on 4 bytes");
  return FV_OK;
}
// Whether an entry lies in both.  Rows of a table do not overlap one another.
bool tables_meet(const fv_table* a, const fv_table* b) {
  if (!a->nseq || !a->width || !b->nseq || !b->width) return false;
  using wide = __int128;  // strides of tables that cannot be are not looked at closer
  const wide step_a = a->nseq > 1 ? a->stride : 0, step_b = b->nseq > 1 ? b->stride : 0, width_a = a->width, width_b = b->width;
  const wide begin = (wide(reinterpret_cast<uintptr_t>(a->table)) - wide(reinterpret_cast<uintptr_t>(b->table))) / 4;  // of a, in b
  if (begin >= (b->nseq - 1) * step_b + width_b || begin + (a->nseq - 1) * step_a + width_a <= 0) return false;
  for (size_t i = 0; i < a->nseq; ++i) {
    const wide row = begin + i * step_a;
    wide j = step_b && row > width_b ? (row - width_b) / step_b : 0;
    for (; j < wide(b->nseq) && j * step_b < row + width_a; ++j)
      if (row < j * step_b + width_b) return true;
  }
  return false;
}
int caches_check(const fv_pages* p, const fv_kv* const* caches, size_t n, const char* who) {
  const std::string w(who);
  if (n && !caches) return fail(FV_ERR_ARG, w + ": NULL caches");
  const fv_kv_batch none = {};
  for (size_t i = 0; i < n; ++i) {
    FV_TRY(kv_check(caches[i], &none, who));
    if (caches[i]->device != p->device || caches[i]->pages != p->pages || caches[i]->page_size != p->page_size)
      return fail(FV_ERR_ARG, w + ": a cache has other pages, or is on another device");
  }
  return FV_OK;
}
Pages pages_of(const fv_pages* p) { return Pages{p->refs, int(p->pages), __builtin_ctz(p->page_size)}; }
Table table_of(const fv_table* t) { return Table{t->table, t->stride, int(t->width), int(t->nseq)}; }
dim3 table_grid(const fv_table* t) { return dim3(unsigned((t->width + 255) / 256), unsigned(t->nseq < 65535 ? t->nseq : 65535)); }

// pages that a call can give or move
size_t most_pages(const fv_pages* p, const fv_table* t) {
  const size_t entries = t->nseq * t->width;
  return entries < p->pages ? entries : p->pages;
}

}  // namespace
}  // namespace fv

extern "C" int fv_kv_copy_pages_dev(const fv_kv* kv, void* stream, const int32_t* src, const int32_t* dst, size_t n, const int32_t* count) {
  const fv_kv_batch none = {};
  FV_TRY(fv::kv_check(kv, &none, "fv_kv_copy_pages_dev"));
  if (n == 0 || kv->pages == 0) return FV_OK;
  if (n > size_t(INT_MAX)) return fv::fail(FV_ERR_UNSUPPORTED, "fv_kv_copy_pages_dev: n does not fit 31 bits");
  if (!src || !dst) return fv::fail(FV_ERR_ARG, "fv_kv_copy_pages_dev: NULL src or dst");
  if (!fv::kv_aligned(src, 4) || !fv::kv_aligned(dst, 4) || !fv::kv_aligned(count, 4)) return fv::fail(FV_ERR_ARG, "fv_kv_copy_pages_dev: src, dst or count does not begin on 4 bytes");
  fv::DeviceGuard g(kv->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  return fv::copy_pages(&kv, 1, kv->pages, static_cast<cudaStream_t>(stream), src, dst, n, count, nullptr, nullptr);
}

extern "C" int fv_pages_fork_dev(const fv_pages* p, void* stream, const fv_table* from, const int32_t* lens, const int32_t* parents, const fv_table* out) {
  const char* w = "fv_pages_fork_dev";
  FV_TRY(fv::pages_check(p, w));
  FV_TRY(fv::table_check(p, from, w));
  FV_TRY(fv::table_check(p, out, w));
  if (out->nseq == 0 || out->width == 0) return FV_OK;
  if (!parents || !fv::kv_aligned(parents, 4) || !fv::kv_aligned(lens, 4)) return fv::fail(FV_ERR_ARG, std::string(w) + ": parents is not there, or it or lens does not begin on 4 bytes");
  if (from->table == out->table || fv::tables_meet(from, out)) return fv::fail(FV_ERR_ARG, std::string(w) + ": out shares entries with the table");
  fv::DeviceGuard g(p->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  fv::pages_fork_kernel<<<fv::table_grid(out), 256, 0, static_cast<cudaStream_t>(stream)>>>(fv::pages_of(p), fv::table_of(from), lens, parents, fv::table_of(out));
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

extern "C" int fv_pages_free_dev(const fv_pages* p, void* stream, const fv_table* t, const int32_t* lens) {
  const char* w = "fv_pages_free_dev";
  FV_TRY(fv::pages_check(p, w));
  FV_TRY(fv::table_check(p, t, w));
  if (!fv::kv_aligned(lens, 4)) return fv::fail(FV_ERR_ARG, std::string(w) + ": lens does not begin on 4 bytes");
  if (t->nseq == 0 || t->width == 0) return FV_OK;
  fv::DeviceGuard g(p->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  fv::pages_free_kernel<<<fv::table_grid(t), 256, 0, static_cast<cudaStream_t>(stream)>>>(fv::pages_of(p), fv::table_of(t), lens);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

// work: the number of copies, where sequences' entries begin, the free pages, sources and places of copies
extern "C" size_t fv_pages_extend_work(const fv_pages* p, const fv_table* t) {
  if (!p || !t) return 0;
  return 4 * (4 + (t->nseq + 4) / 4 * 4 + 3 * ((fv::most_pages(p, t) + 3) / 4 * 4));
}

extern "C" int fv_pages_extend_dev(const fv_pages* p, void* stream, const fv_kv* const* caches, size_t ncaches, const fv_table* t, const int32_t* lens,
                                   const int32_t* more, int32_t* missing, void* work, size_t work_bytes) {
  const char* w = "fv_pages_extend_dev";
  FV_TRY(fv::pages_check(p, w));
  FV_TRY(fv::table_check(p, t, w));
  FV_TRY(fv::caches_check(p, caches, ncaches, w));
  if (t->nseq && (!lens || !more)) return fv::fail(FV_ERR_ARG, std::string(w) + ": NULL lens or more");
  if (!missing || !fv::kv_aligned(missing, 4) || !fv::kv_aligned(lens, 4) || !fv::kv_aligned(more, 4))
    return fv::fail(FV_ERR_ARG, std::string(w) + ": missing is not there, or it, lens or more does not begin on 4 bytes");
  if (!work || !fv::kv_aligned(work, 16) || work_bytes < fv_pages_extend_work(p, t)) return fv::fail(FV_ERR_ARG, std::string(w) + ": work is smaller than fv_pages_extend_work says, or does not begin on 16 bytes");
  if (t->nseq * t->width > size_t(1) << 30) return fv::fail(FV_ERR_UNSUPPORTED, std::string(w) + ": the table has more than 2^30 entries");
  fv::DeviceGuard g(p->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t most = fv::most_pages(p, t), room = (most + 3) / 4 * 4;
  int32_t* const at = static_cast<int32_t*>(work);
  fv::Extend x{lens, more, missing, at, at + 4, nullptr, nullptr, nullptr};
  x.free = x.before + (t->nseq + 4) / 4 * 4, x.src = x.free + room, x.dst = x.src + room;
  fv::pages_extend_kernel<<<1, fv::PAGES_THREADS, 0, s>>>(fv::pages_of(p), fv::table_of(t), x);
  FV_CUDA(cudaGetLastError());
  return fv::copy_pages(caches, ncaches, p->pages, s, x.src, x.dst, most, x.count, nullptr, nullptr);
}

// work: the number of moves, their sources and places, and the windows' counts
static size_t page_windows(const fv_pages* p) { return p->pages > fv::PAGES_WINDOW ? (p->pages + fv::PAGES_WINDOW - 1) / fv::PAGES_WINDOW : 1; }
extern "C" size_t fv_pages_compact_work(const fv_pages* p) { return p ? 4 * (4 + 2 * ((p->pages + 3) / 4 * 4) + (page_windows(p) + 3) / 4 * 4) : 0; }

extern "C" int fv_pages_compact_dev(const fv_pages* p, void* stream, const fv_kv* const* caches, size_t ncaches, int32_t* used, int32_t* map, void* work, size_t work_bytes) {
  const char* w = "fv_pages_compact_dev";
  FV_TRY(fv::pages_check(p, w));
  FV_TRY(fv::caches_check(p, caches, ncaches, w));
  if (!used || (!map && p->pages) || !fv::kv_aligned(used, 4) || !fv::kv_aligned(map, 4)) return fv::fail(FV_ERR_ARG, std::string(w) + ": used or map is not there or does not begin on 4 bytes");
  if (!work || !fv::kv_aligned(work, 16) || work_bytes < fv_pages_compact_work(p)) return fv::fail(FV_ERR_ARG, std::string(w) + ": work is smaller than fv_pages_compact_work says, or does not begin on 16 bytes");
  fv::DeviceGuard g(p->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t* const at = static_cast<int32_t*>(work);
  int32_t *const src = at + 4, *const dst = src + (p->pages + 3) / 4 * 4, *const counts = dst + (p->pages + 3) / 4 * 4;
  const unsigned windows = unsigned(page_windows(p));
  if (windows > 1) {
    fv::pages_count_kernel<<<windows, fv::PAGES_THREADS, 0, s>>>(fv::pages_of(p), counts);
    FV_CUDA(cudaGetLastError());
  }
  fv::pages_compact_kernel<<<windows, fv::PAGES_THREADS, 0, s>>>(fv::pages_of(p), counts, map, used, at, src, dst);
  FV_CUDA(cudaGetLastError());
  return fv::copy_pages(caches, ncaches, p->pages, s, src, dst, p->pages, at, map, p->refs);
}

extern "C" int fv_pages_remap_dev(const fv_pages* p, void* stream, const int32_t* map, const fv_table* t) {
  const char* w = "fv_pages_remap_dev";
  FV_TRY(fv::pages_check(p, w));
  FV_TRY(fv::table_check(p, t, w));
  if (t->nseq == 0 || t->width == 0 || p->pages == 0) return FV_OK;
  if (!map || !fv::kv_aligned(map, 4)) return fv::fail(FV_ERR_ARG, std::string(w) + ": map is not there or does not begin on 4 bytes");
  fv::DeviceGuard g(p->device);
  if (!g.ok) return fv::fail(FV_ERR_CUDA, "cudaSetDevice failed (there is no CPU path)");
  fv::pages_remap_kernel<<<fv::table_grid(t), 256, 0, static_cast<cudaStream_t>(stream)>>>(map, int(p->pages), fv::table_of(t));
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}
