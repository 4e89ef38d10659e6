// Block tables and slot maps of a batch, built on the GPU from its requests'
// lengths, and the way back: pages given up when sequences shrink or end.
//
// With page size S, c_b tokens cached and n_b new ones, sequence b holds
// have_b = ceil(c_b / S) pages and needs need_b = ceil((c_b + n_b) / S). The
// call's new pages are numbered k sequence by sequence; page k is
// free[count - 1 - k] (the free list is a stack). Token i of the packed batch
// belongs to the sequence whose query_start interval holds i; its position is
// c_b + i - query_start[b] and its slot page * S + position % S.
//
// Both kernels are bound by launch latency except for large prompts, where
// extend writes 16 bytes a token. So every CTA of extend repeats the scan over
// the batch and its checks (B lengths and every id to be popped, from L2; no
// message between CTAs, one launch) and then writes its own stretch of tokens
// and pages; page k comes straight from the free stack, never from a table
// entry that another CTA writes. Truncate runs as one cluster of up to 8 CTAs,
// which agree through shared memory on whether an entry is bad before they push
// any (giving back the 21,000 pages of 64 prompts: 10 us, against 19 with one
// CTA; a million pages: 68 us); with reference counts shared pages need steps
// in order, which one CTA takes.
#include <cooperative_groups.h>

#include "common.cuh"
#include "tmap.cuh"

namespace hx {
namespace pg {

namespace cg = cooperative_groups;

constexpr int NT = 512;          // threads of a CTA of extend
constexpr int NTT = 1024;        // threads of truncate's CTA
constexpr int MAXB = 16384;      // sequences a call takes (their prefix sums sit in shared memory)
constexpr size_t kSmallSmem = 40 * 1024;  // dynamic shared memory asked for without more ado (48 KB with the static)
constexpr int kMostRows = 1 << 30;  // tokens, and new pages, of an extend: a thread's next one still fits 32 bits
constexpr int kTokensPerCta = 2048;
constexpr int kMostDropped = (1 << 29) - 1;  // entries a truncate drops (their numbers mark pages, below 3 * -2^29)
constexpr int kCluster = 8;      // CTAs of truncate, at most
constexpr int kHeld = 8;         // entries a thread of truncate holds in registers: a block of 256 a warp

// Inclusive scan of (a, b) over the block's threads; totals to every thread.
template <int N>
HX_DEVINL void block_scan2(long long& a, long long& b, long long& ta, long long& tb, long long (*ws)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  if (lane == 31) ws[warp][0] = a, ws[warp][1] = b;
  __syncthreads();
  long long pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll 4
  for (int w = 0; w < N / 32; ++w) {
    if (w < warp) pa += ws[w][0], pb += ws[w][1];
    ta += ws[w][0], tb += ws[w][1];
  }
  a += pa;
  b += pb;
  __syncthreads();
}

// Largest b with first[b] <= i (first ascending, first[0] = 0): the sequence
// holding item i; sequences without items are passed over.
HX_DEVINL int find_row(const int* first, int B, int i) {
  int lo = 0, hi = B;  // first[lo] <= i, and hi == B or first[hi] > i
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

HX_DEVINL int pages_of(long long tokens, int S) { return (int)((tokens + S - 1) / S); }

struct ExtendParams {
  int32_t* table;
  int64_t stride;
  int B, W, S;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* free_pages;
  int64_t free_cap;
  const int32_t* free_count;
  int32_t* refs;
  int num_pages;
  int32_t* query_start;
  int32_t* seq_lens;
  int64_t* slots;
  int64_t* positions;
  int num_tokens;
  int32_t* free_out;
  uint32_t* err;
};

__global__ void __launch_bounds__(NT) extend_kernel(const ExtendParams p) {
  extern __shared__ int smem[];
  int* qs = smem;            // first token of each sequence
  int* pf = smem + p.B;      // first new page of each sequence
  __shared__ long long ws[NT / 32][2];
  __shared__ uint32_t bad;
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0u;
  __syncthreads();
  // ---- prefix sums of new tokens and new pages, and the checks: the same in every CTA
  const int per = (p.B + NT - 1) / NT, b0 = tid * per, b1 = min(p.B, b0 + per);
  long long st = 0, sp = 0;
  uint32_t mine = 0u;
  for (int b = b0; b < b1; ++b) {
    const long long c = p.cached[b], n = p.fresh[b];
    if (c < 0 || n < 0 || c + n > 0x7fffffffll || (c + n + p.S - 1) / p.S > p.W) {
      mine |= HX_DEV_ERR_BOUNDS;
      continue;
    }
    st += n;
    sp += pages_of(c + n, p.S) - pages_of(c, p.S);
    if (n > 0 && c % p.S != 0) {  // the tokens begin in a page the sequence holds: nobody else may read it
      const int page = p.table[b * p.stride + c / p.S];
      if (page < 0 || page >= p.num_pages) mine |= HX_DEV_ERR_BOUNDS;
      else if (p.refs && p.refs[page] > 1) mine |= HX_DEV_ERR_SHARED;
    }
  }
  long long it = st, ip = sp, tt, tp;
  block_scan2<NT>(it, ip, tt, tp, ws);
  const long long count = *p.free_count;
  if (count >= 0 && count <= p.free_cap && tp <= count && tp <= kMostRows) {  // ids to be popped: all are looked at before any is handed out
    const int n = (int)tp;
#pragma unroll 4
    for (int k = tid; k < n; k += NT) {
      const int page = p.free_pages[count - 1 - k];
      if (page < 0 || page >= p.num_pages) mine |= HX_DEV_ERR_BOUNDS;
    }
  }
  if (mine) atomicOr(&bad, mine);
  if (tid == 0) {
    if (tt > p.num_tokens || count < 0 || count > p.free_cap || tp > kMostRows) atomicOr(&bad, HX_DEV_ERR_BOUNDS);
    else if (tp > count) atomicOr(&bad, HX_DEV_ERR_PAGES);
  }
  __syncthreads();
  const uint32_t fail = bad;
  if (!fail) {
    int t = (int)(it - st), q = (int)(ip - sp);
    for (int b = b0; b < b1; ++b) {
      const int c = p.cached[b], n = p.fresh[b];
      qs[b] = t;
      pf[b] = q;
      t += n;
      q += pages_of((long long)c + n, p.S) - pages_of(c, p.S);
    }
  }
  __syncthreads();
  const int total = fail ? 0 : (int)tt, fresh_pages = fail ? 0 : (int)tp;
  if (blockIdx.x == 0) {
    for (int b = tid; b < p.B; b += NT) {
      p.query_start[b] = fail ? 0 : qs[b];
      p.seq_lens[b] = p.cached[b] + (fail ? 0 : p.fresh[b]);
    }
    if (tid == 0) {
      p.query_start[p.B] = total;
      *p.free_out = (int32_t)(count - fresh_pages);
      if (fail) set_err(p.err, fail);
    }
  }
  // ---- new pages: table entries and reference counts
  for (int k = blockIdx.x * NT + tid; k < fresh_pages; k += gridDim.x * NT) {
    const int b = find_row(pf, p.B, k);
    const int j = pages_of(p.cached[b], p.S) + k - pf[b];
    const int page = p.free_pages[count - 1 - k];
    p.table[(int64_t)b * p.stride + j] = page;
    if (p.refs && page >= 0 && page < p.num_pages) p.refs[page] = 1;  // (the stack may not change meanwhile)
  }
  // ---- tokens: slot and position; rows past the batch get slot -1 (skipped by the pack) and position 0
  for (int i = blockIdx.x * NT + tid; i < p.num_tokens; i += gridDim.x * NT) {
    int64_t slot = -1, pos = 0;
    if (i < total) {
      const int b = find_row(qs, p.B, i);
      const int c = p.cached[b];
      pos = (int64_t)c + i - qs[b];
      const int j = (int)(pos / p.S), have = pages_of(c, p.S);
      const int page = j < have ? p.table[(int64_t)b * p.stride + j] : p.free_pages[count - 1 - (pf[b] + j - have)];
      slot = (int64_t)page * p.S + pos % p.S;
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
}

struct TruncateParams {
  const int32_t* table;
  int64_t stride;
  int B, W, S;
  const int32_t* lens;
  const int32_t* keep;
  int32_t* free_pages;
  int64_t free_cap;
  const int32_t* free_count;
  int32_t* refs;
  int num_pages;
  int32_t* lens_out;
  int32_t* free_out;
  uint32_t* err;
};

// Drops pages [ceil(keep / S), ceil(len / S)) of every sequence. Dropped
// entries are numbered k sequence by sequence and pushed in reverse, so that
// truncating what extend just added leaves the stack as it was. An entry
// outside the pool is an error and gives nothing back; the others do. With
// reference counts an entry takes one reference; a page whose last reference
// goes is pushed once, at the place of the call's last entry naming it (the
// order does not depend on which thread's atomic came first):
//   1  each entry takes a reference by compare-and-swap; the one that takes the
//      last leaves kGone in place of 0. An entry that comes later finds none:
//      an error, counted by one less than kGone so that step 1 can be undone
//      (each entry adds one again, which leaves kGone + the old count), as it
//      is where the stack has no room for the pages freed. An entry of a page
//      that had none is an error and changes nothing
//   2  entries of pages at kGone or below lower it to INT_MIN + N - 1 - k
//      (atomicMin: the last entry's mark stays)
//   3  the entry that finds its own mark pushes the page; the mark becomes 0
__global__ void __launch_bounds__(NTT) truncate_kernel(const TruncateParams p) {
  extern __shared__ int smem[];
  int* pf = smem;          // first dropped entry of each sequence
  int* col = smem + p.B;   // table column of entry k: col + k
  __shared__ long long ws[NTT / 32][2];
  __shared__ uint32_t bad;
  __shared__ int freed, run;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const cg::cluster_group cluster = cg::this_cluster();  // the whole grid
  if (tid == 0) bad = 0u, freed = 0, run = 0;
  __syncthreads();
  const int per = (p.B + NTT - 1) / NTT, b0 = tid * per, b1 = min(p.B, b0 + per);
  long long sp = 0, dummy = 0, tp, td;
  uint32_t mine = 0u;
  for (int b = b0; b < b1; ++b) {
    const long long n = p.lens[b], k = max(0, min(p.keep[b], p.lens[b]));
    if (n < 0 || (n + p.S - 1) / p.S > p.W) mine = HX_DEV_ERR_BOUNDS;
    else sp += pages_of(n, p.S) - pages_of(k, p.S);
  }
  long long ip = sp;
  block_scan2<NTT>(ip, dummy, tp, td, ws);
  const long long count = *p.free_count;
  if (mine) atomicOr(&bad, mine);
  if (tid == 0 && (count < 0 || count > p.free_cap || tp > kMostDropped || (!p.refs && count + tp > p.free_cap)))
    atomicOr(&bad, HX_DEV_ERR_BOUNDS);
  __syncthreads();
  if (bad) {  // nothing is given back
    if (blockIdx.x == 0) {
      for (int b = tid; b < p.B; b += NTT) p.lens_out[b] = p.lens[b];
      if (tid == 0) {
        *p.free_out = (int32_t)count;
        set_err(p.err, bad);
      }
    }
    return;
  }
  if (gridDim.x > 1) cluster.barrier_arrive();  // this CTA's shared memory may be written
  int q = (int)(ip - sp);
  for (int b = b0; b < b1; ++b) {
    const int kept = pages_of(max(0, min(p.keep[b], p.lens[b])), p.S);
    pf[b] = q;
    col[b] = kept - q;
    q += pages_of(p.lens[b], p.S) - kept;
  }
  __syncthreads();
  const int total = (int)tp;
  auto page_at = [&](int b, int k) -> int {  // entry k, of row b
    const int page = p.table[(int64_t)b * p.stride + col[b] + k];
    if (page >= 0 && page < p.num_pages) return page;
    set_err(p.err, HX_DEV_ERR_BOUNDS);
    return -1;
  };
  auto entry = [&](int k) { return page_at(find_row(pf, p.B, k), k); };
  constexpr int kGone = -(1 << 30);
  auto gone = [&](int refs) { return refs > kGone + kGone / 2 && refs < kGone / 2; };
  if (!p.refs) {
    // a warp has a run of consecutive entries, so that a row is searched for once, not for every entry
    const int warps = (int)gridDim.x * (NTT / 32), part = (total + 32 * warps - 1) / (32 * warps) * 32;
    const int lo = min(total, ((int)blockIdx.x * (NTT / 32) + warp) * part), hi = min(total, lo + part);
    int row = 0, held[kHeld];
    auto load = [&](int k0) {  // raw entries k0 + lane, + 32, ...: all on their way before one is looked at
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const int k = k0 + lane + 32 * u;
        held[u] = 0;
        if (k < hi) {
          if (row + 1 < p.B && pf[row + 1] <= k) row = find_row(pf, p.B, k);
          held[u] = p.table[(int64_t)row * p.stride + col[row] + k];
        }
      }
    };
    auto bad_id = [&](int page) { return page < 0 || page >= p.num_pages; };
    bool hole = false;  // an entry outside the pool
    int at = lo;
    for (int k0 = lo; k0 < hi; k0 += 32 * kHeld) {
      load(at = k0);
#pragma unroll
      for (int u = 0; u < kHeld; ++u) hole |= k0 + lane + 32 * u < hi && bad_id(held[u]);
    }
    if (hole) set_err(p.err, HX_DEV_ERR_BOUNDS);
    if (gridDim.x == 1) {
      hole = __syncthreads_or(hole);
    } else {  // every CTA is told
      cluster.barrier_wait();
      if (hole)
        for (unsigned r = 0; r < gridDim.x; ++r) *cluster.map_shared_rank(&run, r) = 1;
      cluster.sync();
      hole = run != 0;
    }
    int good = total;
    if (!hole) {
      for (int k0 = at;;) {  // the last block of entries is still held, the others are loaded again
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
          const int k = k0 + lane + 32 * u;
          if (k < hi) p.free_pages[count + total - 1 - k] = held[u];
        }
        if (k0 == lo) break;
        k0 -= 32 * kHeld;
        row = 0;
        load(k0);
      }
      if (blockIdx.x != 0) return;
    } else {  // an error: one CTA pushes the good ones without a gap
      if (blockIdx.x != 0) return;
      good = 0;
      for (int k0 = 0; k0 < total; k0 += NTT) good += __syncthreads_count(k0 + tid < total && entry(k0 + tid) >= 0);
      int before = 0;
      for (int k0 = 0; k0 < total; k0 += NTT) {
        const int k = k0 + tid;
        const int page = k < total ? entry(k) : -1;
        const uint32_t m = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) ws[warp][0] = __popc(m);
        __syncthreads();
        int rank = before + __popc(m & ((1u << lane) - 1u));
        for (int w = 0; w < NTT / 32; ++w) {
          if (w < warp) rank += (int)ws[w][0];
          before += (int)ws[w][0];
        }
        if (page >= 0) p.free_pages[count + good - 1 - rank] = page;
        __syncthreads();
      }
    }
    if (tid == 0) freed = good;
    __syncthreads();
  } else {
    int here = 0;
    for (int k = tid; k < total; k += NTT) {
      const int page = entry(k);
      if (page < 0) continue;
      int old = p.refs[page];
      while (old > 0 || gone(old)) {
        const int seen = atomicCAS(p.refs + page, old, old == 1 ? kGone : old - 1);
        if (seen == old) break;
        old = seen;
      }
      if (old <= 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
      here += old == 1;
    }
    if (here) atomicAdd(&freed, here);
    __syncthreads();
    const int n_free = freed;
    if (count + n_free > p.free_cap) {  // no room: every reference goes back, and nothing has happened
      for (int k = tid; k < total; k += NTT) {
        const int page = entry(k);
        if (page < 0) continue;
        const int now = __ldcg(p.refs + page);
        if (now > 0 || gone(now)) atomicAdd(p.refs + page, 1);
      }
      __syncthreads();
      for (int k = tid; k < total; k += NTT) {  // kGone + what there was
        const int page = entry(k);
        const int now = page < 0 ? 0 : __ldcg(p.refs + page);
        if (gone(now)) atomicCAS(p.refs + page, now, now - kGone);
      }
      for (int b = tid; b < p.B; b += NTT) p.lens_out[b] = p.lens[b];
      if (tid == 0) {
        *p.free_out = (int32_t)count;
        set_err(p.err, HX_DEV_ERR_BOUNDS);
      }
      return;
    }
    auto mark = [&](int k) { return (int)0x80000000 + (total - 1 - k); };  // below all that gone() takes
    for (int k = tid; k < total; k += NTT) {
      const int page = entry(k);
      if (page >= 0 && __ldcg(p.refs + page) < kGone / 2) atomicMin(p.refs + page, mark(k));
    }
    __syncthreads();
    for (int k0 = 0; k0 < total; k0 += NTT) {  // ranks by a running block scan, chunk by chunk
      const int k = k0 + tid;
      const int page = k < total ? entry(k) : -1;
      const bool mine_now = page >= 0 && __ldcg(p.refs + page) == mark(k);
      const uint32_t m = __ballot_sync(0xffffffffu, mine_now);
      if (lane == 0) ws[warp][0] = __popc(m);
      __syncthreads();
      int before = run, all = 0;
      for (int w = 0; w < NTT / 32; ++w) {
        if (w < warp) before += (int)ws[w][0];
        all += (int)ws[w][0];
      }
      if (mine_now) {
        const int rank = before + __popc(m & ((1u << lane) - 1u));
        if (rank < n_free) p.free_pages[count + n_free - 1 - rank] = page;  // (more: counts that were far below 0)
        p.refs[page] = 0;
      }
      __syncthreads();
      if (tid == 0) run += all;
      __syncthreads();
    }
  }
  for (int b = tid; b < p.B; b += NTT) p.lens_out[b] = max(0, min(p.keep[b], p.lens[b]));
  if (tid == 0) *p.free_out = (int32_t)(count + freed);
}

// Empties pages[lo .. hi) (lo, hi read on the device) as hx_pool_reset_pages does.
__global__ void reset_range_kernel(hx_pool_layer pool, const int32_t* pages, int64_t cap, const int32_t* lo_p,
                                   const int32_t* hi_p, uint32_t* err) {
  const int h = blockIdx.y, D = pool.head_size;
  const int64_t lo = *lo_p, hi = *hi_p;
  if (lo < 0 || hi > cap) {
    if (threadIdx.x == 0) set_err(err, HX_DEV_ERR_BOUNDS);
    return;
  }
  for (int64_t i = lo + blockIdx.x; i < hi; i += gridDim.x) {
    const int pg = pages[i];
    if (pg < 0 || pg >= pool.num_blocks) {
      if (threadIdx.x == 0) set_err(err, HX_DEV_ERR_BOUNDS);
      continue;
    }
    uint16_t* st = pool.stats + ((int64_t)h * pool.num_blocks + pg) * 2 * D;
    for (int d = threadIdx.x; d < 2 * D; d += blockDim.x) st[d] = d < D ? 0x7C00u : 0xFC00u;
    if (threadIdx.x < 2) {
      uint32_t* dr = pool.dir + (((int64_t)h * pool.num_blocks + pg) * 2 + threadIdx.x) * 4;
      dr[2] = 0;
      dr[3] = 0;
    }
  }
}

}  // namespace pg
}  // namespace hx

using namespace hx;

extern "C" {

HX_API int hx_tables_extend(void* stream, int32_t* block_table, int64_t bt_stride, int32_t B, int32_t max_pages,
                            int32_t page_size, const int32_t* cached_lens, const int32_t* new_tokens,
                            const int32_t* free_pages, int64_t free_capacity, const int32_t* free_count,
                            int32_t* page_refs, int32_t num_pages, int32_t* query_start, int32_t* seq_lens,
                            int64_t* slot_mapping, int64_t* positions, int32_t num_tokens, int32_t* free_count_out,
                            uint32_t* dev_err) {
  if (B < 0 || max_pages < 0 || page_size < 1 || num_pages < 0 || num_tokens < 0 || free_capacity < 0)
    return HX_ERR_ARG;
  if (!query_start || !free_count || !free_count_out || free_count == free_count_out) return HX_ERR_ARG;
  if (B > 0 && (!block_table || !cached_lens || !new_tokens || !seq_lens || bt_stride < max_pages)) return HX_ERR_ARG;
  if (B > 0 && (seq_lens == cached_lens || seq_lens == new_tokens)) return HX_ERR_ARG;
  if ((num_tokens > 0 && (!slot_mapping || !positions)) || (free_capacity > 0 && !free_pages)) return HX_ERR_ARG;
  if (B > pg::MAXB || num_tokens > pg::kMostRows) return HX_ERR_UNSUPPORTED;
  pg::ExtendParams p{block_table, bt_stride,   B,        max_pages,   page_size, cached_lens,  new_tokens,
                     free_pages,  free_capacity, free_count, page_refs, num_pages, query_start, seq_lens,
                     slot_mapping, positions,   num_tokens, free_count_out, dev_err};
  const size_t smem = (size_t)2 * (B > 0 ? B : 1) * sizeof(int);
  static unsigned long long done = 0;
  if (smem > pg::kSmallSmem && !allow_smem(pg::extend_kernel, 2 * pg::MAXB * (int)sizeof(int), done)) return HX_ERR_LAUNCH;
  int grid = (num_tokens + pg::kTokensPerCta - 1) / pg::kTokensPerCta;
  grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
  pg::extend_kernel<<<grid, pg::NT, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  HX_LAUNCH_CHECK();
  return HX_OK;
}

HX_API int hx_tables_truncate(void* stream, const int32_t* block_table, int64_t bt_stride, int32_t B,
                              int32_t max_pages, int32_t page_size, const int32_t* seq_lens,
                              const int32_t* keep_lens, int32_t* free_pages, int64_t free_capacity,
                              const int32_t* free_count, int32_t* page_refs, int32_t num_pages, int32_t* seq_lens_out,
                              int32_t* free_count_out, uint32_t* dev_err) {
  if (B < 0 || max_pages < 0 || page_size < 1 || num_pages < 0 || free_capacity < 0) return HX_ERR_ARG;
  if (!free_count || !free_count_out || (free_capacity > 0 && !free_pages)) return HX_ERR_ARG;
  if (B > 0 && (!block_table || !seq_lens || !keep_lens || !seq_lens_out || bt_stride < max_pages)) return HX_ERR_ARG;
  if (free_count == free_count_out || (B > 0 && (seq_lens == seq_lens_out || keep_lens == seq_lens_out))) return HX_ERR_ARG;
  if (B > pg::MAXB) return HX_ERR_UNSUPPORTED;
  pg::TruncateParams p{block_table, bt_stride,  B,         max_pages, page_size,    seq_lens,       keep_lens, free_pages,
                       free_capacity, free_count, page_refs, num_pages, seq_lens_out, free_count_out, dev_err};
  const size_t smem = (size_t)2 * (B > 0 ? B : 1) * sizeof(int);
  static unsigned long long done = 0;
  if (smem > pg::kSmallSmem && !allow_smem(pg::truncate_kernel, 2 * pg::MAXB * (int)sizeof(int), done)) return HX_ERR_LAUNCH;
  // B * max_pages entries at most: more CTAs from two to a thread of one CTA
  const unsigned grid = page_refs || (int64_t)B * max_pages <= 2 * pg::NTT ? 1u : (unsigned)pg::kCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(pg::NTT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = grid;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = grid > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, pg::truncate_kernel, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return HX_ERR_LAUNCH;
  }
  return HX_OK;
}

HX_API int hx_pool_reset_range(void* stream, const hx_pool_layer* pool, const int32_t* pages, int64_t capacity,
                               const int32_t* begin, const int32_t* end, uint32_t* dev_err) {
  if (!pool || !pages || !begin || !end || capacity < 0) return HX_ERR_ARG;
  if (!pool->stats || !pool->dir || pool->num_kv_heads < 1 || pool->num_kv_heads > 65535 || pool->head_size < 1)
    return HX_ERR_ARG;
  if (capacity == 0) return HX_OK;
  const int64_t gx = capacity < 592 ? capacity : 592;  // 4 blocks an SM, striding over the range
  pg::reset_range_kernel<<<dim3((unsigned)gx, pool->num_kv_heads), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      *pool, pages, capacity, begin, end, dev_err);
  HX_LAUNCH_CHECK();
  return HX_OK;
}

}  // extern "C"
