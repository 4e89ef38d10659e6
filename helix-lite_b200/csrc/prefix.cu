// Decode attention of a batch whose sequences share a long prefix of pool
// pages: the prefix is read and dequantised once for each block of query rows
// (two tiles of 128: 36 sequences at a group of 7), not for every sequence.
//
//   o_b = softmax over the sequence's tokens of (scale q_b . k_j) v_j,  the
//   first prefix_len tokens being the same pool pages for every sequence
//
// The query rows of a KV head (sequences x heads of the group) are the M side
// of a matrix product over each dequantised tile of 128 tokens (8 pages). A
// CTA (one an SM) takes work items of one KV head, one after another:
//   prefix  (block of two 128-row query tiles, split of the prefix): both tiles
//           use each dequantised key tile. A block with one tile only runs it
//           twice, on the even and on the odd key tiles
//   suffix  (sequence): the sequence's own pages, its G rows alone, again as two
//           streams of key tiles
// Each leaves unnormalised fp32 partials (m, l, O) per row; a second kernel joins
// a row's partials. Scores, m and l are fp32; P is rounded to fp16 once, as the
// matrix unit's operand (l keeps the unrounded values), and the output once. Roles in a CTA (25 warps):
//   0-7    two softmax warpgroups, a row a thread (as in the prompt kernel: S
//          and P in TMEM, the maximum moves only past 2^8)
//   8-15   K dequantisation: warp w turns page w of each tile into 16 rows of the
//          swizzled operand (per-channel level tables in shared memory, one
//          prmt-built address a code), outliers patched in
//   16-23  V dequantisation likewise: levels picked out of registers by prmt
//          (each token's own row before t_cal, the last row after it)
//   24     the query tiles and the matrix products (tcgen05.mma, one thread)
//
// What bounds it: at 8 sequences behind 1M tokens (nuq4, 409 us, 1.46 TB/s of
// codes, outlier lists and their records; fused.decode, which reads the prefix
// per sequence: 4,964) the shared-memory pipe (59 % for table lookups, operand
// stores and waits, 24 % more for the tensor core's operands) and issue slots
// (55 %) of 16 dequantising warps. At 64 sequences behind 32K (84 us) the softmax's two
// passes and the 64 suffixes. A suffix is one item, whatever its length: 1.6 us
// a key tile, so sequences much longer than the prefix are better served by
// fused.decode, which splits them.
#include "dequant.cuh"
#include "tcgen.cuh"
#include "tmap.cuh"

namespace hx {
namespace px {

constexpr int D = 128, S = 16, KT = 128, ROWS = 128, PAGES = KT / S;
constexpr int STAGES = 4;
constexpr int NTHREADS = 800;  // 25 warps: 72 registers a thread
constexpr int HALF = KT * 128;  // bytes of 128 rows of 64 fp16
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;

struct Smem {
  alignas(1024) uint8_t q[2][ROWS * D * 2];
  alignas(1024) uint8_t kv[STAGES][KT * D * 2];
  alignas(256) uint16_t klut[16 * D + 128];      // K tables, bank-spread (32 bytes of room after every 32 channels)
  alignas(256) uint32_t vpair[16];               // nuq2 V past t_cal: level pairs by code pair
  alignas(16) uint32_t vplane[8];                // nuq4 V past t_cal: byte planes
  alignas(16) uint8_t codes[2][PAGES][1024];     // each producer warp's next page (K, V)
  float2 ml[ROWS];                               // the second stream's (maximum, sum) of each row
  uint64_t q_full[2], kv_full[STAGES], kv_empty[STAGES], s_full[2], p_full[2], o_full[2], ml_full, ml_empty, drain;
  uint32_t tmem, abort;
  int row;                                       // the prefix's table row
};

struct Params {
  CUtensorMap mq;
  hx_pool_layer pool;
  hx_layer_scales sc;
  int B, G, TQ, RB, J;       // sequences, heads of a group, sequences a tile, row blocks, CTAs a head
  float c;                   // softmax scale * log2 e
  const int32_t* bt;
  int bt_stride;
  const int32_t* seq_lens;
  int prefix_pages, n_splits, vphys;
  float* part_o;             // (partials, B * H * G, D)
  float2* part_ml;           // (partials, B * H * G): maximum (exp2 domain), sum
  uint32_t* err;
};

HX_DEVINL uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A CTA's items: its split of the prefix, if it has one, then suffixes. j is the
// CTA's place among the J of its head; the first RB * n_splits have a split,
// and sequence b's suffix is CTA (RB * n_splits + b) mod J's, so that CTAs
// without a split take theirs first. Every role walks the items alike.
struct Item {
  int seq0, page0, pages, tokens, pidx, n;  // first sequence of the rows; pages [page0, page0 + pages) of table row trow
  int64_t trow;
  bool two, suffix;                         // two query tiles (else one tile, two streams of key tiles)
};

// row: the table row that the prefix is read from, -1 if no sequence holds the prefix.
HX_DEVINL bool get_item(const Params& p, int j, int row, int idx, Item& it) {
  const int pre = p.RB * p.n_splits, lead = j < pre ? 1 : 0;
  if (idx < lead) {
    const int rb = j % p.RB, split = j / p.RB;
    it.suffix = false;
    it.seq0 = rb * 2 * p.TQ;
    it.two = it.seq0 + p.TQ < p.B;
    const int nt = (p.prefix_pages + PAGES - 1) / PAGES;
    const int ta = (int)((int64_t)nt * split / p.n_splits), te = (int)((int64_t)nt * (split + 1) / p.n_splits);
    it.page0 = ta * PAGES;
    it.pages = row < 0 ? 0 : min(te * PAGES, p.prefix_pages) - it.page0;
    it.tokens = it.pages * S;
    it.pidx = split;
    it.trow = (int64_t)row * p.bt_stride;
  } else {
    const int first = j - pre % p.J;
    const int b = (first < 0 ? first + p.J : first) + (idx - lead) * p.J;
    if (b >= p.B) return false;
    const int len = p.seq_lens[b];
    it.suffix = true;
    it.two = false;
    it.seq0 = b;
    it.page0 = p.prefix_pages;
    it.tokens = len - p.prefix_pages * S;
    if (it.tokens < 0 || (len - 1) / S >= p.bt_stride) it.tokens = 0;  // the merge flags a bad length
    it.pages = (it.tokens + S - 1) / S;
    it.pidx = p.n_splits;
    it.trow = (int64_t)b * p.bt_stride;
  }
  it.n = (it.pages + PAGES - 1) / PAGES;
  return true;
}

// entry (token << 24 | channel << 16 | value) into the page's rows
HX_DEVINL void patch(uint32_t slab, uint32_t e, int valid, uint32_t* err) {
  const uint32_t tt = e >> 24, d = (e >> 16) & 0xFFu;
  if (tt >= (uint32_t)S || d >= (uint32_t)D) {
    set_err(err, HX_DEV_ERR_BOUNDS);
  } else if ((int)tt < valid) {
    const uint32_t off = (d >> 6) * HALF + tt * 128 + ((((d >> 3) & 7) ^ (tt & 7)) << 4) + (d & 7) * 2;
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(slab + off), "h"((uint16_t)(e & 0xFFFFu)) : "memory");
  }
}

// 16 levels for 16 2-bit codes from a 4-entry table held as byte planes (low, high) in registers
HX_DEVINL void crumbs_reg(uint32_t w, uint32_t lb, uint32_t hb, uint4& o0, uint4& o1) {
  const uint32_t e = w & 0x33333333u, d = (w >> 2) & 0x33333333u;  // codes 0, 2, .. 14 and 1, 3, .. 15 as selectors
  uint32_t o[8];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const uint32_t es = g ? e >> 16 : e, ds = g ? d >> 16 : d;
    const uint32_t le = prmt(lb, 0u, es & 0xFFFFu), he = prmt(hb, 0u, es & 0xFFFFu);
    const uint32_t lo = prmt(lb, 0u, ds & 0xFFFFu), ho = prmt(hb, 0u, ds & 0xFFFFu);
    const uint32_t e01 = prmt(le, he, 0x5140u), e23 = prmt(le, he, 0x7362u);
    const uint32_t d01 = prmt(lo, ho, 0x5140u), d23 = prmt(lo, ho, 0x7362u);
    o[4 * g] = prmt(e01, d01, 0x5410u);
    o[4 * g + 1] = prmt(e01, d01, 0x7632u);
    o[4 * g + 2] = prmt(e23, d23, 0x5410u);
    o[4 * g + 3] = prmt(e23, d23, 0x7632u);
  }
  o0 = make_uint4(o[0], o[1], o[2], o[3]);
  o1 = make_uint4(o[4], o[5], o[6], o[7]);
}

HX_DEVINL void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
HX_DEVINL uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// ---- dequantisation: warp w's page of every tile, K (kv 0) or V (kv 1) operand.
// A lane has 64 channels of one token. Its codes come a tile ahead by cp.async
// into its own 32 bytes of shared memory: as second copies in registers they
// were spilled (8 sequences on 1M tokens: 870 us against 513 at that step). The
// page's list record and table entry come a tile ahead in registers, and none
// is looked at before its turn, since a look at load time waits for the load
// (753 against 644).
template <int BITS, int KV, int SEG, int BASE>
HX_DEVINL void produce(const Params& p, Smem& sm, int h, int j, int w) {
  const int lane = threadIdx.x & 31, t = lane >> 1, half = lane & 1;
  const int Tc = p.sc.t_cal, NB = p.pool.num_blocks;
  constexpr int RB = D * BITS / 8, W = BITS * 2, E = BITS == 2 ? 4 : 1;  // row bytes; code words a lane; entries at once
  const uint8_t* code0 = p.pool.codes + (int64_t)h * NB * SEG + BASE + t * RB + half * (RB / 2);
  const uint32_t* dir0 = p.pool.dir + ((int64_t)h * NB * 2 + KV) * 4;
  const uint32_t own = smem_u32(sm.codes[KV][w]) + 16 * lane;  // 16-byte chunk u of the lane's half row at own + 512 u
  const uint32_t store0 = half * HALF + (16 * w + t) * 128 + 16u * ((4u * half) ^ (t & 7));
  volatile uint32_t* abort = &sm.abort;
  constexpr int kNone = -0x7fffffff;  // past the item's pages
  int g = 0;                          // tiles so far: stage 2 (g & 1) + KV
  Item it;
  for (int idx = 0; get_item(p, j, sm.row, idx, it); ++idx) {
    const int32_t* bt = p.bt + it.trow + it.page0 + w;
    const int pages = it.pages - w;
    auto entry = [&](int i) -> int { return PAGES * i < pages ? bt[PAGES * i] : kNone; };
    uint32_t off = 0u, cap = 0u, cnt = 0u;
    int phys = -1;
    auto load = [&](int e) {  // e: a table entry, itself loaded a tile before
      phys = e >= 0 && e < NB ? e : -1;
      if (phys >= 0) {
        const uint8_t* c = code0 + (int64_t)e * SEG;
        cp16(own, c);
        if (BITS == 4) cp16(own + 512, c + 16);
        const uint4 d = __ldg(reinterpret_cast<const uint4*>(dir0 + (int64_t)e * 8));
        off = d.x, cap = d.y, cnt = d.z;
      } else {
        off = cap = cnt = 0u;
        if (e != kNone && lane == 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int e_next = entry(1);
    load(entry(0));
    for (int i = 0; i < it.n; ++i, ++g) {
      // ---- this page's codes into registers, the next page's on their way
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      uint32_t c[W];
      // half 1 takes its 16-byte output chunks in the order 4 .. 7, 0 .. 3: the stores of four tokens' halves then
      // meet eight bank groups
      if (BITS == 4) {
        const uint4 x = lds128(own + 512 * half), y = lds128(own + 512 * (half ^ 1));
        c[0] = x.x, c[1] = x.y, c[2] = x.z, c[3] = x.w;
        c[W - 4] = y.x, c[W - 3] = y.y, c[W - 2] = y.z, c[W - 1] = y.w;
      } else {
        const uint4 x = lds128(own);
        c[0] = half ? x.z : x.x, c[1] = half ? x.w : x.y, c[2] = half ? x.x : x.z, c[3] = half ? x.y : x.w;
      }
      if (cnt > cap || (int64_t)off + cnt > p.pool.arena_capacity) {  // a record that leaves the arena
        set_err(p.err, HX_DEV_ERR_BOUNDS);
        cnt = 0u;
      }
      const uint32_t* list = p.pool.arena + off + lane;
      const int left = (int)cnt - lane;  // the lane's entries: list[0], list[32], ... while below left
      uint32_t ent[E];
#pragma unroll
      for (int u = 0; u < E; ++u) ent[u] = 32 * u < left ? __ldg(list + 32 * u) : 0u;
      const bool here = phys >= 0;
      // V: the token's own level row, if the page has tokens before the last calibrated position
      const int64_t pos0 = (int64_t)(p.vphys ? phys : it.page0 + PAGES * i + w) * S;
      const bool tail = !KV || pos0 >= Tc - 1;
      constexpr int LW = BITS == 4 ? 8 : 2;
      uint32_t lev[LW];  // levels 2u, 2u + 1
      if (KV && here && !tail) {
        const int L = p.sc.levels_v;
        const uint16_t* row = p.sc.v_poles + ((int64_t)h * Tc + min(pos0 + t, (int64_t)Tc - 1)) * L;
        if (L == (1 << BITS) && (reinterpret_cast<uintptr_t>(p.sc.v_poles) & 15u) == 0) {
          if (BITS == 4) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(row)), y = __ldg(reinterpret_cast<const uint4*>(row) + 1);
            lev[0] = x.x, lev[1] = x.y, lev[2 % LW] = x.z, lev[3 % LW] = x.w;
            lev[4 % LW] = y.x, lev[5 % LW] = y.y, lev[6 % LW] = y.z, lev[7 % LW] = y.w;
          } else {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(row));
            lev[0] = x.x, lev[1] = x.y;
          }
        } else {
#pragma unroll
          for (int u = 0; u < LW; ++u)
            lev[u] = (2 * u < L ? (uint32_t)row[2 * u] : 0u) | ((2 * u + 1 < L ? (uint32_t)row[2 * u + 1] : 0u) << 16);
        }
      }
      __syncwarp();  // the codes are in registers: their place may be filled again
      load(e_next);
      e_next = entry(i + 2);
      const int valid = KV ? min(S, it.tokens - (PAGES * i + w) * S) : S;  // K past the tokens is masked as a score
      const int st = 2 * (g & 1) + KV;
      if (g >= 2 && !tc::wait_warp(&sm.kv_empty[st], ((g >> 1) & 1) ^ 1, abort)) return;
      const uint32_t base = smem_u32(sm.kv[0]) + st * (KT * D * 2), at = base + store0, slab = base + 16 * w * 128;
      if (!here) {  // past the item's pages (masked), or a page id out of range (flagged)
#pragma unroll
        for (int u = 0; u < 8; ++u) sts128(at ^ (16u * u), make_uint4(0u, 0u, 0u, 0u));
      } else {
        if (KV == 0) {
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const uint32_t tab = smem_u32(sm.klut) + 2048u * half + 1024u * (half ^ jj);
            if (BITS == 4) {
              const uint32_t low = (64u * half + 32u * (half ^ jj)) * 0x01010101u;
#pragma unroll
              for (int u = 0; u < 4; ++u)
                sts128(at ^ (64u * jj + 16u * u), lut8_nib<32>(c[(4 * jj + u) % W], low, tab, 256u * u));
            } else {
              const uint32_t low = 64u * half * 0x01010101u;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint4 o0, o1;
                lut8_pair<64>(c[2 * jj + u], low, tab, 512u * u, o0, o1);
                sts128(at ^ (64u * jj + 32u * u), o0);
                sts128(at ^ (64u * jj + 32u * u + 16u), o1);
              }
            }
          }
        } else if (BITS == 4) {
          uint32_t lb[4], hb[4];
          if (tail) {
            const uint4 x = lds128(smem_u32(sm.vplane)), y = lds128(smem_u32(sm.vplane + 4));
            lb[0] = x.x, lb[1] = x.y, lb[2] = x.z, lb[3] = x.w;
            hb[0] = y.x, hb[1] = y.y, hb[2] = y.z, hb[3] = y.w;
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              lb[u] = prmt(lev[(2 * u) % LW], lev[(2 * u + 1) % LW], 0x6420u);
              hb[u] = prmt(lev[(2 * u) % LW], lev[(2 * u + 1) % LW], 0x7531u);
            }
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) sts128(at ^ (16u * u), lut8_reg(c[u % W], lb, hb));
        } else {
          const uint32_t lb = prmt(lev[0], lev[1], 0x6420u), hb = prmt(lev[0], lev[1], 0x7531u);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint4 o0, o1;
            if (tail) lut8_pair<0>(c[u], 0u, smem_u32(sm.vpair), 0u, o0, o1);
            else crumbs_reg(c[u], lb, hb, o0, o1);
            sts128(at ^ (32u * u), o0);
            sts128(at ^ (32u * u + 16u), o1);
          }
        }
        // rows that are not attended are zeroed: P is 0 there, but 0 * inf is not
        if (KV && valid < S && t >= valid) {
#pragma unroll
          for (int u = 0; u < 8; ++u) sts128(at ^ (16u * u), make_uint4(0u, 0u, 0u, 0u));
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < E; ++u)
          if (32 * u < left) patch(slab, ent[u], valid, p.err);
        for (int e = 32 * E; e < left; e += 32) patch(slab, __ldg(list + e), valid, p.err);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::arrive(&sm.kv_full[st]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int BK, int BV>
__global__ void __launch_bounds__(NTHREADS, 1) prefix_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = p.pool.num_kv_heads, G = p.G, TQ = p.TQ, Tc = p.sc.t_cal;
  const int h = blockIdx.x % H, j = blockIdx.x / H;
  pdl_allow_next();  // the merge's CTAs fit beside this one's and wait for the whole grid

  if (warp == 24) {
    if (lane == 0) {
      for (int q = 0; q < 2; ++q) {
        mbar_init(&sm.q_full[q], 1);
        mbar_init(&sm.s_full[q], 1);
        mbar_init(&sm.p_full[q], 4);
        mbar_init(&sm.o_full[q], 1);
      }
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&sm.kv_full[s], PAGES);
        mbar_init(&sm.kv_empty[s], 1);
      }
      mbar_init(&sm.ml_full, 4);
      mbar_init(&sm.ml_empty, 4);
      mbar_init(&sm.drain, 1);
      sm.abort = 0u;
      fence_mbar_init();
    }
    __syncwarp();
    tc::tmem_alloc(&sm.tmem, 512);
    // ---- the first row that is neither padding nor too short names the prefix's pages
    const int64_t least = max((int64_t)p.prefix_pages * S, (int64_t)1);
    int row = -1;
    for (int b0 = 0; b0 < p.B && row < 0; b0 += 32) {
      const uint32_t m = __ballot_sync(0xffffffffu, b0 + lane < p.B && p.seq_lens[b0 + lane] >= least);
      if (m) row = b0 + __ffs(m) - 1;
    }
    if (lane == 0) sm.row = row;
  }
  // ---- level tables of the head
  auto kpole = [&](int d, int c) -> uint32_t {
    return c < p.sc.levels_k ? p.sc.k_poles[((int64_t)h * D + d) * p.sc.levels_k + c] : 0u;
  };
  auto vtail = [&](int c) -> uint32_t {
    return c < p.sc.levels_v ? p.sc.v_poles[((int64_t)h * Tc + (Tc - 1)) * p.sc.levels_v + c] : 0u;
  };
  for (int i = threadIdx.x; i < (BK == 4 ? 16 * D : 16 * (D / 2)); i += NTHREADS) {
    if (BK == 4) {
      const int d = i >> 4;
      sm.klut[16 * d + 16 * (d >> 5) + (i & 15)] = (uint16_t)kpole(d, i & 15);
    } else {
      const int P = i >> 4, e = i & 15;
      reinterpret_cast<uint32_t*>(sm.klut)[16 * P + 16 * (P >> 5) + e] =
          kpole(2 * P, e & 3) | (kpole(2 * P + 1, e >> 2) << 16);
    }
  }
  if (BV == 2 && threadIdx.x < 16) sm.vpair[threadIdx.x] = vtail(threadIdx.x & 3) | (vtail(threadIdx.x >> 2) << 16);
  if (BV == 4 && threadIdx.x < 8) {  // plane k: byte i = byte (k >> 2) of level 4 (k & 3) + i
    const int k = threadIdx.x, sh = 8 * (k >> 2);
    uint32_t v = 0u;
    for (int i = 0; i < 4; ++i) v |= ((vtail(4 * (k & 3) + i) >> sh) & 0xFFu) << (8 * i);
    sm.vplane[k] = v;
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sm.tmem;
  volatile uint32_t* abort = &sm.abort;
  Item it;

  if (warp < 8) {
    // ---- softmax: warpgroup q; with two tiles q is the tile, else the stream of key tiles q, q + 2, ...
    const int q = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sb = tmem + lanes + 128 * q, ob = tmem + lanes + 256 + 128 * q;
    int used = 0, done = 0, joined = 0;  // S tiles, O results and joined items of this warpgroup so far
    bool ok = true;
    for (int idx = 0; ok && get_item(p, j, sm.row, idx, it); ++idx) {
      const int seq = it.seq0 + (it.two ? q * TQ : 0) + r / G;
      const bool live = it.suffix ? r < G : (r < TQ * G && seq < p.B);
      const bool any = __any_sync(0xffffffffu, live);  // warps without rows only keep step
      const int first = it.two ? 0 : q, step = it.two ? 1 : 2;
      float m = -INFINITY, l = 0.0f;
      int k = 0;
      for (int i = first; i < it.n && ok; i += step, ++k, ++used) {
        ok = tc::wait_warp(&sm.s_full[q], used & 1, abort);
        if (!ok) break;
        if (any) {
          tc::fence_after();
          const int lim = it.tokens - KT * i;  // valid keys of the tile
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
          for (int qt = 0; qt < 4; ++qt) {
            uint32_t s[32];
            tc::ld32(s, sb + 32 * qt);
            tc::wait_ld();
            if (lim < KT) {
#pragma unroll
              for (int c = 0; c < 32; ++c) s[c] = 32 * qt + c < lim ? s[c] : 0xff800000u;
            }
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              mx[0] = fmaxf(mx[0], fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 1])));
              mx[1] = fmaxf(mx[1], fmaxf(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])));
            }
          }
          const float mt = fmaxf(mx[0], mx[1]);
          const bool move = (mt - m) * p.c > kSlack;
          if (__any_sync(0xffffffffu, move)) {
            const float mn = move ? mt : m;
            const float a = move ? tc::ex2((m - mn) * p.c) : 1.0f;
            m = mn;
            l *= a;
            if (k > 0) {  // the stream's O is complete: this S was issued after it
              const uint64_t a2 = tc::f2_pack(a, a);
#pragma unroll 1
              for (int u = 0; u < D / 32; ++u) {
                uint32_t o[32];
                tc::ld32(o, ob + 32 * u);
                tc::wait_ld();
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                  float x, y;
                  tc::f2_unpack(tc::f2_mul(tc::f2_pack(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), a2), x, y);
                  o[c] = __float_as_uint(x);
                  o[c + 1] = __float_as_uint(y);
                }
                tc::st32(ob + 32 * u, o);
              }
            }
          }
          const float mb = m == -INFINITY ? 0.0f : -m * p.c;
          const uint64_t c2 = tc::f2_pack(p.c, p.c), mb2 = tc::f2_pack(mb, mb);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll 1
          for (int qt = 0; qt < 4; ++qt) {  // P of a quarter overwrites S columns already used
            uint32_t s[32];
            tc::ld32(s, sb + 32 * qt);
            tc::wait_ld();
            if (lim < KT) {
#pragma unroll
              for (int c = 0; c < 32; ++c) s[c] = 32 * qt + c < lim ? s[c] : 0xff800000u;
            }
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              float x, y;
              tc::f2_unpack(tc::f2_fma(tc::f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, mb2), x, y);
              x = tc::ex2(x);
              y = tc::ex2(y);
              sum[(c >> 1) & 1] = tc::f2_add(sum[(c >> 1) & 1], tc::f2_pack(x, y));
              pk[c >> 1] = pack_h2(x, y);
            }
            tc::st16(sb + 16 * qt, pk);
          }
          float x, y;
          tc::f2_unpack(tc::f2_add(sum[0], sum[1]), x, y);
          l += x + y;
          tc::wait_st();
          tc::fence_before();
        }
        __syncwarp();
        if (lane == 0) tc::arrive(&sm.p_full[q]);
      }
      if (it.n == 0) continue;
      // ---- the rows' partials. The second stream's rows sit in the same TMEM lanes: the first warpgroup joins both
      if (ok && k > 0) ok = tc::wait_warp(&sm.o_full[q], done++ & 1, abort);
      if (!ok) break;
      tc::fence_after();
      if (!it.two && q == 1) {
        sm.ml[r] = make_float2(m * p.c, l);  // -inf, 0 without a tile
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::arrive(&sm.ml_full);
        ok = tc::wait_warp(&sm.ml_empty, joined++ & 1, abort);  // O may be overwritten
        continue;
      }
      const int64_t rows = (int64_t)p.B * H * G;
      const int64_t row = ((int64_t)(it.suffix ? it.seq0 : seq) * H + h) * G + (it.suffix ? r : r % G);
      const int64_t at = (int64_t)it.pidx * rows + row;
      float w0 = 1.0f, w1 = 0.0f, M = m * p.c;
      bool both = false;
      if (!it.two) {
        ok = tc::wait_warp(&sm.ml_full, joined++ & 1, abort);
        if (!ok) break;
        tc::fence_after();
        both = it.n > 1;
        const float2 x = sm.ml[r];
        const float top = fmaxf(M, x.x);
        if (both && top != -INFINITY) {
          w0 = tc::ex2(M - top);
          w1 = tc::ex2(x.x - top);
          M = top;
          l = l * w0 + x.y * w1;
        }
      }
      if (any) {
        if (live) p.part_ml[at] = make_float2(M, l);
#pragma unroll 1
        for (int u = 0; u < D / 16; ++u) {
          uint32_t o[16], o1[16];
          tc::ld16(o, ob + 16 * u);
          if (both) tc::ld16(o1, ob + 128 + 16 * u);
          tc::wait_ld();
          if (both) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              o[c] = __float_as_uint(__uint_as_float(o[c]) * w0 + __uint_as_float(o1[c]) * w1);
          }
          if (live) {
            uint4* dst = reinterpret_cast<uint4*>(p.part_o + at * D + 16 * u);
#pragma unroll
            for (int c = 0; c < 4; ++c) dst[c] = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          }
        }
      }
      tc::fence_before();
      __syncwarp();
      if (!it.two && lane == 0) tc::arrive(&sm.ml_empty);
    }
  } else if (warp < 16) {
    produce<BK, 0, S * D * (BK + BV) / 8, 0>(p, sm, h, j, warp - 8);
  } else if (warp < 24) {
    produce<BV, 1, S * D * (BK + BV) / 8, S * D * BK / 8>(p, sm, h, j, warp - 16);
  } else {
    // ---- query tiles and matrix products
    constexpr uint32_t ids = tc::idesc_f16(0, ROWS, KT, 0), idv = tc::idesc_f16(0, ROWS, D, 1);
    int qn[2] = {0, 0}, used[2] = {0, 0};  // loads into a query buffer; S tiles of a warpgroup so far
    auto load_q = [&](int buf, int seq0) {  // the buffer's last products are complete: their P has been used
      if (tc::elect()) {
        mbar_arrive_expect_tx(&sm.q_full[buf], TQ * G * D * 2);
        for (int u = 0; u < 2; ++u) tc::tma3(sm.q[buf] + u * HALF, &p.mq, 64 * u, h * G, seq0, &sm.q_full[buf]);
      }
      ++qn[buf];
    };
    auto qk = [&](int q, int buf, int g) {
      const uint64_t qd = tc::desc128(smem_u32(sm.q[buf]), 0), kd = tc::desc128(smem_u32(sm.kv[2 * (g & 1)]), 0);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = ((k / 4) * HALF + (k % 4) * 32) >> 4;
        tc::mma_ss(tmem + 128 * q, qd + off, kd + off, ids, k > 0);
      }
      tc::commit(&sm.s_full[q]);
    };
    auto pv = [&](int q, int g, bool more) {
      const uint64_t vd = tc::desc128(smem_u32(sm.kv[2 * (g & 1) + 1]), HALF);
#pragma unroll
      for (int k = 0; k < KT / 16; ++k)
        tc::mma_ts(tmem + 256 + 128 * q, tmem + 128 * q + 8 * k, vd + 128 * k, idv, more || k > 0);
    };
    auto full = [&](int g, int kv) { return tc::wait_warp(&sm.kv_full[2 * (g & 1) + kv], (g >> 1) & 1, abort); };
    auto p_wait = [&](int q) { return tc::wait_warp(&sm.p_full[q], used[q]++ & 1, abort); };
    bool ok = true;
    int g = 0, buf = 0;  // tiles so far; the query buffer of the next one-tile item
    bool ahead = false;  // its rows are on the way
    bool more = get_item(p, j, sm.row, 0, it);
    for (int idx = 0; ok && more; ++idx) {
      const Item now = it;
      more = get_item(p, j, sm.row, idx + 1, it);
      if (now.n == 0) continue;
      if (now.two) {
        load_q(0, now.seq0);
        load_q(1, now.seq0 + TQ);
        ok = tc::wait_warp(&sm.q_full[0], (qn[0] - 1) & 1, abort) && tc::wait_warp(&sm.q_full[1], (qn[1] - 1) & 1, abort);
        if (ok) ok = full(g, 0);
        if (ok && tc::elect()) {
          tc::fence_after();
          qk(0, 0, g);
          qk(1, 1, g);
          tc::commit(&sm.kv_empty[2 * (g & 1)]);
        }
        for (int i = 0; i < now.n && ok; ++i, ++g) {
          ok = full(g, 1);
          if (ok && i + 1 < now.n) ok = full(g + 1, 0);
          for (int q = 0; q < 2 && ok; ++q) {
            ok = p_wait(q);
            if (ok && tc::elect()) {
              tc::fence_after();
              pv(q, g, i > 0);
              if (i + 1 < now.n) qk(q, q, g + 1);
              else tc::commit(&sm.o_full[q]);
            }
            __syncwarp();
          }
          if (ok && tc::elect()) {
            tc::commit(&sm.kv_empty[2 * (g & 1) + 1]);
            if (i + 1 < now.n) tc::commit(&sm.kv_empty[2 * ((g + 1) & 1)]);
          }
          __syncwarp();
        }
      } else {
        // key tile i belongs to stream i & 1
        if (!ahead) load_q(buf, now.seq0);
        ok = tc::wait_warp(&sm.q_full[buf], (qn[buf] - 1) & 1, abort);
        for (int i = 0; i < 2 && i < now.n && ok; ++i) {
          ok = full(g + i, 0);
          if (ok && tc::elect()) {
            tc::fence_after();
            qk(i, buf, g + i);
            tc::commit(&sm.kv_empty[2 * ((g + i) & 1)]);
          }
          __syncwarp();
        }
        ahead = more && it.n > 0 && !it.two;
        if (ahead) load_q(buf ^ 1, it.seq0);  // the item before last is complete
        for (int i = 0; i < now.n && ok; ++i, ++g) {
          const int q = i & 1;
          ok = full(g, 1) && p_wait(q);
          if (ok && tc::elect()) {
            tc::fence_after();
            pv(q, g, i > 1);
            tc::commit(&sm.kv_empty[2 * (g & 1) + 1]);
            if (i + 2 >= now.n) tc::commit(&sm.o_full[q]);
          }
          __syncwarp();
          if (ok && i + 2 < now.n) {
            ok = full(g + 2, 0);
            if (ok && tc::elect()) {
              tc::fence_after();
              qk(q, buf, g + 2);
              tc::commit(&sm.kv_empty[2 * (g & 1)]);
            }
            __syncwarp();
          }
        }
        buf ^= 1;
      }
    }
    for (int b = 0; b < 2; ++b)  // loads still in flight after a timeout land before the CTA's memory goes
      if (qn[b]) (void)mbar_wait(&sm.q_full[b], (qn[b] - 1) & 1);
    if (tc::elect()) tc::commit(&sm.drain);  // and no product may be in flight when TMEM is freed
    __syncwarp();
    (void)mbar_wait(&sm.drain, 0);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 24) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && sm.abort) set_err(p.err, HX_DEV_ERR_TIMEOUT);
}

// Joins a row's partials: weights 2^(m - M), M the largest m; one CTA a row,
// its warps take the partials in turns of 32 (37 splits and a suffix: two warps).
constexpr int MW = 4;
struct MergeParams {
  const float* part_o;
  const float2* part_ml;
  const int32_t* seq_lens;
  int B, Hq, prefix, n_splits, bt_stride;
  uint16_t* out;
  float* lse;
  uint32_t* err;
};

__global__ void __launch_bounds__(32 * MW) merge_kernel(const MergeParams p) {
  __shared__ float4 acc[MW][32];
  __shared__ float2 ml[MW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.B * p.Hq, row = blockIdx.x;
  pdl_wait();
  const int b = (int)(row / p.Hq), len = p.seq_lens[b];
  // a padding row (no tokens), and one shorter than the prefix or past its table (flagged): nothing attended
  const bool bad = len != 0 && (len < p.prefix || (len - 1) / S >= p.bt_stride);
  const int n = len == 0 || bad ? 0 : p.n_splits + (len > p.prefix ? 1 : 0);
  if (bad && threadIdx.x == 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float M = -INFINITY, l = 0.0f;
  for (int i0 = 32 * warp; i0 < n; i0 += 32 * MW) {
    const int i = i0 + lane;
    const float2 x = i < n ? p.part_ml[(int64_t)i * rows + row] : make_float2(-INFINITY, 0.0f);
    float mx = x.x;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    const float Mn = fmaxf(M, mx), a = Mn == -INFINITY ? 1.0f : exp2f(M - Mn);
    M = Mn;
    const float wgt = x.x == -INFINITY ? 0.0f : exp2f(x.x - M);
    l = l * a + wgt * x.y;  // lane-wise: summed over the lanes at the end
    o.x *= a, o.y *= a, o.z *= a, o.w *= a;
    const int cnt = min(32, n - i0);
#pragma unroll 8
    for (int j = 0; j < cnt; ++j) {
      const float wj = __shfl_sync(0xffffffffu, wgt, j);
      if (wj != 0.0f) {  // no weight: nothing to add (and nothing stored, where there were no keys)
        const float4 v = reinterpret_cast<const float4*>(p.part_o + ((int64_t)(i0 + j) * rows + row) * D)[lane];
        o.x += wj * v.x, o.y += wj * v.y, o.z += wj * v.z, o.w += wj * v.w;
      }
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  acc[warp][lane] = o;
  if (lane == 0) ml[warp] = make_float2(M, l);
  __syncthreads();
  if (warp == 0) {
    float Mt = -INFINITY;
    for (int w = 0; w < MW; ++w) Mt = fmaxf(Mt, ml[w].x);
    float lt = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = 0; w < MW; ++w) {
      const float a = ml[w].x == -INFINITY ? 0.0f : exp2f(ml[w].x - Mt);
      const float4 v = acc[w][lane];
      lt += a * ml[w].y;
      o.x += a * v.x, o.y += a * v.y, o.z += a * v.z, o.w += a * v.w;
    }
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
    reinterpret_cast<uint2*>(p.out + row * D)[lane] = make_uint2(pack_h2(o.x * inv, o.y * inv), pack_h2(o.z * inv, o.w * inv));
    if (lane == 0 && p.lse) p.lse[row] = lt == 0.0f ? -INFINITY : (Mt + log2f(lt)) * kLn2;
  }
}

// Splits of the prefix: CTAs for one wave (one fits an SM), at most one split
// per key tile. Holding CTAs back for the suffixes (two key tiles a sequence
// assumed, since their lengths are not known on the host) was slower: 32K
// tokens and 64 suffixes of up to 512 took 91 us against 84, 128K and 16 of up
// to 777 85 against 81.
int default_splits(int H, int RB, int tiles) {
  int ns = 148 / (H * RB);
  ns = ns < 1 ? 1 : ns;
  return ns > tiles ? tiles : ns;
}

}  // namespace px
}  // namespace hx

using namespace hx;

extern "C" {

HX_API int32_t hx_prefix_splits(int32_t B, int32_t H, int32_t group, int32_t prefix_pages) {
  if (B < 1 || H < 1 || group < 1 || group > px::ROWS || prefix_pages < 1) return 0;
  const int per = 2 * (px::ROWS / group);
  return px::default_splits(H, (B + per - 1) / per, (prefix_pages + px::PAGES - 1) / px::PAGES);
}

HX_API int64_t hx_prefix_scratch_bytes(int32_t B, int32_t H, int32_t group, int32_t n_splits) {
  if (B < 1 || H < 1 || group < 1 || n_splits < 0) return 0;
  return (int64_t)(n_splits + 1) * B * H * group * (px::D + 2) * 4;
}

HX_API int hx_prefix_decode(void* stream, const hx_pool_layer* pool, const hx_layer_scales* sc, const uint16_t* q,
                            int32_t B, int32_t group, float softmax_scale, const int32_t* block_table,
                            int32_t bt_stride, const int32_t* seq_lens, int32_t prefix_pages, int32_t flags,
                            int32_t n_splits, void* scratch, uint16_t* out, float* lse, uint32_t* dev_err) {
  if (!pool || !sc || B < 0 || group < 1 || prefix_pages < 0 || prefix_pages > bt_stride) return HX_ERR_ARG;
  if ((flags & ~HX_VPOS_PHYSICAL) != 0 || !(softmax_scale > 0.0f) || softmax_scale > 3.0e38f) return HX_ERR_ARG;
  if (B == 0) return HX_OK;
  if (!q || !block_table || !seq_lens || !scratch || !out) return HX_ERR_ARG;
  if (pool->head_size != px::D || pool->block_size != px::S || group > px::ROWS) return HX_ERR_UNSUPPORTED;
  if ((pool->bits_k != 2 && pool->bits_k != 4) || (pool->bits_v != 2 && pool->bits_v != 4)) return HX_ERR_UNSUPPORTED;
  if (sc->levels_k < 1 || sc->levels_k > (1 << pool->bits_k) || sc->levels_v < 1 ||
      sc->levels_v > (1 << pool->bits_v) || sc->t_cal < 1)
    return HX_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(scratch) % 16 ||
      reinterpret_cast<uintptr_t>(out) % 8 || reinterpret_cast<uintptr_t>(pool->codes) % 16 ||
      reinterpret_cast<uintptr_t>(pool->dir) % 16)
    return HX_ERR_ARG;
  const int H = pool->num_kv_heads;
  const int tiles = (prefix_pages + px::PAGES - 1) / px::PAGES;
  if (n_splits < 0 || n_splits > tiles || (n_splits == 0) != (tiles == 0)) return HX_ERR_ARG;
  px::Params p;
  p.TQ = px::ROWS / group;
  p.RB = (B + 2 * p.TQ - 1) / (2 * p.TQ);
  if (!make_tmap3(&p.mq, false, q, px::D, H * group, B, px::D, (int64_t)H * group * px::D, group, p.TQ))
    return HX_ERR_LAUNCH;
  const int64_t rows = (int64_t)B * H * group;
  p.pool = *pool;
  p.sc = *sc;
  p.B = B;
  p.G = group;
  p.c = softmax_scale * px::kLog2e;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.seq_lens = seq_lens;
  p.prefix_pages = prefix_pages;
  p.n_splits = n_splits;
  p.vphys = (flags & HX_VPOS_PHYSICAL) ? 1 : 0;
  p.part_o = reinterpret_cast<float*>(scratch);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)(n_splits + 1) * rows * px::D);
  p.err = dev_err;
  // a CTA for each split of each row block and head, and more for the suffixes while SMs are left
  const int pre = p.RB * n_splits, wave = 148 / H > 1 ? 148 / H : 1;
  p.J = pre + B < wave ? pre + B : (pre > wave ? pre : wave);
  const int64_t grid = (int64_t)H * p.J;
  if (grid > 0x7fffffffll || rows > 0x7fffffffll) return HX_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  constexpr int smem = (int)sizeof(px::Smem) + 1024;
  static_assert(smem <= 232448, "a CTA has 227 KB of shared memory");
  auto kern = pool->bits_k == 4 ? (pool->bits_v == 4 ? px::prefix_kernel<4, 4> : px::prefix_kernel<4, 2>)
                                : (pool->bits_v == 4 ? px::prefix_kernel<2, 4> : px::prefix_kernel<2, 2>);
  static unsigned long long done[4] = {0, 0, 0, 0};
  if (!allow_smem(kern, smem, done[(pool->bits_k == 4) * 2 + (pool->bits_v == 4)])) return HX_ERR_LAUNCH;
  kern<<<(unsigned)grid, px::NTHREADS, smem, s>>>(p);
  HX_LAUNCH_CHECK();
  px::MergeParams mp{p.part_o, p.part_ml, seq_lens, B, H * group, prefix_pages * px::S, n_splits, bt_stride, out,
                     lse, dev_err};
  if (hx_launch_pdl(px::merge_kernel, dim3((unsigned)rows), dim3(32 * px::MW), 0, s, mp) != cudaSuccess) {
    (void)cudaGetLastError();
    return HX_ERR_LAUNCH;
  }
  return HX_OK;
}

}  // extern "C"
