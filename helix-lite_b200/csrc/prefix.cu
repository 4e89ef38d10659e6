// Decode attention of a batch whose sequences share a long prefix of pool
// pages: the prefix is read and dequantised once for the whole batch.
//
//   o_b = softmax over the sequence's tokens of (scale q_b . k_j) v_j,  the
//   first prefix_len tokens being the same pool pages for every sequence
//
// The query rows of a KV head (sequences x heads of the group) are the M side
// of a matrix product over each dequantised tile of 128 tokens (8 pages). Work
// items, one a CTA:
//   prefix  (KV head, block of two 128-row query tiles, split of the prefix):
//           both tiles use each dequantised key tile. A block with one tile
//           only runs it twice, on the even and on the odd key tiles
//   suffix  (KV head, sequence): the sequence's own pages, its G rows alone,
//           again as two streams of key tiles
// Each leaves unnormalised partials (m, l, O) per row; a second kernel joins a
// row's partials. Roles in a CTA (20 warps):
//   0-7    two softmax warpgroups, a row a thread (as in the prompt kernel: S
//          and P in TMEM, the maximum moves only past 2^8)
//   8-15   dequantisation: warp w turns page w of each tile into 16 rows of the
//          swizzled K and V operands (level tables by prmt-built addresses,
//          registers for nuq4 V past t_cal), outliers patched in
//   16     the matrix products (tcgen05.mma, one thread); 17 the query tiles
#include "dequant.cuh"
#include "tcgen.cuh"
#include "tmap.cuh"

namespace hx {
namespace px {

constexpr int D = 128, S = 16, KT = 128, ROWS = 128, PAGES = KT / S;
constexpr int STAGES = 4;
constexpr int NTHREADS = 640;
constexpr int HALF = KT * 128;  // bytes of 128 rows of 64 fp16
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;

struct Smem {
  alignas(1024) uint8_t q[2][ROWS * D * 2];
  alignas(1024) uint8_t kv[STAGES][KT * D * 2];
  alignas(256) uint16_t klut[16 * D + 128];      // K tables, bank-spread (32 bytes of room after every 32 channels)
  alignas(256) uint16_t vlut[PAGES][S * 16];     // V levels per token of each warp's page (before t_cal)
  alignas(256) uint32_t vpair[16];               // nuq2 V past t_cal: level pairs by code pair
  alignas(16) uint32_t vplane[8];                // nuq4 V past t_cal: byte planes
  uint64_t q_full[2], kv_full[STAGES], kv_empty[STAGES], s_full[2], p_full[2], o_full[2], drain;
  uint32_t tmem, abort;
};

struct Params {
  CUtensorMap mq;
  hx_pool_layer pool;
  hx_layer_scales sc;
  int B, G, TQ, RB;          // sequences, heads of a group, sequences a tile, row blocks
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

template <int BK, int BV>
__global__ void __launch_bounds__(NTHREADS, 1) prefix_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  constexpr int RBK = D * BK / 8, RBV = D * BV / 8, SEG = S * (RBK + RBV);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = p.pool.num_kv_heads, G = p.G, TQ = p.TQ, NB = p.pool.num_blocks, Tc = p.sc.t_cal;

  // ---- the work item
  const int n_pre = H * p.RB * p.n_splits;
  const bool suffix = (int)blockIdx.x >= n_pre;
  const int it = suffix ? (int)blockIdx.x - n_pre : (int)blockIdx.x;
  const int h = it % H;
  int seq0, page0, pages, tokens, pidx;  // first sequence of the rows; the item's pages in table row `trow`
  bool two;                              // two query tiles (else one tile, two streams of key tiles)
  if (suffix) {
    seq0 = it / H;
    const int len = p.seq_lens[seq0], pre = p.prefix_pages * S;
    tokens = len - pre;
    if (tokens <= 0 || (len - 1) / S >= p.bt_stride) return;  // the merge flags a bad length
    page0 = p.prefix_pages;
    pages = (tokens + S - 1) / S;
    two = false;
    pidx = 2 * p.n_splits;
  } else {
    const int rb = (it / H) % p.RB, split = it / H / p.RB;
    seq0 = rb * 2 * TQ;
    two = seq0 + TQ < p.B;
    const int nt = (p.prefix_pages + PAGES - 1) / PAGES;
    const int ta = (int)((int64_t)nt * split / p.n_splits), te = (int)((int64_t)nt * (split + 1) / p.n_splits);
    page0 = ta * PAGES;
    pages = min(te * PAGES, p.prefix_pages) - page0;
    tokens = pages * S;
    pidx = 2 * split;
  }
  const int64_t trow = suffix ? (int64_t)seq0 * p.bt_stride : 0;
  const int n = (pages + PAGES - 1) / PAGES;  // key tiles

  if (warp == 16) {
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
      mbar_init(&sm.drain, 1);
      sm.abort = 0u;
      fence_mbar_init();
    }
    __syncwarp();
    tc::tmem_alloc(&sm.tmem, 512);
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

  if (warp < 8) {
    // ---- softmax: warpgroup q; with two tiles q is the tile, else the stream of key tiles q, q + 2, ...
    tc::regs_inc<120>();
    const int q = warp >> 2, r = threadIdx.x & 127;
    const int seq = seq0 + (two ? q * TQ : 0) + r / G;
    const bool live = suffix ? r < G : (r < TQ * G && seq < p.B);
    const bool any = __any_sync(0xffffffffu, live);  // warps without rows only keep step
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sb = tmem + lanes + 128 * q, ob = tmem + lanes + 256 + 128 * q;
    const int first = two ? 0 : q, step = two ? 1 : 2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    int k = 0;
    for (int i = first; i < n && ok; i += step, ++k) {
      ok = tc::wait_warp(&sm.s_full[q], k & 1, abort);
      if (!ok) break;
      if (any) {
        tc::fence_after();
        const int lim = tokens - KT * i;  // valid keys of the tile
        uint32_t s[64];
        float mt = -INFINITY;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          tc::ld32(s, sb + 64 * hf);
          tc::ld32(s + 32, sb + 64 * hf + 32);
          tc::wait_ld();
          if (lim < KT) {
#pragma unroll
            for (int j = 0; j < 64; ++j) s[j] = 64 * hf + j < lim ? s[j] : 0xff800000u;
          }
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 64; j += 4) {
            mx[0] = fmaxf(mx[0], fmaxf(__uint_as_float(s[j]), __uint_as_float(s[j + 1])));
            mx[1] = fmaxf(mx[1], fmaxf(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])));
          }
          mt = fmaxf(mt, fmaxf(mx[0], mx[1]));
        }
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
              for (int j = 0; j < 32; j += 2) {
                float x, y;
                tc::f2_unpack(tc::f2_mul(tc::f2_pack(__uint_as_float(o[j]), __uint_as_float(o[j + 1])), a2), x, y);
                o[j] = __float_as_uint(x);
                o[j + 1] = __float_as_uint(y);
              }
              tc::st32(ob + 32 * u, o);
            }
          }
        }
        const float mb = m == -INFINITY ? 0.0f : -m * p.c;
        const uint64_t c2 = tc::f2_pack(p.c, p.c), mb2 = tc::f2_pack(mb, mb);
        uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // P of a half overwrites S columns already used
          tc::ld32(s, sb + 64 * hf);
          tc::ld32(s + 32, sb + 64 * hf + 32);
          tc::wait_ld();
          if (lim < KT) {
#pragma unroll
            for (int j = 0; j < 64; ++j) s[j] = 64 * hf + j < lim ? s[j] : 0xff800000u;
          }
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            float x, y;
            tc::f2_unpack(tc::f2_fma(tc::f2_pack(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), c2, mb2), x, y);
            x = tc::ex2(x);
            y = tc::ex2(y);
            sum[(j >> 1) & 1] = tc::f2_add(sum[(j >> 1) & 1], tc::f2_pack(x, y));
            pk[j >> 1] = pack_h2(x, y);
          }
          tc::st32(sb + 32 * hf, pk);
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
    // ---- the rows' partials
    if (ok && k > 0) ok = tc::wait_warp(&sm.o_full[q], 0, abort);
    tc::fence_after();
    if (ok && any) {
      const int64_t rows = (int64_t)p.B * H * G;
      const int64_t row = ((int64_t)(suffix ? seq0 : seq) * H + h) * G + (suffix ? r : r % G);
      const int64_t at = (int64_t)(pidx + (two ? 0 : q)) * rows + row;
      if (live) p.part_ml[at] = make_float2(m * p.c, l);
      if (k > 0) {
#pragma unroll 1
        for (int u = 0; u < D / 32; ++u) {
          uint32_t o[32];
          tc::ld32(o, ob + 32 * u);
          tc::wait_ld();
          if (live) {
            uint4* dst = reinterpret_cast<uint4*>(p.part_o + at * D + 32 * u);
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
      }
      // a block of two tiles has one partial per split: the second place stays empty
      if (two && live) p.part_ml[at + rows] = make_float2(-INFINITY, 0.0f);
    }
  } else if (warp < 16) {
    // ---- dequantisation: warp w's page of every tile
    const int w = warp - 8, t = lane >> 1, half = lane & 1;
    const uint8_t* codes = p.pool.codes + (int64_t)h * NB * SEG;
    const uint32_t* dirs = p.pool.dir + (int64_t)h * NB * 8;
    constexpr int EK = BK == 2 ? 4 : 1, EV = BV == 2 ? 4 : 1;  // outlier entries a lane holds ahead
    constexpr int WK = BK * 2, WV = BV * 2;                      // code words a lane holds (64 channels)
    struct Ahead {
      uint32_t k[WK], v[WV];
      uint4 dk, dv;
      int phys;
    };
    auto phys_of = [&](int i) -> int {
      const int pg = PAGES * i + w;
      if (pg >= pages) return -1;
      const int pp = p.bt[trow + page0 + pg];
      if (pp >= 0 && pp < NB) return pp;
      if (lane == 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
      return -1;
    };
    auto load = [&](Ahead& a, int pp) {
      a.phys = pp;
      if (pp < 0) {
        a.dk = a.dv = make_uint4(0u, 0u, 0u, 0u);
        return;
      }
      // half 1 takes its 16-byte chunks in the order 4 .. 7, 0 .. 3: the stores of a row pair then meet 8 bank groups
      const uint8_t* seg = codes + (int64_t)pp * SEG;
      const uint8_t* kr = seg + t * RBK + half * (RBK / 2);
      const uint8_t* vr = seg + S * RBK + t * RBV + half * (RBV / 2);
      if (BK == 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(kr + 16 * half));
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(kr + 16 * (half ^ 1)));
        a.k[0] = x.x, a.k[1] = x.y, a.k[2] = x.z, a.k[3] = x.w;
        a.k[WK - 4] = y.x, a.k[WK - 3] = y.y, a.k[WK - 2] = y.z, a.k[WK - 1] = y.w;
      } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(kr + 8 * half));
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(kr + 8 * (half ^ 1)));
        a.k[0] = x.x, a.k[1] = x.y, a.k[2] = y.x, a.k[3] = y.y;
      }
      if (BV == 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(vr + 16 * half));
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(vr + 16 * (half ^ 1)));
        a.v[0] = x.x, a.v[1] = x.y, a.v[2] = x.z, a.v[3] = x.w;
        a.v[WV - 4] = y.x, a.v[WV - 3] = y.y, a.v[WV - 2] = y.z, a.v[WV - 1] = y.w;
      } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(vr + 8 * half));
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(vr + 8 * (half ^ 1)));
        a.v[0] = x.x, a.v[1] = x.y, a.v[2] = y.x, a.v[3] = y.y;
      }
      a.dk = __ldg(reinterpret_cast<const uint4*>(dirs + (int64_t)pp * 8));
      a.dv = __ldg(reinterpret_cast<const uint4*>(dirs + (int64_t)pp * 8 + 4));
    };
    auto fits = [&](uint4& d) {  // a record that leaves the arena is flagged and its entries left out
      if (d.z > d.y || (int64_t)d.x + d.z > p.pool.arena_capacity) {
        if (lane == 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
        d.z = 0u;
      }
    };
    const uint32_t t7 = t & 7;
    const uint32_t store0 = half * HALF + (16 * w + t) * 128 + 16u * ((4u * half) ^ t7);
    // entry -> byte offset in the page's rows: token << 24 | channel << 16 | value
    auto patch = [&](uint32_t slab, uint32_t e, int valid) {
      const uint32_t tt = e >> 24, d = (e >> 16) & 0xFFu;
      if (tt >= (uint32_t)S || d >= (uint32_t)D) {
        set_err(p.err, HX_DEV_ERR_BOUNDS);
      } else if ((int)tt < valid) {
        const uint32_t off = (d >> 6) * HALF + tt * 128 + ((((d >> 3) & 7) ^ (tt & 7)) << 4) + (d & 7) * 2;
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(slab + off), "h"((uint16_t)(e & 0xFFFFu)) : "memory");
      }
    };
    uint32_t lb[4], hb[4];
    if (BV == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) lb[i] = sm.vplane[i], hb[i] = sm.vplane[4 + i];
    }
    Ahead cur, nxt;
    load(cur, phys_of(0));
    int pp1 = n > 1 ? phys_of(1) : -1;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      fits(cur.dk);
      fits(cur.dv);
      uint32_t ek[EK], ev[EV];
#pragma unroll
      for (int u = 0; u < EK; ++u) ek[u] = lane + 32 * u < (int)cur.dk.z ? __ldg(p.pool.arena + cur.dk.x + lane + 32 * u) : ~0u;
#pragma unroll
      for (int u = 0; u < EV; ++u) ev[u] = lane + 32 * u < (int)cur.dv.z ? __ldg(p.pool.arena + cur.dv.x + lane + 32 * u) : ~0u;
      if (i + 1 < n) {
        load(nxt, pp1);
        pp1 = i + 2 < n ? phys_of(i + 2) : -1;
      }
      const int valid = min(S, tokens - (PAGES * i + w) * S);  // tokens of the page that are attended
      // ---- K
      {
        const int c = 2 * i, s = c % STAGES;
        if (c >= STAGES) ok = tc::wait_warp(&sm.kv_empty[s], ((c / STAGES) & 1) ^ 1, abort);
        if (!ok) break;
        const uint32_t base = smem_u32(sm.kv[s]), at = base + store0, slab = base + 16 * w * 128;
        if (cur.phys >= 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t tab = smem_u32(sm.klut) + 2048u * half + 1024u * (half ^ j);
            if (BK == 4) {
              const uint32_t low = (64u * half + 32u * (half ^ j)) * 0x01010101u;
#pragma unroll
              for (int u = 0; u < 4; ++u) sts128(at ^ (64u * j + 16u * u), lut8_nib<32>(cur.k[(4 * j + u) % WK], low, tab, 256u * u));
            } else {
              const uint32_t low = 64u * half * 0x01010101u;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint4 o0, o1;
                lut8_pair<64>(cur.k[(2 * j + u) % WK], low, tab, 512u * u, o0, o1);
                sts128(at ^ (64u * j + 32u * u), o0);
                sts128(at ^ (64u * j + 32u * u + 16u), o1);
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < EK; ++u)
            if (lane + 32 * u < (int)cur.dk.z) patch(slab, ek[u], S);
          for (int e = lane + 32 * EK; e < (int)cur.dk.z; e += 32) patch(slab, __ldg(p.pool.arena + cur.dk.x + e), S);
        } else {  // past the item's pages (masked), or a page id out of range (flagged)
#pragma unroll
          for (int u = 0; u < 8; ++u) sts128(at ^ (16u * u), make_uint4(0u, 0u, 0u, 0u));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::arrive(&sm.kv_full[s]);
      }
      // ---- V; rows that are not attended are zeroed (P is 0 there, but 0 * inf is not)
      {
        const int c = 2 * i + 1, s = c % STAGES;
        if (c >= STAGES) ok = tc::wait_warp(&sm.kv_empty[s], ((c / STAGES) & 1) ^ 1, abort);
        if (!ok) break;
        const uint32_t base = smem_u32(sm.kv[s]), at = base + store0, slab = base + 16 * w * 128;
        if (cur.phys >= 0) {
          const int64_t pos0 = (int64_t)(p.vphys ? cur.phys : page0 + PAGES * i + w) * S;
          const bool tail = pos0 >= Tc - 1;  // every token of the page reads the last row
          if (!tail) {
            const int L = p.sc.levels_v;
            __syncwarp();  // the tables' last readers are done
            for (int x = lane; x < S * 16; x += 32) {
              const int64_t row = min(pos0 + (x >> 4), (int64_t)Tc - 1);
              sm.vlut[w][x] = (x & 15) < L ? p.sc.v_poles[((int64_t)h * Tc + row) * L + (x & 15)] : (uint16_t)0;
            }
            __syncwarp();
          }
          const uint32_t vt = smem_u32(sm.vlut[w]) + 256u * (t >> 3), vlow = 32u * t7 * 0x01010101u;
          const bool mine = t < valid;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (BV == 4) {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const uint32_t cw = cur.v[(4 * j + u) % WV];
                uint4 o = tail ? lut8_reg(cw, lb, hb) : lut8_nib<0>(cw, vlow, vt, 0u);
                if (!mine) o = make_uint4(0u, 0u, 0u, 0u);
                sts128(at ^ (64u * j + 16u * u), o);
              }
            } else {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint32_t cw = cur.v[(2 * j + u) % WV];
                uint4 o0, o1;
                if (tail) lut8_pair<0>(cw, 0u, smem_u32(sm.vpair), 0u, o0, o1);
                else lut16_crumb<0>(cw, vlow, vt, 0u, o0, o1);
                if (!mine) o0 = o1 = make_uint4(0u, 0u, 0u, 0u);
                sts128(at ^ (64u * j + 32u * u), o0);
                sts128(at ^ (64u * j + 32u * u + 16u), o1);
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < EV; ++u)
            if (lane + 32 * u < (int)cur.dv.z) patch(slab, ev[u], valid);
          for (int e = lane + 32 * EV; e < (int)cur.dv.z; e += 32) patch(slab, __ldg(p.pool.arena + cur.dv.x + e), valid);
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u) sts128(at ^ (16u * u), make_uint4(0u, 0u, 0u, 0u));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::arrive(&sm.kv_full[s]);
      }
      cur = nxt;
    }
  } else {
    tc::regs_dec<48>();
    if (warp == 16) {
      // ---- matrix products
      constexpr uint32_t ids = tc::idesc_f16(0, ROWS, KT, 0), idv = tc::idesc_f16(0, ROWS, D, 1);
      auto qk = [&](int q, int tile, int stage) {
        const uint32_t qa = smem_u32(sm.q[tile]), ka = smem_u32(sm.kv[stage]);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * HALF + (k % 4) * 32;
          tc::mma_ss(tmem + 128 * q, tc::desc128(qa + off, 0), tc::desc128(ka + off, 0), ids, k > 0);
        }
        tc::commit(&sm.s_full[q]);
      };
      auto pv = [&](int q, int stage, bool more) {
        const uint32_t va = smem_u32(sm.kv[stage]);
#pragma unroll
        for (int k = 0; k < KT / 16; ++k)
          tc::mma_ts(tmem + 256 + 128 * q, tmem + 128 * q + 8 * k, tc::desc128(va + 2048 * k, HALF), idv, more || k > 0);
      };
      auto full = [&](int c) { return tc::wait_warp(&sm.kv_full[c % STAGES], (c / STAGES) & 1, abort); };
      bool ok = tc::wait_warp(&sm.q_full[0], 0, abort);
      if (two && ok) ok = tc::wait_warp(&sm.q_full[1], 0, abort);
      if (two) {
        // tile q of both uses every key tile
        if (ok) ok = full(0);
        if (ok && lane == 0) {
          tc::fence_after();
          qk(0, 0, 0);
          qk(1, 1, 0);
          tc::commit(&sm.kv_empty[0]);
        }
        for (int i = 0; i < n && ok; ++i) {
          const int cv = 2 * i + 1, ck = 2 * i + 2;
          ok = full(cv);
          if (ok && i + 1 < n) ok = full(ck);
          for (int q = 0; q < 2 && ok; ++q) {
            ok = tc::wait_warp(&sm.p_full[q], i & 1, abort);
            if (ok && lane == 0) {
              tc::fence_after();
              pv(q, cv % STAGES, i > 0);
              if (i + 1 < n) qk(q, q, ck % STAGES);
              else tc::commit(&sm.o_full[q]);
            }
            __syncwarp();
          }
          if (ok && lane == 0) {
            tc::commit(&sm.kv_empty[cv % STAGES]);
            if (i + 1 < n) tc::commit(&sm.kv_empty[ck % STAGES]);
          }
          __syncwarp();
        }
      } else {
        // key tile i belongs to stream i & 1
        for (int i = 0; i < 2 && i < n && ok; ++i) {
          ok = full(2 * i);
          if (ok && lane == 0) {
            tc::fence_after();
            qk(i, 0, (2 * i) % STAGES);
            tc::commit(&sm.kv_empty[(2 * i) % STAGES]);
          }
          __syncwarp();
        }
        for (int i = 0; i < n && ok; ++i) {
          const int q = i & 1, cv = 2 * i + 1, ck = 2 * (i + 2);
          ok = full(cv);
          if (ok) ok = tc::wait_warp(&sm.p_full[q], (i >> 1) & 1, abort);
          if (ok && lane == 0) {
            tc::fence_after();
            pv(q, cv % STAGES, i > 1);
            tc::commit(&sm.kv_empty[cv % STAGES]);
            if (i + 2 >= n) tc::commit(&sm.o_full[q]);
          }
          __syncwarp();
          if (ok && i + 2 < n) {
            ok = full(ck);
            if (ok && lane == 0) {
              tc::fence_after();
              qk(q, 0, ck % STAGES);
              tc::commit(&sm.kv_empty[ck % STAGES]);
            }
            __syncwarp();
          }
        }
      }
      if (lane == 0) tc::commit(&sm.drain);  // no product may be in flight when TMEM is freed
      __syncwarp();
      (void)mbar_wait(&sm.drain, 0);
    } else if (warp == 17 && lane == 0) {
      // ---- query tiles: TQ sequences x G heads
      const int nq = two ? 2 : 1;
      for (int q = 0; q < nq; ++q) {
        mbar_arrive_expect_tx(&sm.q_full[q], TQ * G * D * 2);
        for (int u = 0; u < 2; ++u) tc::tma3(sm.q[q] + u * HALF, &p.mq, 64 * u, h * G, seq0 + q * TQ, &sm.q_full[q]);
      }
      for (int q = 0; q < nq; ++q) (void)mbar_wait(&sm.q_full[q], 0);  // landed before the CTA's memory goes
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 16) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && sm.abort) set_err(p.err, HX_DEV_ERR_TIMEOUT);
}

// Joins a row's partials: weights 2^(m - M), M the largest m; one CTA a row,
// its warps take every fourth partial.
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
  const int n = len == 0 || bad ? 0 : 2 * p.n_splits + (len > p.prefix ? 2 : 0);
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
      if (wj != 0.0f) {  // a place without a partial holds nothing
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

int default_splits(int H, int RB, int tiles) {
  // one wave of prefix CTAs (one fits an SM); at most one split per key tile
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
  return (int64_t)(2 * n_splits + 2) * B * H * group * (px::D + 2) * 4;
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
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)(2 * n_splits + 2) * rows * px::D);
  p.err = dev_err;
  const int64_t grid = (int64_t)H * p.RB * n_splits + (int64_t)B * H;
  if (grid > 0x7fffffffll || rows > 0x7fffffffll) return HX_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  constexpr int smem = (int)sizeof(px::Smem) + 1024;
  static_assert(smem <= 232448, "a CTA has 227 KB of shared memory");
  auto kern = pool->bits_k == 4 ? (pool->bits_v == 4 ? px::prefix_kernel<4, 4> : px::prefix_kernel<4, 2>)
                                : (pool->bits_v == 4 ? px::prefix_kernel<2, 4> : px::prefix_kernel<2, 2>);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    (void)cudaGetLastError();
    return HX_ERR_LAUNCH;
  }
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
