// Causal attention over whole prompts, packed back to back, grouped heads.
//
//   s_ij = scale * q_i . k_j  (j <= i, same sequence),  o_i = sum_j softmax(s_i)_j v_j,
//   lse_i = log sum_j exp(s_ij)
//
// One CTA = (two tiles of 128 query rows, KV head, sequence). A row is one
// (token, head of the group) pair, TQ = 128 / G tokens a tile, so all heads of
// a group share the K and V tiles and short prompts fill the tiles' rows. Keys
// stream in tiles of 128. Per tile and key tile:
//   S = Q K^T    tcgen05.mma, both operands in shared memory (tensor-map loads,
//                128-byte swizzle), S (128 x 128 fp32) in TMEM
//   P            a warpgroup holds one row of S a thread: running maximum and
//                sum in fp32 (exp2 domain), P rounded to the inputs' type (the
//                matrix unit's operand; the sum keeps the fp32 values) and
//                stored over S in TMEM. The maximum used for P moves only when
//                a score passes it by 2^8, so O is rescaled rarely
//   O += P V     tcgen05.mma, P from TMEM, V from shared memory
// The two query tiles alternate on the tensor core: one tile's products run
// under the other's softmax. The products of a tile are issued in the order
// PV(i), S(i + 1), so that S(i + 1) complete means O(i) complete.
//
// What bounds it: 20,011 tokens (fp16, 28 heads on 4) take 2,190 us, 1,310
// TFLOP/s of unmasked products (cuBLAS 1,668 in a burst), at burst clocks and
// 2,535 under the power cap (1,132; cuBLAS 1,395). A key tile's products are
// 2,700 of its about 3,500 cycles: those with both operands in shared memory run at
// 106 cycles of 64; the rest is the part of a tile's softmax (exponentials on
// the special-function unit: 1,024 cycles at least) that the other tile's
// products do not cover.
//
// Masked places: a masked score is replaced by -inf, never added to, so K there
// may hold anything. V there meets P = 0 in the product, and 0 * inf is NaN: in
// the key tiles that hold masked places a warp replaces rows past the
// sequence's end and non-finite values by 0 before the product, and rows
// allowed to see a non-finite value get it added at the end (P > 0 there).
#include "tcgen.cuh"
#include "tmap.cuh"

namespace hx {
namespace pr {

constexpr int NTHREADS = 384;   // 2 softmax warpgroups; 2 product warps, the load warp, the V-check warp
constexpr int STAGES = 4;       // K and V tiles in flight
constexpr int KT = 128;         // keys per tile
constexpr int ROWS = 128;       // query rows per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.0f;  // P <= 2^8 before the maximum moves
constexpr int kOutRow = 80;     // bytes of a staged output row: 64, and 16 so that eight rows meet all banks

// A work item: two tiles of query rows of one (sequence, KV head).
struct Item {
  int h, s0, len, t0;  // KV head; first row and tokens of the sequence; first token of the item (len 0: no more items)
};

template <int D>
struct Smem {
  alignas(1024) uint8_t q[2][ROWS * D * 2];
  alignas(1024) uint8_t kv[STAGES][KT * D * 2];
  alignas(16) uint8_t out[8][32 * kOutRow];  // 32 columns of a softmax warp's output rows
  alignas(16) uint32_t answer[2][4];         // next_cta
  Item item[2];
  uint64_t q_full[2], q_empty[2], kv_full[STAGES], kv_empty[STAGES], s_full[2], p_half[2], p_full[2], o_full[2], turn[2];
  uint64_t v_clean[3], item_full[2], item_empty[2], next, drain;
  uint32_t tmem, abort, bad_v[2];
};

struct Params {
  CUtensorMap mq, mk, mv;
  const int32_t* start;
  int B, T, H, G, TQ;
  float c;  // softmax scale * log2 e
  const uint16_t* v;
  int64_t v_st, v_sh;
  uint16_t* out;
  float* lse;
  uint32_t* err;
};

// Work item of a slot. Sequence b's tiles are slots f(b) .. f(b) + ceil(len / n)
// - 1 with f(b) = floor(start_b / n) + b, n tokens a CTA: ceil(len_b / n) <=
// floor(start_{b+1} / n) - floor(start_b / n) + 1, so slots never meet and no
// prefix sum over the batch is needed; floor(T / n) + B slots hold all. b is the
// last with f(b) <= slot, found by the warp 32 candidates at a time.
HX_DEVINL int find_seq(const int32_t* start, int B, int n, int slot) {
  const int lane = lane_id();
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int b = lo + lane * step;
    const bool le = b < hi && start[b] / n + b <= slot;
    const uint32_t m = __ballot_sync(0xffffffffu, le);
    const int last = m ? 31 - __clz(m) : 0;
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

template <bool BF16>
HX_DEVINL uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// bits of the 16-bit halves whose value is not finite
template <bool BF16>
HX_DEVINL uint32_t nonfinite2(uint32_t x) {
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return ((x & e) == e ? 0xFFFFu : 0u) | (((x >> 16) & e) == e ? 0xFFFF0000u : 0u);
}
// a * 0 + c on both halves
template <bool BF16>
HX_DEVINL uint32_t times_zero(uint32_t a, uint32_t c) {
  uint32_t r;
  if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0u), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0u), "r"(c));
  return r;
}
template <bool BF16>
HX_DEVINL float to_float(uint16_t x) {
  return BF16 ? __uint_as_float((uint32_t)x << 16) : h2f(x);
}

// Stage and parity of every second tile of the ring (K tiles, or V tiles).
struct Ring {
  int stage, phase;
  HX_DEVINL void next() {
    stage += 2;
    if (stage >= STAGES) stage -= STAGES, phase ^= 1;
  }
};

// What the roles derive from an item.
struct Work {
  int h, s0, len, t0, nq, n, i_mask;  // query tiles with tokens; key tiles; the first of them with masked places
  HX_DEVINL bool read(const volatile Item& it, int TQ) {
    h = it.h, s0 = it.s0, len = it.len, t0 = it.t0;
    nq = t0 + TQ < len ? 2 : 1;
    n = (min(t0 + 2 * TQ, len) + KT - 1) / KT;
    i_mask = min((t0 + 1) / KT, n - 1);
    return len > 0;
  }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1) prompt_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int TQ = p.TQ, G = p.G, per = 2 * TQ;

  if (warp == 8) {
    if (lane == 0) {
      for (int q = 0; q < 2; ++q) {
        mbar_init(&sm.q_full[q], 1);
        mbar_init(&sm.q_empty[q], 1);
        mbar_init(&sm.s_full[q], 1);
        mbar_init(&sm.p_full[q], 4);
        mbar_init(&sm.p_half[q], 4);
        mbar_init(&sm.o_full[q], 1);
        mbar_init(&sm.turn[q], 1);
        mbar_init(&sm.item_full[q], 1);
        mbar_init(&sm.item_empty[q], 11);  // 8 softmax warps, 2 product warps, the V-check warp
      }
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&sm.kv_full[s], 1);
        mbar_init(&sm.kv_empty[s], 2 + (s & 1));  // both query tiles' products; for V (odd stages) the V-check warp
      }
      for (int i = 0; i < 3; ++i) mbar_init(&sm.v_clean[i], 1);
      mbar_init(&sm.next, 1);
      mbar_init(&sm.drain, 2);
      sm.abort = 0u;
      fence_mbar_init();
    }
    __syncwarp();
    tc::tmem_alloc(&sm.tmem, 512);
  }
  if (warp == 9 && lane == 0) {
    tc::prefetch_map(&p.mq);
    tc::prefetch_map(&p.mk);
    tc::prefetch_map(&p.mv);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sm.tmem;
  volatile uint32_t* abort = &sm.abort;
  constexpr int HALF = KT * 128;  // bytes of 128 rows of 64 elements
  constexpr int NH = D / 64;
  Work w;

  if (warp < 8) {
    // ---- softmax: warpgroup q holds tile q's rows, one a thread
    tc::regs_inc<216>();
    const int q = warp >> 2, r = threadIdx.x & 127;
    const uint32_t sb = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * q;
    const uint32_t ob = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 256 + 128 * q;
    const int rt = r / G, rg = r - rt * G;  // token of the row in the tile, head of the group
    const uint32_t stage = smem_u32(sm.out[warp]);
    int used = 0, done = 0;  // S tiles and O results of this warpgroup so far
    bool ok = true;
    for (int it = 0; ok; ++it) {
      ok = tc::wait_warp(&sm.item_full[it & 1], (it >> 1) & 1, abort);
      if (!ok || !w.read(sm.item[it & 1], TQ)) break;
      if (q < w.nq) {
        const int tile0 = w.t0 + q * TQ;        // lowest position of the tile
        const int ti = tile0 + rt;              // token of the row, in the sequence
        const bool live = r < TQ * G && ti < w.len;
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; i < w.n; ++i, ++used) {
          ok = tc::wait_warp(&sm.s_full[q], used & 1, abort);
          if (!ok) break;
          tc::fence_after();
          uint32_t s[KT];
#pragma unroll
          for (int u = 0; u < 4; ++u) tc::ld32(s + 32 * u, sb + 32 * u);
          tc::wait_ld();
          if (KT * i + KT - 1 > tile0) {  // masked places: keys past the row's position
            const int lim = ti - KT * i;
#pragma unroll
            for (int j = 0; j < KT; ++j) s[j] = j <= lim ? s[j] : 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < KT; j += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              mx[u] = fmaxf(mx[u], fmaxf(__uint_as_float(s[j + 2 * u]), __uint_as_float(s[j + 2 * u + 1])));
          const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool move = (mt - m) * p.c > kSlack;  // also the first finite maximum (m = -inf)
          if (__any_sync(0xffffffffu, move)) {
            const float mn = move ? mt : m;
            const float a = move ? tc::ex2((m - mn) * p.c) : 1.0f;
            m = mn;
            l *= a;
            if (i > 0) {  // O(i - 1) is complete: S(i) was issued after it
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
          for (int hf = 0; hf < 2; ++hf) {  // the product over the first 64 keys starts while the others' exponentials run
            uint32_t pk[KT / 4];
#pragma unroll
            for (int j = 0; j < KT / 2; j += 2) {
              float x, y;
              tc::f2_unpack(
                  tc::f2_fma(tc::f2_pack(__uint_as_float(s[64 * hf + j]), __uint_as_float(s[64 * hf + j + 1])), c2, mb2), x, y);
              x = tc::ex2(x);
              y = tc::ex2(y);
              sum[(j >> 1) & 1] = tc::f2_add(sum[(j >> 1) & 1], tc::f2_pack(x, y));
              pk[j >> 1] = pack2<BF16>(x, y);
            }
            tc::st32(sb + 32 * hf, pk);
            tc::wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::arrive(hf == 0 ? &sm.p_half[q] : &sm.p_full[q]);
          }
          float x, y;
          tc::f2_unpack(tc::f2_add(sum[0], sum[1]), x, y);
          l += x + y;
        }
        // ---- O / l
        if (ok) ok = tc::wait_warp(&sm.o_full[q], done++ & 1, abort);
        if (ok) {
          tc::fence_after();
          const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
          const int64_t row = ((int64_t)(w.s0 + ti) * p.H + w.h) * G + rg;
          const bool bad = *(volatile uint32_t*)&sm.bad_v[it & 1] != 0u;
#pragma unroll 1
          for (int u = 0; u < D / 32; ++u) {
            uint32_t o[32];
            tc::ld32(o, ob + 32 * u);
            tc::wait_ld();
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(o[j]) * inv;
            // through shared memory, so that four lanes write 64 bytes of a row and a store meets 8 rows, not 32
            // (a row a lane: 5500 cycles for the tile's output, as long as one and a half key tiles)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * kOutRow + 16 * j),
                           "r"(pack2<BF16>(f[8 * j], f[8 * j + 1])), "r"(pack2<BF16>(f[8 * j + 2], f[8 * j + 3])),
                           "r"(pack2<BF16>(f[8 * j + 4], f[8 * j + 5])), "r"(pack2<BF16>(f[8 * j + 6], f[8 * j + 7]))
                           : "memory");
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int from = 8 * j + (lane >> 2);
              const int64_t to = __shfl_sync(0xffffffffu, live ? row : -1, from);
              uint4 x;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                           : "r"(stage + from * kOutRow + 16 * (lane & 3))
                           : "memory");
              if (to >= 0) *reinterpret_cast<uint4*>(p.out + to * D + 32 * u + 8 * (lane & 3)) = x;
            }
            __syncwarp();
          }
          if (bad) {  // rare: non-finite V that the row sees in the masked tiles, over the finite part written above
            __syncwarp();
            if (live) {
#pragma unroll 1
              for (int c = 0; c < D; ++c) {
                float sum = 0.0f;
#pragma unroll 1
                for (int key = w.i_mask * KT; key <= ti; ++key) {
                  const float x = to_float<BF16>(p.v[(int64_t)(w.s0 + key) * p.v_st + w.h * p.v_sh + c]);
                  if (!(fabsf(x) < INFINITY)) sum += x;
                }
                if (sum != 0.0f) p.out[row * D + c] = (uint16_t)pack2<BF16>(to_float<BF16>(p.out[row * D + c]) + sum, 0.0f);
              }
            }
          }
          if (live && p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (m * p.c + log2f(l)) * kLn2;
          tc::fence_before();
        }
      }
      __syncwarp();
      if (lane == 0) tc::arrive(&sm.item_empty[it & 1]);
    }
  } else {
    tc::regs_dec<72>();
    if (warp == 8 || warp == 10) {
      // ---- matrix products: a warp for each query tile, since issuing blocks (68 cycles a product at 64 of work) and
      // a wait that is over already still costs 200 to 300: with one warp for both tiles the tensor core stood still
      // for a third of the time. elect.sync tells the compiler that a single lane runs (a test of the lane number
      // cost 8%).
      const int q = warp == 8 ? 0 : 1;
      constexpr uint32_t ids = tc::idesc_f16(BF16, ROWS, KT, 0), idv = tc::idesc_f16(BF16, ROWS, D, 1);
      const uint32_t ts = tmem + 128 * q, to = tmem + 256 + 128 * q;
      Ring rk = {0, 0}, rv = {1, 0};  // stages of the next K and V tile
      int vc = 0, qc = 0, pc = 0, turns = 0;  // checked V tiles, items, P tiles and turns so far
      if (q == 1 && lane == 0) tc::arrive(&sm.turn[0]);
      auto qk = [&](int stage) {
        const uint32_t qa = smem_u32(sm.q[q]), ka = smem_u32(sm.kv[0]) + stage * (KT * D * 2);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * HALF + (k % 4) * 32;
          tc::mma_ss(ts, tc::desc128(qa + off, 0), tc::desc128(ka + off, 0), ids, k > 0);
        }
        tc::commit(&sm.s_full[q]);
        tc::commit(&sm.kv_empty[stage]);
      };
      // checked tile m completes barrier m % 3. The check and either product warp are at most two key tiles apart, not
      // three (the ring has STAGES < 6 stages), so no warp meets a barrier one phase too early or too late
      static_assert(STAGES < 6, "three barriers for checked tiles");
      auto v_clean = [&](int m) { return tc::wait_warp(&sm.v_clean[m % 3], (m / 3) & 1, abort); };
      auto full = [&](const Ring& r) { return tc::wait_warp(&sm.kv_full[r.stage], r.phase, abort); };
      bool ok = true;
      for (int it = 0; ok; ++it) {
        ok = tc::wait_warp(&sm.item_full[it & 1], (it >> 1) & 1, abort);
        if (!ok || !w.read(sm.item[it & 1], TQ)) break;
        if (q >= w.nq) {  // no rows: only give the tiles back
          for (int i = 0; i < 2 * w.n && ok; ++i) {
            Ring& r = i & 1 ? rv : rk;
            ok = full(r);
            if (ok && lane == 0) tc::arrive(&sm.kv_empty[r.stage]);
            r.next();
          }
        } else {
          ok = full(rk) && tc::wait_warp(&sm.q_full[q], qc++ & 1, abort);
          if (ok && tc::elect()) {
            tc::fence_after();
            qk(rk.stage);
            if (w.n == 1) tc::commit(&sm.q_empty[q]);
          }
          __syncwarp();
          rk.next();
          for (int i = 0; i < w.n && ok; ++i) {
            const bool more = i + 1 < w.n, check = i >= w.i_mask;
            ok = full(rv);
            if (ok && more) ok = full(rk);
            if (ok && check) ok = v_clean(vc++);
            // the tiles take turns, PV and S of one in a row: left to interleave, both finish together, both
            // softmaxes run together, and the tensor core waits for them (4280 cycles a key tile). The turn comes before P
            // as a rule, so P is waited for last (2%)
            if (ok && w.nq == 2) ok = tc::wait_warp(&sm.turn[q], turns++ & 1, abort);
            if (ok) ok = tc::wait_warp(&sm.p_half[q], pc & 1, abort);
            if (ok && tc::elect()) {
              tc::fence_after();
              const uint32_t va = smem_u32(sm.kv[0]) + rv.stage * (KT * D * 2);
#pragma unroll
              for (int k = 0; k < KT / 32; ++k)
                tc::mma_ts(to, ts + 8 * k, tc::desc128(va + 2048 * k, HALF), idv, i > 0 || k > 0);
            }
            if (ok) ok = tc::wait_warp(&sm.p_full[q], pc++ & 1, abort);
            if (ok && tc::elect()) {
              tc::fence_after();
              const uint32_t va = smem_u32(sm.kv[0]) + rv.stage * (KT * D * 2);
#pragma unroll
              for (int k = KT / 32; k < KT / 16; ++k)
                tc::mma_ts(to, ts + 8 * k, tc::desc128(va + 2048 * k, HALF), idv, 1);
              tc::commit(&sm.kv_empty[rv.stage]);
              if (more) {
                qk(rk.stage);
                if (i + 2 == w.n) tc::commit(&sm.q_empty[q]);  // the item's last use of the query tile
              } else {
                tc::commit(&sm.o_full[q]);
              }
            }
            __syncwarp();
            if (ok && w.nq == 2 && lane == 0) tc::arrive(&sm.turn[q ^ 1]);
            rv.next();
            if (more) rk.next();
          }
        }
        if (q >= w.nq) vc += w.n - w.i_mask;
        if (lane == 0) tc::arrive(&sm.item_empty[it & 1]);
      }
      if (tc::elect()) tc::commit(&sm.drain);  // no product may be in flight when TMEM is freed
      __syncwarp();
      (void)mbar_wait(&sm.drain, 0);
    } else if (warp == 9) {
      // ---- work items (this CTA's own, then those of CTAs not started yet), and their loads: Q tiles, K0 V0 K1 V1 ...
      bool ok = true;
      int c = 0, it = 0, requests = 0, qc[2] = {0, 0};
      auto load = [&](const CUtensorMap* map, int key) {
        const int s = c % STAGES;
        if (c >= STAGES) ok = tc::wait(&sm.kv_empty[s], ((c / STAGES) & 1) ^ 1, abort);
        if (!ok) return;
        mbar_arrive_expect_tx(&sm.kv_full[s], KT * D * 2);
#pragma unroll
        for (int u = 0; u < NH; ++u) tc::tma3(sm.kv[s] + u * HALF, map, 64 * u, w.h, w.s0 + key, &sm.kv_full[s]);
        ++c;
      };
      auto load_q = [&](int q) {
        if (qc[q] > 0) ok = tc::wait(&sm.q_empty[q], (qc[q] & 1) ^ 1, abort);
        if (!ok) return;
        mbar_arrive_expect_tx(&sm.q_full[q], TQ * G * D * 2);
#pragma unroll
        for (int u = 0; u < NH; ++u)
          tc::tma3(sm.q[q] + u * HALF, &p.mq, 64 * u, w.h * G, w.s0 + w.t0 + q * TQ, &sm.q_full[q]);
        ++qc[q];
      };
      int cta = blockIdx.x;
      for (int asked = 0; ok; ++asked) {
        if (cta >= 0 && lane == 0) {
          fence_proxy_async();  // the answer's place was read before
          tc::next_cta_request(sm.answer[asked & 1], &sm.next);
          ++requests;
        }
        Item x = {0, 0, 0, 0};
        if (cta >= 0) {
          const int slot = (int)(gridDim.x / p.H) - 1 - cta / p.H;
          const int b = find_seq(p.start, p.B, per, slot);
          x.h = cta % p.H;
          x.s0 = p.start[b];
          x.len = p.start[b + 1] - x.s0;
          x.t0 = (slot - x.s0 / per - b) * per;
          if (x.s0 < 0 || x.len < 0 || x.len > p.T - x.s0) {
            if (lane == 0) set_err(p.err, HX_DEV_ERR_BOUNDS);
            x.len = 0;
          }
          if (x.t0 < 0 || x.t0 >= x.len) x.len = 0;
        }
        if (x.len > 0 || cta < 0) {  // an item, or the word that there are no more
          if (it >= 2) ok = tc::wait_warp(&sm.item_empty[it & 1], ((it >> 1) & 1) ^ 1, abort);
          if (ok && lane == 0) {
            sm.item[it & 1] = x;
            sm.bad_v[it & 1] = 0u;
            tc::arrive(&sm.item_full[it & 1]);
          }
          __syncwarp();
          ++it;
        }
        if (cta < 0) break;
        if (ok && x.len > 0) {
          w.read(x, TQ);
          if (lane == 0) {
            load_q(0);
            if (ok) load(&p.mk, 0);
            if (ok && w.nq > 1) load_q(1);
            if (ok) load(&p.mv, 0);
            for (int i = 1; i < w.n && ok; ++i) {
              load(&p.mk, KT * i);
              if (ok) load(&p.mv, KT * i);
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
        if (!tc::wait_warp(&sm.next, asked & 1, abort)) ok = false;
        cta = ok ? tc::next_cta(sm.answer[asked & 1]) : -1;
      }
      if (*abort && lane == 0) {  // given up: let what is in flight land before the CTA's memory goes
        for (int q = 0; q < 2; ++q)
          if (qc[q]) (void)mbar_wait(&sm.q_full[q], (qc[q] - 1) & 1);
        for (int s = max(0, c - STAGES); s < c; ++s) (void)mbar_wait(&sm.kv_full[s % STAGES], (s / STAGES) & 1);
        if (requests) (void)mbar_wait(&sm.next, (requests - 1) & 1);
      }
      __syncwarp();
    } else {
      // ---- V tiles with masked places: rows past the sequence and non-finite values to 0. The warp sees every V tile
      // as it lands (and gives back its hold on it), so the check is off the products' path.
      static_assert(STAGES % 2 == 0, "V tiles on odd stages");
      int vc = 0;
      Ring rv = {1, 0};
      bool ok = true;
      for (int it = 0; ok; ++it) {
        ok = tc::wait_warp(&sm.item_full[it & 1], (it >> 1) & 1, abort);
        if (!ok || !w.read(sm.item[it & 1], TQ)) break;
        for (int i = 0; i < w.n; ++i, rv.next()) {
          const int s = rv.stage;
          ok = tc::wait_warp(&sm.kv_full[s], rv.phase, abort);
          if (!ok) break;
          if (i < w.i_mask) {
            if (lane == 0) tc::arrive(&sm.kv_empty[s]);
            continue;
          }
          // chunk u: 16 bytes of row (u >> 3) & 127. x * 0 is NaN exactly for a value that is not finite, so a packed
          // multiply-add per pair looks at a chunk in four instructions (a test of each exponent took 4 us a tile)
          const int rows = min(KT, w.len - KT * i), first = lane;
          uint4* tile = reinterpret_cast<uint4*>(sm.kv[s]);
          uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
          for (int u = first; u < KT * D / 8; u += 32) {  // rows to be zeroed are looked at too: at worst once more below
            const uint4 x = tile[u];
            acc[0] = times_zero<BF16>(x.x, acc[0]);
            acc[1] = times_zero<BF16>(x.y, acc[1]);
            acc[2] = times_zero<BF16>(x.z, acc[2]);
            acc[3] = times_zero<BF16>(x.w, acc[3]);
          }
#pragma unroll
          for (int hf = 0; hf < NH; ++hf)
            for (int u = hf * (KT * 8) + rows * 8 + lane; u < (hf + 1) * (KT * 8); u += 32)
              tile[u] = make_uint4(0u, 0u, 0u, 0u);
          __syncwarp();
          uint32_t found = 0u;
          if (nonfinite2<BF16>(acc[0]) | nonfinite2<BF16>(acc[1]) | nonfinite2<BF16>(acc[2]) | nonfinite2<BF16>(acc[3])) {
            for (int u = first; u < KT * D / 8; u += 32) {
              const uint4 x = tile[u];
              const uint4 e = make_uint4(nonfinite2<BF16>(x.x), nonfinite2<BF16>(x.y), nonfinite2<BF16>(x.z),
                                         nonfinite2<BF16>(x.w));
              if (e.x | e.y | e.z | e.w) {
                found = 1u;
                tile[u] = make_uint4(x.x & ~e.x, x.y & ~e.y, x.z & ~e.z, x.w & ~e.w);
              }
            }
          }
          if (found) sm.bad_v[it & 1] = 1u;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tc::arrive(&sm.v_clean[vc % 3]);
            tc::arrive(&sm.kv_empty[s]);
          }
          ++vc;
        }
        __syncwarp();
        if (lane == 0) tc::arrive(&sm.item_empty[it & 1]);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && sm.abort) set_err(p.err, HX_DEV_ERR_TIMEOUT);
}

template <int D, bool BF16>
int launch(const Params& p, int64_t grid, cudaStream_t s) {
  constexpr int smem = (int)sizeof(Smem<D>) + 1024;
  static_assert(smem <= 232448, "a CTA has 227 KB of shared memory");
  static unsigned long long done = 0;
  if (!allow_smem(prompt_kernel<D, BF16>, smem, done)) return HX_ERR_LAUNCH;
  prompt_kernel<D, BF16><<<(unsigned)grid, NTHREADS, smem, s>>>(p);
  HX_LAUNCH_CHECK();
  return HX_OK;
}

}  // namespace pr
}  // namespace hx

using namespace hx;

extern "C" {

HX_API int hx_prompt_attn(void* stream, int32_t dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                          const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                          int64_t v_token_stride, int64_t v_head_stride, const int32_t* query_start, int32_t B,
                          int32_t T, int32_t H, int32_t group, int32_t D, float softmax_scale, void* out, float* lse,
                          uint32_t* dev_err) {
  if (B < 0 || T < 0 || H < 1 || group < 1) return HX_ERR_ARG;
  if (!(softmax_scale > 0.0f) || softmax_scale > 3.0e38f) return HX_ERR_ARG;
  if (dtype != 1 && dtype != 2) return HX_ERR_UNSUPPORTED;
  if ((D != 64 && D != 128) || group > pr::ROWS) return HX_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return HX_OK;
  if (!q || !k || !v || !query_start || !out) return HX_ERR_ARG;
  const int64_t strides[6] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                              v_head_stride};
  for (int64_t s : strides)
    if (s < D || s % 8 || s >= (1ll << 38)) return HX_ERR_ARG;
  for (const void* x : {q, k, v, (const void*)out})
    if (reinterpret_cast<uintptr_t>(x) % 16) return HX_ERR_ARG;
  pr::Params p;
  const bool bf = dtype == 2;
  p.TQ = pr::ROWS / group;
  if (!make_tmap3(&p.mq, bf, q, D, H * group, T, q_head_stride, q_token_stride, group, p.TQ) ||
      !make_tmap3(&p.mk, bf, k, D, H, T, k_head_stride, k_token_stride, 1, pr::KT) ||
      !make_tmap3(&p.mv, bf, v, D, H, T, v_head_stride, v_token_stride, 1, pr::KT))
    return HX_ERR_LAUNCH;
  p.start = query_start;
  p.B = B;
  p.T = T;
  p.H = H;
  p.G = group;
  p.c = softmax_scale * pr::kLog2e;
  p.v = reinterpret_cast<const uint16_t*>(v);
  p.v_st = v_token_stride;
  p.v_sh = v_head_stride;
  p.out = reinterpret_cast<uint16_t*>(out);
  p.lse = lse;
  p.err = dev_err;
  const int64_t grid = ((int64_t)T / (2 * p.TQ) + B) * H;
  if (grid > 0x7fffffffll) return HX_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (D == 128) return bf ? pr::launch<128, true>(p, grid, s) : pr::launch<128, false>(p, grid, s);
  return bf ? pr::launch<64, true>(p, grid, s) : pr::launch<64, false>(p, grid, s);
}

}  // extern "C"
