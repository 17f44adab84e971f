// Attention of 128-query tiles against a list of 128-key tiles on the tcgen05
// tensor cores (head_dim 128, bf16, GQA). Two kernels share the body:
//
//   fb_window_prefill_q{1,2}  packed prompts; key j is visible to the query at
//                             position i iff j <= i and (j > i - window or
//                             j < sinks); writes bf16 rows
//   fb_prefix_attn_q{1,2}     a decode batch against pages that a group of its
//                             sequences shares: the group's queries x G heads
//                             of one KV head are the rows of the tile. The
//                             pages are split over the CTAs of a cluster, which
//                             join their results through each other's shared
//                             memory; writes an unnormalised fp32 result and
//                             (max, sum) per row and head (a few, where a
//                             cluster's CTAs are not enough), from which
//                             attention_span.cu goes on
//
// Per key tile and 128-row query tile:
//   S = Q K^T          tcgen05.mma M=128 N=128 K=128, both from shared memory
//   softmax            one thread per row: the row's 128 scores are read from
//                      TMEM once into registers; running max m, sum l;
//                      p = exp2(s - m) goes back to TMEM as bf16 over S
//   O += P V           tcgen05.mma with P from TMEM (no shared-memory traffic
//                      for it), V MN-major from the image that TMA wrote
// A CTA holds QT query tiles: with QT = 2 they share every K/V tile and take
// turns, the tensor cores working on one tile's products while the other's
// 128 threads do its softmax; QT = 1 has half the shared memory and TMEM, and two
// CTAs per SM. A prefill's two tiles are two heads of one KV head: with an odd
// number of them, QT = 1. (Heads 32 / 8: 154 us with QT = 2, 216 with QT = 1 on 8192
// tokens, 47 and 64 on short prompts; 24 / 8, which has only QT = 1, 162 and 49.)
// The prefix kernel takes either, by the estimate of PrefixPlan. TMEM: QT x (128 columns S/P +
// 128 columns O).
//
// The MMA thread issues P_t V_i and then Q_t K_{i+1}, which overwrites P_t's
// columns: MMAs of one CTA execute in issue order. The commit behind Q_t K_{i+1}
// therefore also covers P_t V_i, so a softmax thread that has seen S_{i+1} may
// rescale O. A row's max moves only when a tile's max exceeds it by more than
// 8 (log2 units; p stays below 256, exact in the fp32 sum), so O is rarely
// rescaled.
//
// p is rounded to bf16 for the second product (half a step: relative 2^-8 of
// each term, with random signs), as much as the output's own rounding; the sum l
// is of the unrounded p, and it and both products accumulate in fp32.
//
// Roles: 4 QT softmax warps (a thread per query row), one TMA warp, one MMA warp,
// and for the two-tile prefill four warps that normalise and store an item's O
// while the softmax warps are at the next item (two more fill their warpgroup);
// elsewhere the softmax warps do that. With QT = 2 the other warps give registers
// to the softmax warps, which hold 128 scores each; even so each variant spills a
// few registers (24 to 200 bytes of stores a thread).
//
// Measured (B200): prefill of 8192 tokens, 32 / 8 heads, window 1024 and 4 sinks
// 154 to 163 us (129 GFLOP of visible pairs: 840 to 795 TFLOP/s), 184 us (700) where
// repeated calls bring the clocks down to the power cap; 13 prompts of 1 to 700
// tokens, window 128 48 us. Prefix of 32768 tokens for 128 rows of 64 / 8 heads 133 us
// (137 GFLOP, 1030 TFLOP/s); of 2048 tokens for 256 rows of 32 / 8 heads 21 us.
// Bound by the chain of a step rather than by a pipe: softmax 1900 clocks, signal
// to the MMA warp 440, P V and the next Q K^T 1020; two query tiles overlap their
// chains (the tensor pipe is busy 55% of a long prompt's 3700-clock steps), TMEM
// has no room for a third. Slower or within 2%: two threads per row; P handed over in halves; 1 in 2, 1 in
// 3 or no exponentials by polynomial; masks block by block; skipping masked
// blocks of 32 keys.
// No TMA multicast; every wait bounded (fb_common.cuh).
#include <type_traits>

#include "attn_tile.cuh"

FB_DEFINE_STATUS

using namespace fbk;

namespace {

constexpr int D = 128;
constexpr int PAGE = 64;
constexpr int BQ = 128;              // query rows per tile
constexpr int BK = 128;              // keys per tile
constexpr int HALF = 128 * 128;      // one 64-dim half of a 128-row tile: 128 rows x 128 B
constexpr int TILE = 2 * HALF;       // 128 rows x 128 dims bf16
constexpr float RESCALE_LOG2 = 8.f;  // lazy-rescale threshold
constexpr int EVERY_KEY = 0x3fffffff;
constexpr int MAX_CLUSTER = 8;
constexpr int FEW = 32;  // keys of a tile of nothing but sinks

// STAGE: bytes per row of the output that a warp stages for its stores (0: none).
template <int QT_, int STAGE_>
struct Smem {
  static constexpr int QT = QT_, STAGE = STAGE_;
  static constexpr int SLOTS = QT == 1 ? 2 : STAGE ? 4 : 5;  // ring of K_0, V_0, K_1, V_1, ...
  uint8_t q[QT][TILE];
  uint8_t kv[SLOTS][TILE];
  uint8_t stage[4][STAGE ? 32 * STAGE : 16];
  float l[QT][STAGE && QT == 2 ? BQ : 1];  // the rows' sums for the epilogue
  uint64_t q_full[QT], q_empty[QT], kv_full[SLOTS], kv_empty[SLOTS];
  uint64_t s_full[QT], p_full[QT], o_full[QT], l_full[QT], o_empty[QT];
  uint64_t mma_done;  // the products of an MMA warp that gave up
  uint32_t tmem;
  // (max, sum) of each row for the cluster's join: in q's memory, when the products are done
  __device__ __forceinline__ float2* ml(int t) { return reinterpret_cast<float2*>(q[0]) + t * BQ; }
};
using PrefixSmem1 = Smem<1, 0>;
using PrefixSmem2 = Smem<2, 0>;
using WindowSmem1 = Smem<1, 64>;
using WindowSmem2 = Smem<2, 256>;
static_assert(sizeof(PrefixSmem2) + 1024 <= 227 * 1024 && sizeof(WindowSmem2) + 1024 <= 227 * 1024,
              "host requests 227 KB of dynamic shared memory (2 tiles)");
static_assert(sizeof(PrefixSmem1) + 1024 <= 108 * 1024 && sizeof(WindowSmem1) + 1024 <= 108 * 1024,
              "host requests 108 KB of dynamic shared memory (1 tile)");

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for x in [-inf, 16], one of POLY_OF pairs of scores: the special-function
// unit gives 16 exponentials a clock and SM, as many as the two products of a tile
// take time for; some on the FMA pipes bring the softmax below the products.
// x = n + f, |f| <= 1/2; 2^f by the polynomial of degree 4 with the least relative
// error (2.7e-6, found by linear programming; p is rounded to 2^-8 next, and
// the sum l, which takes it as it is, is off by no more than that). x below
// -126 gives 2^-126 at least, and so does NaN: the caller sees to it that the sum
// of a row with such a score is NaN.
constexpr int POLY_OF = 4;
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 magic = make_float2(12582912.f, 12582912.f), unmagic = make_float2(-12582912.f, -12582912.f);
  const float2 t = __fadd2_rn(x, magic);  // the low bits are n
  const float2 n = __fadd2_rn(t, unmagic);
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 p = make_float2(0.00957010165f, 0.00957010165f);
  p = __ffma2_rn(p, f, make_float2(0.0559178605f, 0.0559178605f));
  p = __ffma2_rn(p, f, make_float2(0.240247448f, 0.240247448f));
  p = __ffma2_rn(p, f, make_float2(0.693121815f, 0.693121815f));
  p = __ffma2_rn(p, f, make_float2(0.999999261f, 0.999999261f));
  p.x = __uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23));
  p.y = __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23));
  return p;
}

// mbar_wait of a warp that stays together: all lanes get the answer of all, so that a
// wait that ran out for some of them takes every lane out of the same loop.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

// ---- thread-block clusters ----
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared variable in the CTA of rank `rank`.
__device__ __forceinline__ uint32_t map_to(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 load_remote4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 load_remote2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// The softmax threads hold a row of scores: with two tiles they take registers
// that the other warps do not need. With epilogue warps 512 threads have 128
// each at launch (256 x 200 + 256 x 56), without 384 have 168 (256 x 208 + 128 x 88).
template <int QT, bool EPILOGUE>
__device__ __forceinline__ void take_registers() {
  if constexpr (QT == 2 && EPILOGUE) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
  else if constexpr (QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
}
template <int QT, bool EPILOGUE>
__device__ __forceinline__ void give_registers() {
  if constexpr (QT == 2 && EPILOGUE) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  else if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
}

// What the body needs of a CTA's work: its items one after another (next() in
// every role); an item's n key tiles, tile i starting at key position key0(i),
// tile 0 of FEW keys only if `few`; loads; and each row's visible keys
// {kp : kp <= hi and (kp >= lo or kp < sinks)}.
template <class Work, class Smem>
__device__ __forceinline__ void tile_attention(Work w, Smem& sm, float scale_log2) {
  constexpr int QT = Smem::QT, SLOTS = Smem::SLOTS;
  constexpr bool EPILOGUE = Work::EPILOGUE;  // warps of their own normalise and store O
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&sm.kv_full[s], 1);
      mbar_init(&sm.kv_empty[s], 1);
    }
    for (int t = 0; t < QT; ++t) {
      mbar_init(&sm.q_full[t], 1);
      mbar_init(&sm.q_empty[t], 1);
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_full[t], 4);
      mbar_init(&sm.o_full[t], 1);
      mbar_init(&sm.l_full[t], 4);
      mbar_init(&sm.o_empty[t], 4);
    }
    mbar_init(&sm.mma_done, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 4 * QT + 1) {
    tmem_alloc(&sm.tmem, QT * 256);
    tmem_relinquish();
  }
  w.clear_q(sm);
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // not before: a dependent's CTA must not take TMEM that this one has yet to allocate
  const uint32_t tmem = sm.tmem;  // S_t at columns 128 t, O_t at 128 (QT + t)

  if (warp == 4 * QT) {
    // ---------------- TMA producer ----------------
    give_registers<QT, EPILOGUE>();
    if (lane == 0) {
      int slot = 0, items = 0, q_loads[QT] = {};
      uint32_t phase = 0;
      bool ok = true;
      for (; ok && w.next(); ++items) {
        for (int i = 0; ok && i < w.n; ++i) {
#pragma unroll 1
          for (int v = 0; v < 2; ++v) {
            // q comes behind the first K, whose slot is free before the last item's q is
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              if (i > 0 || v == 0) break;
              ok = ok && mbar_wait(&sm.q_empty[t], (items & 1) ^ 1, FB_KERR_TIMEOUT_EMPTY);
              if (!ok) break;
              w.load_q(sm, &sm.q_full[t], t);
              ++q_loads[t];
            }
            if (!ok) break;
            if (!mbar_wait(&sm.kv_empty[slot], phase ^ 1, FB_KERR_TIMEOUT_EMPTY)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&sm.kv_full[slot], TILE);
            w.load_kv(sm.kv[slot], &sm.kv_full[slot], i, v);
            if (++slot == SLOTS) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      }
      // Drain: every copy has landed and been consumed before the CTA leaves ..
      for (int s = 0; ok && s < SLOTS; ++s)
        ok = mbar_wait(&sm.kv_empty[s], s < slot ? phase : phase ^ 1, FB_KERR_TIMEOUT_EMPTY);
      // .. or, if a wait ran out, has landed at least: slots below `slot` were filled
      // in this turn of the ring, the others in the last one (parity 1 of a barrier
      // that nothing was ever sent to is behind it).
      if (!ok) {
        for (int s = 0; s < SLOTS; ++s) mbar_wait(&sm.kv_full[s], s < slot ? phase : phase ^ 1, FB_KERR_TIMEOUT_FULL);
#pragma unroll
        for (int t = 0; t < QT; ++t) mbar_wait(&sm.q_full[t], (q_loads[t] & 1) ^ 1, FB_KERR_TIMEOUT_FULL);
      }
    }
  } else if (warp == 4 * QT + 1) {
    // ---------------- MMA issuer ----------------
    give_registers<QT, EPILOGUE>();
    // The warp stays together: what the instructions take (descriptors, addresses)
    // is then computed once for the warp, and one elected lane issues them.
    constexpr uint32_t id_qk = idesc_bf16<128, 128>(), id_qk_few = idesc_bf16<128, FEW>();
    constexpr uint32_t id_pv = idesc_bf16<128, 128>() | (1u << 16);  // B (V) MN-major
    const uint64_t q_desc = sdesc_sw128(smem_u32(sm.q[0])), k_desc = sdesc_sw128(smem_u32(sm.kv[0]));
    const uint64_t v_desc = sdesc_mn_sw128(smem_u32(sm.kv[0]), HALF, 1024);
    const bool issuer = elect_one();
    int kslot = 0, vslot = 1 % SLOTS;
    uint32_t kphase = 0, vphase = 0;
    auto next = [](int& s, uint32_t& ph) {
      s += 2;
      if (s >= SLOTS) {
        s -= SLOTS;
        ph ^= 1;
      }
    };
    auto qk = [&](int t, uint32_t id) {
      const uint64_t qd = q_desc + t * (TILE / 16), kd = k_desc + kslot * (TILE / 16);
      if (issuer) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // K = 128 head dims, 16 per MMA
          const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) / 16;
          mma_bf16(tmem + t * 128, qd + off, kd + off, id, k > 0 ? 1u : 0u);
        }
        mma_commit(&sm.s_full[t]);
      }
    };
    auto commit = [&](uint64_t* bar) {
      if (issuer) mma_commit(bar);
    };
    uint32_t tiles = 0, items = 0;  // key tiles and items so far
    bool ok = true, more = w.next() && w.n > 0;
    int n = w.n;
    bool few = w.few;
    if (more) {
      ok = mbar_wait(&sm.kv_full[kslot], kphase, FB_KERR_TIMEOUT_FULL);
      for (int t = 0; t < QT; ++t) ok = ok && mbar_wait(&sm.q_full[t], 0, FB_KERR_TIMEOUT_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < QT; ++t) {
          qk(t, few ? id_qk_few : id_qk);
          if (n == 1) commit(&sm.q_empty[t]);
        }
        commit(&sm.kv_empty[kslot]);
        next(kslot, kphase);
      }
    }
    for (; ok && more; ++items) {
      for (int i = 0; ok && i < n; ++i, ++tiles) {
        // Behind P_t V_i comes the next key tile's product for the same query
        // tile: of the next item, behind the last of this one, so that neither
        // query tile waits for the other one's end.
        const bool last = i == n - 1;
        if (last) more = w.next();
        const bool next_qk = !last || more, next_ends = last ? w.n == 1 : i + 2 == n;
        const uint32_t next_id = last && w.few ? id_qk_few : id_qk;
        ok = mbar_wait(&sm.kv_full[vslot], vphase, FB_KERR_TIMEOUT_FULL);
        const uint64_t vd = v_desc + vslot * (TILE / 16);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          ok = ok && mbar_wait(&sm.p_full[t], tiles & 1, FB_KERR_TIMEOUT_TMEM);
          if (EPILOGUE && i == 0) ok = ok && mbar_wait(&sm.o_empty[t], (items & 1) ^ 1, FB_KERR_TIMEOUT_TMEM);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (issuer) {
            const int steps = i == 0 && few ? FEW / 16 : 8;
#pragma unroll
            for (int k = 0; k < 8; ++k)  // K = 128 keys, 16 per MMA
              if (k < steps)
                mma_bf16_ts(tmem + (QT + t) * 128, tmem + t * 128 + k * 8, vd + k * (2048 / 16), id_pv,
                            (i > 0 || k > 0) ? 1u : 0u);
          }
          if (t == QT - 1) commit(&sm.kv_empty[vslot]);
          if (last) commit(&sm.o_full[t]);
          if (next_qk) {
            if (t == 0) ok = mbar_wait(&sm.kv_full[kslot], kphase, FB_KERR_TIMEOUT_FULL);
            if (last) ok = ok && mbar_wait(&sm.q_full[t], (items & 1) ^ 1, FB_KERR_TIMEOUT_FULL);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            qk(t, next_id);
            if (next_ends) commit(&sm.q_empty[t]);
          }
        }
        if (ok && next_qk) {
          commit(&sm.kv_empty[kslot]);
          next(kslot, kphase);
        }
        next(vslot, vphase);
      }
      n = w.n;
      few = w.few;
    }
    if (!ok) {  // no product is under way when the CTA frees its tensor memory
      commit(&sm.mma_done);
      warp_wait(&sm.mma_done, 0, FB_KERR_TIMEOUT_TMEM);
    }
  } else if (warp < 4 * QT) {
    // ---------------- softmax + epilogue ----------------
    take_registers<QT, EPILOGUE>();
    const int t = warp >> 2;                         // query tile
    const int r = (warp & 3) * 32 + lane;            // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + lane_base, t_o = tmem + (QT + t) * 128 + lane_base;
    uint32_t tiles = 0, items = 0;
    bool ok = true;
    w.begin(t);
#pragma unroll 1
    for (; ok && w.next(); ++items) {
      int hi, lo;
      w.row_range(t, r, hi, lo);
      const int sinks = w.sinks, n = w.n;
      float m_run = -INFINITY, l_run = 0.f;
      // The keys k0 .. k0 + 31 that the row sees, as bits.
      auto seen = [&](int k0) {
        return bits_below(hi + 1 - k0) & (~bits_below(lo - k0) | bits_below(sinks - k0));
      };
#pragma unroll 1
      for (int i = 0; i < n; ++i, ++tiles) {
        const int k0 = w.key0(i);
        // A wait that ran out is each lane's own until the next tile's vote, which is
        // off the path from S to P: what the lane computes meanwhile is thrown away.
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ok = mbar_wait(&sm.s_full[t], tiles & 1, FB_KERR_TIMEOUT_TMEM);
        tc_fence_after();
        if (i == 0 && w.few) {
          // A few sinks far before the window: a tile of FEW keys.
          uint32_t sr[FEW], pk[FEW / 2];
          tmem_ld32(t_s, sr);
          tmem_ld_wait();
          const uint32_t bits = seen(k0);
#pragma unroll
          for (int e = 0; e < FEW; ++e) {
            if (!((bits >> e) & 1u)) sr[e] = 0xff800000u;
            m_run = fmaxf(m_run, __uint_as_float(sr[e]) * scale_log2);
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
          for (int e = 0; e < FEW; e += 2) {
            const float p0 = exp2f(fmaf(__uint_as_float(sr[e]), scale_log2, -m_use));
            const float p1 = exp2f(fmaf(__uint_as_float(sr[e + 1]), scale_log2, -m_use));
            l_run += p0 + p1;
            const bf162 b = __floats2bfloat162_rn(p0, p1);
            pk[e / 2] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tmem_st16(t_s, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[t]);
          continue;
        }
        uint32_t sr[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(t_s + c, sr + c);
        tmem_ld_wait();
        // Edge tiles: scores of keys that the row does not see become -inf.
        const bool edge = __any_sync(0xffffffffu, k0 + BK - 1 > hi || (k0 < lo && k0 + BK > sinks));
        if (edge) {
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            const uint32_t bits = seen(k0 + c);
            if (!__all_sync(0xffffffffu, bits == ~0u)) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((bits >> e) & 1u)) sr[c + e] = 0xff800000u;
            }
          }
        }
        if (t == 0 && w.zero_row(i, r)) {
          // A key that no row sees (behind the prompt's end, or every row's) holds
          // another prompt's values or nothing at all, and 0 * NaN = NaN: its V row
          // is zeroed once the copy has landed (tile 0's P V runs first, so once is
          // enough).
          const uint32_t at = 2 * tiles + 1, slot = at % SLOTS;
          ok = mbar_wait(&sm.kv_full[slot], (at / SLOTS) & 1, FB_KERR_TIMEOUT_FULL) && ok;
          uint8_t* vrow = sm.kv[slot] + r * 128;
#pragma unroll
          for (int e = 0; e < 16; ++e)  // (each lane from its own 16 bytes on: a warp's lanes in different banks)
            *reinterpret_cast<uint4*>(vrow + (e >> 3) * HALF + ((e ^ r) & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c += 2)
          mx4[(c >> 1) & 3] = max3_nan(mx4[(c >> 1) & 3], __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        const float mx = max_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3]) * scale_log2;
        const float m_new = mx <= m_run + RESCALE_LOG2 ? m_run : max_nan(m_run, mx);  // (from -inf it always moves)
        // A NaN score makes the maximum NaN, and an infinite one what is subtracted
        // here (inf - inf): all p of the row and its sum are then NaN.
        const float m_use = m_new == -INFINITY ? 0.f : fmaf(m_new, 0.f, m_new);
        const float alpha = exp2f(m_run - m_use);  // 1 unless the max moved; 0 while nothing was seen
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(t_o + c, o);
          }
        }
        // p = 2^(s scale - m)
        float2 rs[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 scale2 = make_float2(scale_log2, scale_log2), m2 = make_float2(-m_use, -m_use);
        auto half = [&](int h, auto poly) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int c = 64 * h + 2 * e;
            float2 y = __ffma2_rn(make_float2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, m2);
            if (poly && QT == 2 && e % POLY_OF == POLY_OF - 1) {
              y = exp2_poly(y);
            } else {
              y.x = exp2f(y.x);
              y.y = exp2f(y.y);
            }
            rs[e & 1] = __fadd2_rn(rs[e & 1], y);
            const bf162 b = __floats2bfloat162_rn(y.x, y.y);
            pk[e] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tmem_st32(t_s + 32 * h, pk);
        };
        if (edge) {  // exact zeros for what is masked
          half(0, std::false_type());
          half(1, std::false_type());
        } else {
          half(0, std::true_type());
          half(1, std::true_type());
        }
        tmem_st_wait();
        tc_fence_before();
        l_run = l_run * alpha + ((rs[0].x + rs[0].y) + (rs[1].x + rs[1].y));
        m_run = m_new;
        if (EPILOGUE && i == n - 1) {
          // Not before the epilogue has read the last item's: with one key tile per
          // item nothing else would keep this warp from running two items ahead.
          ok = mbar_wait(&sm.o_empty[t], (items & 1) ^ 1, FB_KERR_TIMEOUT_TMEM) && ok;
          sm.l[t][r] = l_run;
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.p_full[t]);
          if (EPILOGUE && i == n - 1) mbar_arrive(&sm.l_full[t]);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if constexpr (!EPILOGUE) {
        for (int i = 0; ok && n > 0 && i < QT; ++i)  // of every tile: a store may reuse the ring
          if (i == t || Work::JOINS) ok = warp_wait(&sm.o_full[i], items & 1, FB_KERR_TIMEOUT_TMEM);
        if (ok) {
          tc_fence_after();
          w.store(sm, t, r, t_o, m_run, l_run, [] {});
        }
      }
    }
  } else if (EPILOGUE && warp >= 4 * QT + 4) {
    // ---------------- epilogue ----------------
    // O of an item is read while the softmax warps are at the next one.
    give_registers<QT, EPILOGUE>();
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t items = 0;
    bool ok = true;
#pragma unroll 1
    for (; ok && w.next(); ++items)
#pragma unroll 1
      for (int t = 0; ok && t < QT; ++t) {
        ok = mbar_wait(&sm.l_full[t], items & 1, FB_KERR_TIMEOUT_TMEM) &&
             mbar_wait(&sm.o_full[t], items & 1, FB_KERR_TIMEOUT_TMEM);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        w.store(sm, t, r, tmem + (QT + t) * 128 + lane_base, 0.f, sm.l[t][r], [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.o_empty[t]);
        });
      }
  } else {
    give_registers<QT, EPILOGUE>();
  }
  __syncwarp();  // the lane that copies is back with its warp
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Before a cluster's join: a CTA that waits for another one, which may itself be
  // waiting for tensor memory, holds none.
  if (warp == 4 * QT + 1) tmem_dealloc(tmem, QT * 256);
  w.finish(sm);
}

template <class Smem>
__device__ __forceinline__ Smem& tile_smem() {
  extern __shared__ uint8_t smem_raw[];
  return *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
}

// ---- windowed causal prefill -----------------------------------------------------------
// An item is a query tile [qp0, qp0 + 128) of a prompt for QT heads of one KV
// head. Its key tiles: those of the sinks, then those of the window, at multiples
// of 128 of the prompt. The grid is persistent: a prompt tile has few key tiles,
// and the next item's copies and first product run during this one's end.
template <class Smem>
struct WindowWork {
  static constexpr int QT = Smem::QT;
  const CUtensorMap *tmQ, *tmK, *tmV;
  bf16* out;
  const int *cu_seqlens, *tile_seq, *tile_start;
  int ld_o, rows, n_seqs, n_tiles, heads, group, window, all_sinks;
  // Items go tile by tile, head by head. What the tables say of an item is read
  // two items ahead (the tile's prompt), then one (where that begins and ends), so
  // that nothing waits for them.
  int item;  // one ahead
  int seq2, start2, s0_1, s1_1, start1;
  int head0, s0, s1, qp0, n, n_sink, first, sinks;
  bool few;

  __device__ __forceinline__ void read_tile(int i) {
    const int tile = min(i / heads, n_tiles - 1);
    seq2 = tile_seq[tile];
    start2 = tile_start[tile];
  }
  __device__ __forceinline__ void read_prompt() {
    const int seq = min(max(seq2, 0), n_seqs - 1);  // whatever the tables say, nothing outside the tensors is touched
    start1 = start2;
    s0_1 = cu_seqlens[seq];
    s1_1 = cu_seqlens[seq + 1];
  }
  __device__ __forceinline__ void start() {
    item = blockIdx.x;
    read_tile(item);
    read_prompt();
    read_tile(item + gridDim.x);
  }
  __device__ __forceinline__ bool next() {
    for (bool found = false; !found;) {
      if (item >= n_tiles * heads) return false;
      s0 = max(s0_1, 0);
      s1 = min(s1_1, rows);
      qp0 = start1;
      head0 = item % heads * QT;
      item += gridDim.x;
      read_prompt();
      read_tile(item + gridDim.x);
      found = qp0 >= 0 && qp0 < s1 - s0;  // (else: a tile table that does not match cu_seqlens)
    }
    const int end = min(qp0 + BQ, s1 - s0);  // queries and keys of this tile end here
    const int last = (end - 1) / BK, in_window = max(qp0 - window + 1, 0) / BK;
    sinks = min(all_sinks, end);
    n_sink = min((sinks + BK - 1) / BK, last + 1);
    first = max(in_window, n_sink);
    n = n_sink + last + 1 - first;
    few = n_sink == 1 && sinks <= FEW && in_window > 0;
    return true;
  }
  __device__ __forceinline__ int key0(int i) const { return (i < n_sink ? i : i - n_sink + first) * BK; }
  __device__ __forceinline__ bool zero_row(int i, int r) const { return key0(i) + r >= s1 - s0; }
  __device__ __forceinline__ void clear_q(Smem&) const {}
  __device__ __forceinline__ void begin(int) const {}
  __device__ __forceinline__ void load_q(Smem& sm, uint64_t* bar, int t) const {
    mbar_arrive_expect_tx(bar, TILE);
    for (int h = 0; h < 2; ++h) tma_load_2d(sm.q[t] + h * HALF, tmQ, bar, (head0 + t) * D + h * 64, s0 + qp0);
  }
  __device__ __forceinline__ void load_kv(uint8_t* dst, uint64_t* bar, int i, int v) const {
    const int row = s0 + key0(i);
    for (int h = 0; h < 2; ++h) tma_load_2d(dst + h * HALF, v ? tmV : tmK, bar, head0 / group * D + h * 64, row);
  }
  __device__ __forceinline__ void row_range(int, int r, int& hi, int& lo) const {
    const int qpos = qp0 + r;
    hi = s0 + qpos < s1 ? qpos : -1;
    lo = qpos - window + 1;
  }
  __device__ __forceinline__ void finish(Smem&) const {}
  static constexpr bool EPILOGUE = QT == 2;
  [[maybe_unused]] static constexpr bool JOINS = false;
  // Rows go through shared memory (32 dims of them at a time, or whole), 16-byte
  // chunks swizzled by the row, so that a store instruction writes 64 bytes of
  // eight rows or two whole rows: straight from a row per thread it would touch 32
  // lines, and the stores of a tile took as long as two key tiles. `read` is called
  // when O has been read: with whole rows, before any of them is stored.
  template <class Read>
  __device__ __forceinline__ void store(Smem& sm, int t, int r, uint32_t t_o, float, float l, Read read) const {
    constexpr int CHUNKS = Smem::STAGE / 16, ROWS = 32 / CHUNKS;  // chunks of a staged row; rows of a store
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (NaN stays NaN)
    const int lane = r & 31, row0 = s0 + qp0 + (r & ~31), my_row = lane / CHUNKS, my_chunk = lane % CHUNKS;
    uint8_t* stage = sm.stage[r >> 5];
    auto at = [&](int row, int chunk) {
      const int swizzle = CHUNKS == 16 ? row & 15 : (row >> 1) & 3;
      return reinterpret_cast<uint4*>(stage + row * Smem::STAGE + ((chunk ^ swizzle) << 4));
    };
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      tmem_ld32(t_o + c, o);
      tmem_ld_wait();
      if (c == D - 32) read();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[8 * e + x]) * inv;
        *at(lane, CHUNKS == 16 ? c / 8 + e : e) = pack8(f);
      }
      if (CHUNKS == 16 && c < D - 32) continue;
      __syncwarp();
      bf16* to = out + static_cast<size_t>(row0 + my_row) * ld_o + (head0 + t) * D + (CHUNKS == 16 ? 0 : c) + my_chunk * 8;
#pragma unroll 4
      for (int row = my_row; row < 32; row += ROWS, to += static_cast<size_t>(ROWS) * ld_o)
        if (row0 + row < s1) *reinterpret_cast<uint4*>(to) = *at(row, my_chunk);
      __syncwarp();
    }
  }
};

template <class Smem>
__device__ __forceinline__ void window_prefill(const CUtensorMap* tmQ, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                               bf16* out, int ld_o, int rows, int n_seqs, const int* cu_seqlens,
                                               const int* tile_seq, const int* tile_start, int n_tiles, int Hq, int Hkv, int window,
                                               int sinks, float scale_log2) {
  pdl_wait();
  WindowWork<Smem> w;
  w.tmQ = tmQ;
  w.tmK = tmK;
  w.tmV = tmV;
  w.out = out;
  w.ld_o = ld_o;
  w.rows = rows;
  w.n_seqs = n_seqs;
  w.cu_seqlens = cu_seqlens;
  w.tile_seq = tile_seq;
  w.tile_start = tile_start;
  w.n_tiles = n_tiles;
  w.heads = Hq / Smem::QT;
  w.group = Hq / Hkv;
  w.window = window;
  w.all_sinks = sinks;
  w.start();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(tmQ);
    tma_prefetch_desc(tmK);
    tma_prefetch_desc(tmV);
  }
  tile_attention(w, tile_smem<Smem>(), scale_log2);
}

// ---- shared prefix of a decode batch ---------------------------------------------------
// items[blockIdx.x] = {first row, rows, first page, pages, part}: the rows
// (sequences) of one group against a range of the pages that its first row's block
// table begins with; the CTAs of a cluster have the same rows and part. Row r of query tile t is head r / nb of the group's
// KV head for sequence first + t * nb + r % nb, nb = 128 / G rounded down to a
// multiple of 8 (whole swizzle atoms), so one TMA box of nb rows fetches one head.
struct PrefixItem {
  int row0, rows, page0, pages, part, pad[3];
};

template <class Smem>
struct PrefixWork {
  static constexpr int QT = Smem::QT;
  const CUtensorMap *tmQ, *tmK, *tmV;
  const int *pages, *seq_lens;
  float *o_part, *ml_part;
  PrefixItem it;
  int kvh, G, nb, Hq, Hkv, parts, blocks;
  int n, sinks;
  static constexpr bool few = false;
  bool more = true;  // a CTA has one item (of no pages, maybe)
  __device__ __forceinline__ bool next() {
    const bool had = more;
    more = false;
    return had;
  }

  __device__ __forceinline__ int key0(int i) const { return it.page0 * PAGE + i * BK; }
  int longest;  // of the item's rows, in query tile 0's softmax warps (which look for it while the first K is on its way)
  __device__ __forceinline__ void begin(int t) {
    if (t != 0) return;
    int n_keys = 0;
    for (int b = threadIdx.x & 31; b < it.rows; b += 32) n_keys = max(n_keys, seq_lens[it.row0 + b]);
    longest = __reduce_max_sync(0xffffffffu, n_keys);
  }
  __device__ __forceinline__ bool zero_row(int i, int r) const {
    const int key = key0(i) + r;
    return key >= longest && key < (it.page0 + it.pages) * PAGE;  // (TMA has filled what is behind with zeros)
  }
  // Rows that no head and sequence uses hold zeros and see every key: what
  // they compute is finite and dropped, and keeps no warp on the masked path.
  __device__ __forceinline__ void clear_q(Smem& sm) const {
    const int rows = 128 - G * nb;
    for (int e = threadIdx.x; e < QT * 2 * rows * 8; e += blockDim.x) {
      const int half = e / (rows * 8);  // tile * 2 + dim half
      *reinterpret_cast<uint4*>(sm.q[half >> 1] + (half & 1) * HALF + G * nb * 128 + (e % (rows * 8)) * 16) =
          make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void load_q(Smem& sm, uint64_t* bar, int t) const {
    mbar_arrive_expect_tx(bar, 2 * G * nb * 128);
    for (int g = 0; g < G; ++g)
      for (int h = 0; h < 2; ++h)
        tma_load_2d(sm.q[t] + h * HALF + g * nb * 128, tmQ, bar, (kvh * G + g) * D + h * 64, it.row0 + t * nb);
  }
  __device__ __forceinline__ void load_kv(uint8_t* dst, uint64_t* bar, int i, int v) const {
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      // No page (a tile's second one behind the end): rows past the cache, which TMA fills with zeros.
      int page = blocks;
      if (2 * i + pg < it.pages) {
        page = pages[it.page0 + 2 * i + pg];
        if (page < 0 || page >= blocks) {
          set_status(FB_KERR_BAD_ARG);
          page = blocks;
        }
      }
      const int row = (page * Hkv + kvh) * PAGE;
      for (int h = 0; h < 2; ++h)
        tma_load_2d(dst + h * HALF + pg * PAGE * 128, v ? tmV : tmK, bar, h * 64, row);
    }
  }
  __device__ __forceinline__ int row_of(int t, int r) const { return t * nb + r % nb; }  // of the item
  __device__ __forceinline__ void row_range(int t, int r, int& hi, int& lo) const {
    const int b = row_of(t, r);
    const int end = (it.page0 + it.pages) * PAGE;
    hi = r < G * nb && b < it.rows ? min(seq_lens[it.row0 + b], end) - 1 : EVERY_KEY;
    lo = 0;
  }
  // Index of a tile row's result; -1 if no head and sequence uses it.
  __device__ __forceinline__ long long result_of(int t, int r) const {
    const int b = row_of(t, r);
    if (r >= G * nb || b >= it.rows) return -1;
    return ((it.row0 + b) * static_cast<long long>(Hq) + kvh * G + r / nb) * parts + it.part;
  }
  static constexpr bool EPILOGUE = false, JOINS = true;
  // O rows of the tiles in the ring's memory, 16-byte chunks swizzled by the row.
  __device__ __forceinline__ static uint32_t o_at(Smem& sm, int t, int r, int chunk) {
    return smem_u32(sm.kv[0]) + (t * BQ + r) * (D * 4) + ((chunk ^ (r & 31)) << 4);
  }
  template <class Read>
  __device__ __forceinline__ void store(Smem& sm, int t, int r, uint32_t t_o, float m, float l, Read) const {
    sm.ml(t)[r] = make_float2(m, l);
    if (n == 0) return;  // O is nothing
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      tmem_ld32(t_o + c, o);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(o_at(sm, t, r, (c + e) / 4)), "r"(o[e]),
                     "r"(o[e + 1]), "r"(o[e + 2]), "r"(o[e + 3])
                     : "memory");
    }
  }
  // The cluster's CTAs have the same rows: a warp joins one row at a time, of
  // the rows that fall to its CTA.
  __device__ __forceinline__ void finish(Smem& sm) const {
    cluster_sync();
    const int size = cluster_size(), warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    for (int i = cluster_rank() * warps + (threadIdx.x >> 5); i < QT * BQ; i += size * warps) {
      const int t = i / BQ, r = i % BQ;
      const long long at = result_of(t, r);
      if (at < 0) continue;
      float2 ml[MAX_CLUSTER];
      float4 o[MAX_CLUSTER];
      float m = -INFINITY;
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) {
        ml[c] = make_float2(-INFINITY, 0.f);
        if (c < size) {
          ml[c] = load_remote2(map_to(smem_u32(sm.ml(t) + r), c));
          o[c] = load_remote4(map_to(o_at(sm, t, r, lane), c));
        }
        m = fmaxf(m, ml[c].x);
      }
      const float ref = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) {
        const float e = exp2f(ml[c].x - ref);
        if (ml[c].y == 0.f) continue;  // (an empty part's O is no number)
        l = fmaf(ml[c].y, e, l);
        sum.x = fmaf(o[c].x, e, sum.x);
        sum.y = fmaf(o[c].y, e, sum.y);
        sum.z = fmaf(o[c].z, e, sum.z);
        sum.w = fmaf(o[c].w, e, sum.w);
      }
      reinterpret_cast<float4*>(o_part + at * D)[lane] = sum;
      if (lane == 0) *reinterpret_cast<float2*>(ml_part + 2 * at) = make_float2(m, l);
    }
    cluster_sync();  // the others may still be reading this CTA's shared memory
  }
};

template <class Smem>
__device__ __forceinline__ void prefix_attention(const CUtensorMap* tmQ, const CUtensorMap* tmK,
                                                 const CUtensorMap* tmV, const PrefixItem* items,
                                                 const int* block_tables, int max_blocks, const int* seq_lens,
                                                 float* o_part, float* ml_part, int G, int Hq, int Hkv, int parts,
                                                 int blocks, float scale_log2) {
  pdl_wait();
  PrefixWork<Smem> w;
  w.it = items[blockIdx.x];
  w.tmQ = tmQ;
  w.tmK = tmK;
  w.tmV = tmV;
  w.pages = block_tables + static_cast<size_t>(w.it.row0) * max_blocks;
  w.seq_lens = seq_lens;
  w.o_part = o_part;
  w.ml_part = ml_part;
  w.kvh = blockIdx.y;
  w.G = G;
  w.nb = (128 / G) & ~7;
  w.Hq = Hq;
  w.Hkv = Hkv;
  w.parts = parts;
  w.blocks = blocks;
  w.n = (w.it.pages + 1) / 2;
  w.sinks = 0;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(tmQ);
    tma_prefetch_desc(tmK);
    tma_prefetch_desc(tmV);
  }
  tile_attention(w, tile_smem<Smem>(), scale_log2);
}

}  // namespace

// Boxes of 64 dims, 128B swizzle: of q, then of k and v.
struct TileMaps {
  CUtensorMap q, k, v;
};

// q [T, Hq * 128], k, v [T, Hkv * 128]: maps over the packed rows, boxes of 128
// rows. n_tiles query tiles of tile_seq / tile_start. out [T, ld_o] bf16, head h at columns h * 128; rows outside every prompt are not written.
#define FB_WINDOW_PREFILL(QT, CTAS)                                                                               \
  extern "C" __global__ void __launch_bounds__(QT == 2 ? 512 : 192, CTAS) fb_window_prefill_q##QT(                \
      const __grid_constant__ TileMaps maps, bf16* out, int ld_o, int rows, int n_seqs, const int* cu_seqlens,    \
      const int* tile_seq, const int* tile_start, int n_tiles, int Hq, int Hkv, int window, int sinks,            \
      float scale_log2) {                                                                                         \
    window_prefill<WindowSmem##QT>(&maps.q, &maps.k, &maps.v, out, ld_o, rows, n_seqs, cu_seqlens, tile_seq,      \
                                   tile_start, n_tiles, Hq, Hkv, window, sinks, scale_log2);                      \
  }
FB_WINDOW_PREFILL(1, 2)
FB_WINDOW_PREFILL(2, 1)

// q [B, Hq * 128] with boxes of nb rows; caches viewed as [blocks * Hkv * 64,
// 128] with boxes of one page. Grid: (items, Hkv), clusters of the items that
// share their rows. Part p of the result of (row, head) is at index
// (row * Hq + head) * parts + p.
#define FB_PREFIX_ATTN(QT, CTAS)                                                                                  \
  extern "C" __global__ void __launch_bounds__(QT == 2 ? 384 : 192, CTAS) fb_prefix_attn_q##QT(                   \
      const __grid_constant__ TileMaps maps, const PrefixItem* items, const int* block_tables, int max_blocks,    \
      const int* seq_lens, float* o_part, float* ml_part, int G, int Hq, int Hkv, int parts, int blocks,          \
      float scale_log2) {                                                                                         \
    prefix_attention<PrefixSmem##QT>(&maps.q, &maps.k, &maps.v, items, block_tables, max_blocks, seq_lens,        \
                                     o_part, ml_part, G, Hq, Hkv, parts, blocks, scale_log2);                     \
  }
FB_PREFIX_ATTN(1, 2)
FB_PREFIX_ATTN(2, 1)
