// Paged GQA decode attention over part of each sequence, on the tcgen05 tensor
// cores (head_dim 128, bf16 K/V pages of 64 tokens, fp32 softmax state). The
// visible tokens of a sequence of n tokens are
//
//   window > 0:  [0, min(sinks, n)) and [max(n - window, 0), n)
//   window = 0:  [start, n), start = the tokens that fb_prefix_attn_* has
//                attended to for the whole group (row_info)
//
// Pages without a visible token are never touched; of a page that is visible
// in part, only the 16-token blocks with a visible token are read.
//
// A sequence's visible pages, in order, make chunks of two pages. Per chunk and
// KV head (G query heads):
//   S^T[tok, h] = K Q^T      tcgen05.mma M=128 (tokens) N=16 (heads, zero padded) K=128
//   softmax                  one token per thread, running max per head over the chunk
//   O^T[d, h]  = V^T P^T     tcgen05.mma M=128 (dims) N=16 K=128 (tokens), V read MN-major
//                            from the image the K-major TMA load produced
//   O                        in registers, one head dim per thread
//
// The kernel is bound by reading K and V once, so what matters is that every
// SM reads all the time. Lengths differ from row to row and are known on the
// device only: each CTA sums the chunks of all rows, and the (row, KV head,
// chunk) sequence is cut into one equal share per CTA. A (row, KV head) that a
// cut falls into is joined by the CTA that finishes its last piece, through
// fp32 partials in a workspace of two pieces per CTA and one ticket per cut
// (zero before and after every launch). So one launch does it all, the
// workspace does not grow with batch or length, and the order of the join is
// that of the tokens: results do not depend on which CTA comes last.
//
// Single 64 KB stage per CTA and three CTAs per SM (two for more than eight
// heads per KV head, by registers): K and V have their own barriers, so the
// next chunk's K loads during this chunk's softmax and P V.
//
// Roles: warp 0 TMA producer, warp 1 TMEM owner + MMA issuer, warps 2..5
// softmax and epilogue. No TMA multicast. All waits bounded (fb_common.cuh).
#include "attn_tile.cuh"

FB_DEFINE_STATUS

using namespace fbk;

namespace {

constexpr int D = 128;
constexpr int PAGE = 64;
constexpr int NH = 16;                       // padded head count (MMA N)
constexpr int THREADS = 192;
constexpr int BOX_BYTES = 64 * 128;          // 64 tokens x 64 dims x 2 B
constexpr int SUB_BYTES = 16 * 128;          // 16 tokens x 64 dims x 2 B
constexpr int KV_BYTES = 2 * 2 * BOX_BYTES;  // one chunk of K (or V): 2 pages x 2 dim halves
constexpr int HALF_STRIDE = 2 * BOX_BYTES;   // dim-half block: 128 tokens x 128 B
constexpr int QP_BYTES = 2 * NH * 128;       // [2 halves][16 rows][128 B]

struct Smem {
  uint8_t k[KV_BYTES];
  uint8_t v[KV_BYTES];
  uint8_t q[QP_BYTES];
  uint8_t p[QP_BYTES];
  uint64_t kfull, vfull, kempty, vempty;
  uint64_t s_full, s_empty, p_full, o_full, o_empty, q_ready;
  float red[4][NH];      // per-warp max, then per-warp sum, of every head
  float alpha[NH];       // this chunk's rescale factor per head
  float mrun[2][NH];     // running max per head, by chunk parity
  int scan[THREADS / 32];
  int total, first_row, first_off;
  uint32_t tmem;
  int last;
  int abort;
  int give_up;  // a softmax thread's wait ran out: read by all of them between the same two barriers
};
static_assert(sizeof(Smem) + 1024 <= 74 * 1024, "host requests 74 KB of dynamic shared memory (3 CTAs per SM)");

// M=128, N=16, bf16 in, f32 accumulate; a_major: 0 K-major, 1 MN-major.
__device__ __forceinline__ constexpr uint32_t idesc_span(uint32_t a_major) {
  return idesc_bf16<128, NH>() | (a_major << 15);
}

// Byte offset of element (row, k) in a [2 k-halves][16 rows][128 B] swizzled tile.
__device__ __forceinline__ uint32_t qp_offset(int row, int k) {
  const int kk = k & 63;
  return (k >> 6) * (NH * 128) + row * 128 + (((kk >> 3) ^ (row & 7)) << 4) + (kk & 7) * 2;
}

__device__ __forceinline__ void sync_softmax() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

struct Params {
  const bf16* q;
  const int* block_tables;
  const int* seq_lens;
  const int2* row_info;  // {tokens attended to by the prefix kernel, its parts} per row, or null
  bf16* out;
  const float *prefix_o, *prefix_ml;  // partial (row * Hq + head) * prefix_parts + part
  float *ws_o, *ws_ml;                // [2 * gridDim][Hq / Hkv rounded up to the variant][128] and [..][2]
  int* tickets;                       // [gridDim], zero between launches
  long long ld_q, ld_o;
  int max_blocks, blocks, B, Hkv, G, prefix_parts, window, sinks;
  float scale_log2;
};

// The visible tokens of a row: t < n and (t >= lo or t < sinks), on the
// virtual pages 0 .. pages - 1: first those of the sinks, then from page `wp`.
struct Span {
  int n, lo, sinks, sp, wp, pages, chunks;
  __device__ __forceinline__ int page(int v) const { return v < sp ? v : v - sp + wp; }
};

__device__ __forceinline__ Span row_span(const Params& a, int b) {
  Span s;
  s.n = min(max(a.seq_lens[b], 0), a.max_blocks * PAGE);
  const int start = a.row_info ? min(a.row_info[b].x, s.n) : 0;
  s.lo = a.window > 0 ? max(s.n - a.window, 0) : start;
  s.sinks = a.window > 0 ? min(a.sinks, s.lo) : 0;
  s.sp = (s.sinks + PAGE - 1) / PAGE;
  s.wp = max(s.sp, s.lo / PAGE);
  s.pages = s.lo < s.n ? s.sp + (s.n - 1) / PAGE + 1 - s.wp : 0;
  s.chunks = max(1, (s.pages + 1) / 2);  // a row that sees nothing has an empty chunk: its output is written too
  return s;
}

// The pieces of a CTA's share [begin, end) of the flat (row, KV head, chunk)
// sequence: chunks [c0, c1) of (b, kvh), the flat position of chunk c0 being `at`.
struct Walk {
  int b, kvh, c0, c1, at, end;
  Span s;
  bool fresh;
  __device__ __forceinline__ Walk(const Params& a, const Smem& sm, int begin, int e)
      : b(sm.first_row), at(begin), end(e), fresh(true) {
    if (begin >= end) return;
    s = row_span(a, b);
    kvh = sm.first_off / s.chunks;
    c0 = sm.first_off % s.chunks;
    c1 = min(s.chunks, c0 + end - at);
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  __device__ __forceinline__ void next(const Params& a) {
    at += c1 - c0;
    if (at >= end) return;
    c0 = 0;
    if (++kvh == a.Hkv) {
      kvh = 0;
      s = row_span(a, ++b);
    }
    c1 = min(s.chunks, end - at);
  }
};

template <int GP>
__device__ __forceinline__ void span_body(const CUtensorMap* tmK, const CUtensorMap* tmV, const CUtensorMap* tmK16,
                                          const CUtensorMap* tmV16, const Params& a) {
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&sm.kfull, 1);
    mbar_init(&sm.vfull, 1);
    mbar_init(&sm.kempty, 1);
    mbar_init(&sm.vempty, 1);
    mbar_init(&sm.s_full, 1);
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.s_empty, 4);
    mbar_init(&sm.p_full, 4);
    mbar_init(&sm.o_empty, 4);
    mbar_init(&sm.q_ready, 4);
    sm.abort = sm.give_up = 0;
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(tmK);
    tma_prefetch_desc(tmV);
    tma_prefetch_desc(tmK16);
    tma_prefetch_desc(tmV16);
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 32);
    tmem_relinquish();
  }
  // Rows of heads >= G stay zero for the whole kernel.
  for (int i = threadIdx.x; i < QP_BYTES / 16; i += THREADS) {
    reinterpret_cast<uint4*>(sm.p)[i] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(sm.q)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // not before: a dependent's CTA must not take TMEM that this one has yet to allocate
  pdl_wait();  // set-up above overlapped the previous kernel; what it wrote (q, caches, lengths) is read below

  // ---- this CTA's share: exclusive sums of the rows' chunks, R rows per thread ----
  const int R = (a.B + THREADS - 1) / THREADS;
  const int row0 = min(static_cast<int>(threadIdx.x) * R, a.B), row1 = min(row0 + R, a.B);
  int mine = 0;
  for (int b = row0; b < row1; ++b) {
    mine += row_span(a, b).chunks * a.Hkv;
    if (blockIdx.x == 0 && (a.seq_lens[b] < 0 || a.seq_lens[b] > a.max_blocks * PAGE)) set_status(FB_KERR_BAD_ARG);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sm.scan[warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += sm.scan[w];
    total += sm.scan[w];
  }
  const int share = max(1, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  const int begin = min(static_cast<int>(blockIdx.x) * share, total), end = min(begin + share, total);
  if (begin < end && begin >= before && begin < before + mine) {
    int off = begin - before, b = row0;
    for (;; ++b) {
      const int len = row_span(a, b).chunks * a.Hkv;
      if (off < len) break;
      off -= len;
    }
    sm.first_row = b;
    sm.first_off = off;
  }
  __syncthreads();
  const uint32_t tmem = sm.tmem;
  const uint32_t t_s = tmem, t_o = tmem + NH;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      uint32_t phase = 0;
      for (Walk w(a, sm, begin, end); w.more() && !*(volatile int*)&sm.abort; w.next(a)) {
        const int* bt = a.block_tables + static_cast<size_t>(w.b) * a.max_blocks;
        // Rows [16 * lo16, 16 * hi16) of a chunk's two pages and the pages' first cache row.
        auto chunk_pages = [&](int c, int (&lo16)[2], int (&hi16)[2], int (&rows)[2]) {
#pragma unroll
          for (int pg = 0; pg < 2; ++pg) {
            lo16[pg] = hi16[pg] = rows[pg] = 0;
            if (2 * c + pg >= w.s.pages) continue;
            const int p = w.s.page(2 * c + pg), t0 = p * PAGE;
            const int to = t0 + PAGE > w.s.lo ? w.s.n : w.s.sinks;
            const int from = t0 < w.s.sinks ? 0 : max(w.s.lo - t0, 0);
            lo16[pg] = from / 16;
            hi16[pg] = (min(to - t0, PAGE) + 15) / 16;
            int id = bt[p];
            if (id < 0 || id >= a.blocks) {
              set_status(FB_KERR_BAD_ARG);
              id = a.blocks;  // past the cache: TMA fills zeros
            }
            rows[pg] = (id * a.Hkv + w.kvh) * PAGE;
          }
        };
        int nl[2], nh[2], nr[2];
        chunk_pages(w.c0, nl, nh, nr);
        for (int c = w.c0; c < w.c1; ++c) {
          const int l[2] = {nl[0], nl[1]}, h[2] = {nh[0], nh[1]}, rows[2] = {nr[0], nr[1]};
          if (c + 1 < w.c1) chunk_pages(c + 1, nl, nh, nr);  // read ahead, off the critical path
          const uint32_t bytes = static_cast<uint32_t>(h[0] - l[0] + h[1] - l[1]) * (2 * SUB_BYTES);  // K or V
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = kv ? &sm.vfull : &sm.kfull;
            if (!mbar_wait(kv ? &sm.vempty : &sm.kempty, phase ^ 1, FB_KERR_TIMEOUT_EMPTY)) {
              sm.abort = 1;
              continue;  // no copies for this chunk; the loop ends below
            }
            mbar_arrive_expect_tx(full, bytes);
            uint8_t* buf = kv ? sm.v : sm.k;
#pragma unroll
            for (int pg = 0; pg < 2; ++pg) {
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                uint8_t* dst = buf + hf * HALF_STRIDE + pg * BOX_BYTES;
                if (h[pg] - l[pg] == 4) {
                  tma_load_2d(dst, kv ? tmV : tmK, full, hf * 64, rows[pg]);
                } else {
                  // a 16-row box at a 2 KB offset lands in the same swizzled image as a full box
                  for (int j = l[pg]; j < h[pg]; ++j)
                    tma_load_2d(dst + j * SUB_BYTES, kv ? tmV16 : tmK16, full, hf * 64, rows[pg] + 16 * j);
                }
              }
            }
          }
          if (*(volatile int*)&sm.abort) break;
          phase ^= 1;
        }
      }
      // Drain: every issued copy has been consumed (or the kernel gave up).
      mbar_wait(&sm.kempty, phase ^ 1, FB_KERR_TIMEOUT_EMPTY);
      mbar_wait(&sm.vempty, phase ^ 1, FB_KERR_TIMEOUT_EMPTY);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t kb = smem_u32(sm.k), vb = smem_u32(sm.v), qb = smem_u32(sm.q), pb = smem_u32(sm.p);
      uint32_t cc = 0, items = 0;  // chunks and pieces so far
      bool ok = true;
      for (Walk w(a, sm, begin, end); ok && w.more() && !*(volatile int*)&sm.abort; w.next(a)) {
        if (!mbar_wait(&sm.q_ready, items & 1, FB_KERR_TIMEOUT_FULL)) {
          ok = false;
          break;
        }
        ++items;
        for (int c = w.c0; c < w.c1; ++c, ++cc) {
          if (!mbar_wait(&sm.kfull, cc & 1, FB_KERR_TIMEOUT_FULL) ||
              !mbar_wait(&sm.s_empty, (cc & 1) ^ 1, FB_KERR_TIMEOUT_TMEM)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 8; ++j) {  // K = 128 head dims, 16 per MMA
            const uint32_t h = j >> 2, off = (j & 3) * 32;
            mma_bf16(t_s, sdesc_sw128(kb + h * HALF_STRIDE + off), sdesc_sw128(qb + h * (NH * 128) + off),
                     idesc_span(0), j > 0 ? 1u : 0u);
          }
          mma_commit(&sm.s_full);
          mma_commit(&sm.kempty);
          if (!mbar_wait(&sm.p_full, cc & 1, FB_KERR_TIMEOUT_TMEM) ||
              !mbar_wait(&sm.o_empty, (cc & 1) ^ 1, FB_KERR_TIMEOUT_TMEM) ||
              !mbar_wait(&sm.vfull, cc & 1, FB_KERR_TIMEOUT_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 8; ++j) {  // K = 128 tokens, 16 per MMA
            const uint32_t h = j >> 2, off = (j & 3) * 32;
            mma_bf16(t_o, sdesc_mn_sw128(vb + j * 2048, HALF_STRIDE, 1024), sdesc_sw128(pb + h * (NH * 128) + off),
                     idesc_span(1), j > 0 ? 1u : 0u);
          }
          mma_commit(&sm.o_full);
          mma_commit(&sm.vempty);
        }
      }
      if (!ok) sm.abort = 1;
    }
  } else {
    // ---------------- softmax / epilogue (warps 2..5) ----------------
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // TMEM lane: token (for S) / head dim (for O)
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const int G = a.G, Hq = a.Hkv * G;
    uint32_t cc = 0;
    volatile int* give_up = &sm.give_up;
    for (Walk w(a, sm, begin, end); w.more(); w.next(a)) {
      for (int e = r; e < G * 16; e += 128) {  // the heads' q rows, 16 B at a time
        const int row = e >> 4, col = (e & 15) * 8;
        *reinterpret_cast<uint4*>(sm.q + qp_offset(row, col)) =
            *reinterpret_cast<const uint4*>(a.q + w.b * a.ld_q + (w.kvh * G + row) * D + col);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_ready);

      float l_thr[GP], o[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        // chunk k reads mrun[k & 1]; thread 0 writes the next one's after the first barrier of chunk k
        if (r == 0) sm.mrun[cc & 1][g] = -INFINITY;
        l_thr[g] = 0.f;
        o[g] = 0.f;
      }
      for (int c = w.c0; c < w.c1; ++c, ++cc) {
        if (!mbar_wait(&sm.s_full, cc & 1, FB_KERR_TIMEOUT_TMEM)) *give_up = 1;
        tc_fence_after();
        uint32_t sr[GP];
        tmem_ld_cols<GP>(t_s + lane_base, sr);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_empty);
        const int vp = 2 * c + (r >> 6), tok = w.s.page(vp) * PAGE + (r & 63);
        const bool valid = vp < w.s.pages && tok < w.s.n && (tok >= w.s.lo || tok < w.s.sinks);
        if (!valid) {
          // The P V product reads all 128 rows of V: those that no token is
          // visible in hold stale or never-written memory, and 0 * NaN = NaN,
          // so they are zeroed once this chunk's V copies have landed.
          if (!mbar_wait(&sm.vfull, cc & 1, FB_KERR_TIMEOUT_FULL)) *give_up = 1;
          uint8_t* vrow = sm.v + r * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint4*>(vrow + h * HALF_STRIDE)[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float s = valid ? __uint_as_float(sr[g]) * a.scale_log2 : -INFINITY;
          sr[g] = __float_as_uint(s);
          const float cmax = warp_max(s);
          if (lane == 0) sm.red[quarter][g] = cmax;
        }
        sync_softmax();
        if (*give_up) break;  // the same in every softmax thread: written only outside this pair of barriers
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float mx = fmaxf(fmaxf(sm.red[0][g], sm.red[1][g]), fmaxf(sm.red[2][g], sm.red[3][g]));
          const float m_old = sm.mrun[cc & 1][g];
          const float m_new = fmaxf(m_old, mx);
          const float m_use = m_new == -INFINITY ? 0.f : m_new;
          const float alpha = exp2f(m_old - m_use);
          if (r == 0) {
            sm.alpha[g] = alpha;
            sm.mrun[(cc + 1) & 1][g] = m_new;
          }
          const float p = exp2f(__uint_as_float(sr[g]) - m_use);
          l_thr[g] = l_thr[g] * alpha + p;
          if (g < G) *reinterpret_cast<bf16*>(sm.p + qp_offset(g, r)) = f2bf(p);
        }
        fence_proxy_async();
        sync_softmax();  // red and alpha are rewritten next chunk
        if (lane == 0) mbar_arrive(&sm.p_full);
        if (!mbar_wait(&sm.o_full, cc & 1, FB_KERR_TIMEOUT_TMEM)) *give_up = 1;
        tc_fence_after();
        uint32_t orr[GP];
        tmem_ld_cols<GP>(t_o + lane_base, orr);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty);
#pragma unroll
        for (int g = 0; g < GP; ++g) o[g] = o[g] * sm.alpha[g] + __uint_as_float(orr[g]);
      }
      // Sum of a head over the 128 token lanes.
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const float ls = warp_sum(l_thr[g]);
        if (lane == 0) sm.red[quarter][g] = ls;
      }
      sync_softmax();
      if (*give_up) break;  // again the same in every thread; the workspace's tickets are then left as they are
      float m[GP], l[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        l[g] = (sm.red[0][g] + sm.red[1][g]) + (sm.red[2][g] + sm.red[3][g]);
        m[g] = sm.mrun[cc & 1][g];
      }
      // This piece's item starts at flat position `at0` and lies in the shares of CTAs [f, e].
      const int at0 = w.at - w.c0, f = at0 / share, pieces = (at0 + w.s.chunks - 1) / share - f + 1;
      bool finish = true;
      if (pieces > 1) {
        const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (w.at == begin ? 0 : 1);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          __stcg(a.ws_o + (slot * GP + g) * D + r, o[g]);
          if (r == 0) __stcg(reinterpret_cast<float2*>(a.ws_ml) + slot * GP + g, make_float2(m[g], l[g]));
        }
        __threadfence();
        sync_softmax();
        if (r == 0) {
          __threadfence();
          const int done = atomicAdd(a.tickets + f, 1) + 1;
          sm.last = done == pieces;
          if (done == pieces) a.tickets[f] = 0;
          __threadfence();
        }
        sync_softmax();
        finish = sm.last;
        if (finish) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            m[g] = -INFINITY;
            l[g] = o[g] = 0.f;
          }
          for (int k = 0; k < pieces; ++k) {
            const size_t from = 2 * static_cast<size_t>(f + k) + (k == 0 && at0 % share ? 1 : 0);
#pragma unroll
            for (int g = 0; g < GP; ++g) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + from * GP + g);
              const float op = __ldcg(a.ws_o + (from * GP + g) * D + r);
              const float mx = fmaxf(m[g], ml.x), ref = mx == -INFINITY ? 0.f : mx;
              const float w0 = exp2f(m[g] - ref), w1 = exp2f(ml.x - ref);
              l[g] = l[g] * w0 + ml.y * w1;
              o[g] = o[g] * w0 + op * w1;
              m[g] = mx;
            }
          }
        }
      }
      if (finish) {
        const int np = a.row_info ? a.row_info[w.b].y : 0;
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          if (g >= G) break;
          const int hq = w.kvh * G + g;
          const size_t at = (static_cast<size_t>(w.b) * Hq + hq) * a.prefix_parts;
          for (int k = 0; k < np; ++k) {
            const float2 ml = *(reinterpret_cast<const float2*>(a.prefix_ml) + at + k);
            const float op = a.prefix_o[(at + k) * D + r];
            const float mx = fmaxf(m[g], ml.x), ref = mx == -INFINITY ? 0.f : mx;
            const float w0 = exp2f(m[g] - ref), w1 = exp2f(ml.x - ref);
            l[g] = l[g] * w0 + ml.y * w1;
            o[g] = o[g] * w0 + op * w1;
            m[g] = mx;
          }
          a.out[w.b * a.ld_o + hq * D + r] = f2bf(l[g] > 0.f ? o[g] / l[g] : 0.f);
        }
      }
      sync_softmax();  // red, mrun and last are rewritten by the next piece
    }
    if (*give_up) sm.abort = 1;
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 32);
}

}  // namespace

// Caches viewed as [blocks * Hkv * 64, 128], K and V with boxes of a page x 64
// dims, then K and V with boxes of 16 rows x 64 dims, 128B swizzle.
struct SpanMaps {
  CUtensorMap k, v, k16, v16;
};

#define FB_SPAN_INSTANCE(GP, CTAS)                                                                                \
  extern "C" __global__ void __launch_bounds__(THREADS, CTAS) fb_span_attn_g##GP(                                 \
      const __grid_constant__ SpanMaps maps, const bf16* q, long long ld_q, const int* block_tables,              \
      int max_blocks, int blocks, const int* seq_lens, bf16* out, long long ld_o, int B, int Hkv, int G,          \
      int window, int sinks, const int2* row_info, const float* prefix_o, const float* prefix_ml,                 \
      int prefix_parts, float* ws_o, float* ws_ml, int* tickets, float scale_log2) {                              \
    const Params a{q,     block_tables, seq_lens, row_info, out, prefix_o, prefix_ml,    ws_o,   ws_ml, tickets,  \
                   ld_q,  ld_o,         max_blocks, blocks, B,   Hkv,      G,            prefix_parts, window,    \
                   sinks, scale_log2};                                                                            \
    span_body<GP>(&maps.k, &maps.v, &maps.k16, &maps.v16, a);                                                     \
  }

FB_SPAN_INSTANCE(4, 3)
FB_SPAN_INSTANCE(8, 3)
FB_SPAN_INSTANCE(16, 2)
