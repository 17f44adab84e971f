// Paged GQA decode attention over part of each sequence, on the tcgen05 tensor
// cores (head_dim 128, bf16 K/V pages of 64 tokens, fp32 softmax state). The
// visible tokens of a sequence of n tokens are
//
//   window > 0:  [0, min(sinks, n)) and [max(n - window, 0), n)
//   window = 0:  [start, n), start = the tokens that fb_prefix_attn_* has
//                attended to for the whole group (row_prefix)
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
// Measured (B200), K and V of the visible tokens over the time: 256 rows of 1024
// tokens, 32 / 8 heads 168 us (97% of the 6545 GB/s of a plain copy); 61 rows of
// 4160 tokens, 32 / 4 heads 88 us (89%); 256 rows of 1 to 640 tokens 63 us (81%);
// 1024 rows of 64 tokens 57 us (72%); one row of 1028 tokens 9.2 us. A launch's
// start (lengths, page numbers, first K) and end (last chunk, join) take 6 to 9 us;
// between them a full chunk's chain is hidden by the other CTAs' loads, a row of
// one chunk takes 3.9 k clocks of a CTA.
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
  uint64_t s_full, s_empty, p_full, o_full, o_empty;
  uint64_t mma_done;  // the products of an MMA warp that gave up
  float red_max[4][NH], red_sum[4][NH];  // of a warp's tokens, for every head
  float mrun[2][NH];   // running max per head: one in use, one for the next move
  int scan[THREADS / 32];
  int first_row, first_off;
  int2 first_length;
  uint32_t tmem;
  struct {
    int f, pieces, odd, b, kvh, last;
  } cut[2];  // the pieces of items that lie in other CTAs' shares too: at most the first and the last one
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

// The softmax threads' barrier, and whether any of them brings true.
__device__ __forceinline__ bool sync_softmax_or(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void sync_softmax() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Caches viewed as [blocks * Hkv * 64, 128], K and V with boxes of a page x 64
// dims, then K and V with boxes of 16 rows x 64 dims; q [B][Hq][128] with boxes
// of one KV head's heads x 64 dims. 128B swizzle.
struct SpanMaps {
  CUtensorMap k, v, k16, v16, q;
};

struct Params {
  const int* block_tables;
  const int* seq_lens;
  const int* row_prefix;  // tokens of each row that the prefix kernel has attended to, or null
  bf16* out;
  const float *prefix_o, *prefix_ml;  // its results, (row * Hq + head) * parts + part
  float *ws_o, *ws_ml;                // [2 * gridDim][Hq / Hkv rounded up to the variant][128] and [..][2]
  int* tickets;                       // [gridDim], zero between launches
  long long ld_o;
  int max_blocks, blocks, B, Hkv, G, parts, window, sinks;
  float scale_log2;
};

// The visible tokens of a row: t < n and (t >= lo or t < sinks), on the
// virtual pages 0 .. pages - 1: first those of the sinks, then from page `wp`.
struct Span {
  int n, lo, sinks, sp, wp, pages, chunks;
  bool prefix;  // the row has a partial result from the prefix kernel
  __device__ __forceinline__ int page(int v) const { return v < sp ? v : v - sp + wp; }
};

// (length, prefix tokens) of a row; a row behind the last one is empty.
__device__ __forceinline__ int2 row_length(const Params& a, int b) {
  return b < a.B ? make_int2(a.seq_lens[b], a.row_prefix ? a.row_prefix[b] : 0) : make_int2(0, 0);
}

__device__ __forceinline__ Span row_span(const Params& a, int2 length) {
  Span s;
  s.n = min(max(length.x, 0), a.max_blocks * PAGE);
  s.prefix = length.y > 0;
  s.lo = a.window > 0 ? max(s.n - a.window, 0) : min(length.y, s.n);
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
  int2 ahead;  // the next row's length, read a row ahead: off the critical path
  __device__ __forceinline__ Walk(const Params& a, const Smem& sm, int begin, int e) : b(sm.first_row), at(begin), end(e) {
    if (begin >= end) return;
    s = row_span(a, sm.first_length);
    ahead = row_length(a, b + 1);
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
      s = row_span(a, ahead);
      ahead = row_length(a, ++b + 1);
    }
    c1 = min(s.chunks, end - at);
  }
};

__device__ __forceinline__ int add_acq_rel(int* p, int v) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// One head's output row from the partial results of n pieces: *ml(k) = (max, sum),
// part(k)[0 .. 127], a lane with four dims. The loads of JOIN pieces are on their
// way at a time: one by one, their latency is what the join would take.
constexpr int JOIN = 8;
template <class Ml, class Part>
__device__ __forceinline__ float4 join_pieces(int n, Ml ml, Part part) {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += JOIN) {
    float2 s[JOIN];
    float4 v[JOIN];
#pragma unroll
    for (int k = 0; k < JOIN; ++k) {
      s[k] = __ldcg(ml(min(k0 + k, n - 1)));
      v[k] = __ldcg(reinterpret_cast<const float4*>(part(min(k0 + k, n - 1))) + (threadIdx.x & 31));
    }
    float mx = m;
#pragma unroll
    for (int k = 0; k < JOIN; ++k) {
      if (k0 + k >= n) s[k] = make_float2(-INFINITY, 0.f);
      mx = fmaxf(mx, s[k].x);
    }
    const float ref = mx == -INFINITY ? 0.f : mx, w = exp2f(m - ref);
    l *= w;
    o = make_float4(o.x * w, o.y * w, o.z * w, o.w * w);
#pragma unroll
    for (int k = 0; k < JOIN; ++k) {
      const float e = exp2f(s[k].x - ref);
      l = fmaf(s[k].y, e, l);
      o = make_float4(fmaf(v[k].x, e, o.x), fmaf(v[k].y, e, o.y), fmaf(v[k].z, e, o.z), fmaf(v[k].w, e, o.w));
    }
    m = mx;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros; NaN stays NaN
  return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

template <int GP>
__device__ __forceinline__ void span_body(const SpanMaps& maps, const Params& a) {
  const CUtensorMap *tmK = &maps.k, *tmV = &maps.v, *tmK16 = &maps.k16, *tmV16 = &maps.v16;
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
    mbar_init(&sm.mma_done, 1);
    sm.abort = sm.give_up = 0;
    fence_barrier_init();
    fence_proxy_async();
    tma_prefetch_desc(tmK);
    tma_prefetch_desc(tmV);
    tma_prefetch_desc(tmK16);
    tma_prefetch_desc(tmV16);
    tma_prefetch_desc(&maps.q);
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 32);
    tmem_relinquish();
  }
  // Rows of heads >= G are never written: zeros, if only so that what the
  // products make of them is finite (each head's column depends on its own row).
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
    mine += row_span(a, row_length(a, b)).chunks * a.Hkv;
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
      sm.first_length = row_length(a, b);
      const int len = row_span(a, sm.first_length).chunks * a.Hkv;
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
      uint32_t loads[2] = {};  // of K and of V
      bool ok = true;
      for (Walk w(a, sm, begin, end); ok && w.more() && !*(volatile int*)&sm.abort; w.next(a)) {
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
            ok = mbar_wait(kv ? &sm.vempty : &sm.kempty, (loads[kv] & 1) ^ 1, FB_KERR_TIMEOUT_EMPTY);
            if (!ok) break;
            ++loads[kv];
            // An item's q rows come with its first K: the last item's Q K^T is done by then.
            const bool first = kv == 0 && c == w.c0;
            mbar_arrive_expect_tx(full, bytes + (first ? a.G * D * 2 : 0));
            if (first)
              for (int hf = 0; hf < 2; ++hf)
                tma_load_3d(sm.q + hf * (NH * 128), &maps.q, full, hf * 64, w.kvh * a.G, w.b);
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
          if (!ok || *(volatile int*)&sm.abort) break;
        }
      }
      // Drain: every issued copy has been consumed, or has landed at least where a
      // wait ran out (parity 1 of a barrier that nothing was ever sent to is behind it).
      ok = ok && mbar_wait(&sm.kempty, (loads[0] & 1) ^ 1, FB_KERR_TIMEOUT_EMPTY) &&
           mbar_wait(&sm.vempty, (loads[1] & 1) ^ 1, FB_KERR_TIMEOUT_EMPTY);
      if (!ok) {
        sm.abort = 1;
        mbar_wait(&sm.kfull, (loads[0] & 1) ^ 1, FB_KERR_TIMEOUT_FULL);
        mbar_wait(&sm.vfull, (loads[1] & 1) ^ 1, FB_KERR_TIMEOUT_FULL);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t kb = smem_u32(sm.k), vb = smem_u32(sm.v), qb = smem_u32(sm.q), pb = smem_u32(sm.p);
      uint32_t cc = 0;  // chunks so far
      bool ok = true;
      for (Walk w(a, sm, begin, end); ok && w.more() && !*(volatile int*)&sm.abort; w.next(a)) {
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
      if (!ok) {
        sm.abort = 1;
        // no product is under way when the CTA frees its tensor memory
        mma_commit(&sm.mma_done);
        mbar_wait(&sm.mma_done, 0, FB_KERR_TIMEOUT_TMEM);
      }
    }
  } else {
    // ---------------- softmax / epilogue (warps 2..5) ----------------
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // TMEM lane: token (for S) / head dim (for O)
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const int G = a.G, Hq = a.Hkv * G;
    uint32_t cc = 0;
    int cuts = 0;
    bool stop = false;
    int cur = 0;  // which of mrun is in use (the same in all threads)
    volatile int* give_up = &sm.give_up;
    for (Walk w(a, sm, begin, end); w.more(); w.next(a)) {
      float l_thr[GP], o[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        if (r == 0) sm.mrun[cur][g] = -INFINITY;
        l_thr[g] = o[g] = 0.f;
      }
      if (w.s.prefix && w.c0 == 0) {
        // The item's first piece goes on from the prefix's results (read while its
        // first chunk is on its way).
        const size_t head = static_cast<size_t>(w.b) * Hq + w.kvh * G;
        if (a.parts == 1) {  // nothing waits for these loads before the first P V is there
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const size_t at = head + min(g, G - 1);
            o[g] = a.prefix_o[at * D + r];
            if (r == 0) {
              sm.mrun[cur][g] = a.prefix_ml[2 * at];
              l_thr[g] = a.prefix_ml[2 * at + 1];
            }
          }
        }
#pragma unroll
        for (int g0 = 0; g0 < GP; g0 += 4) {
          if (a.parts == 1) break;
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int k = 0; k < a.parts; ++k) {
            float2 ml[4];
            float op[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const size_t at = (head + min(g0 + g, G - 1)) * a.parts + k;
              ml[g] = __ldcg(reinterpret_cast<const float2*>(a.prefix_ml) + at);
              op[g] = __ldcg(a.prefix_o + at * D + r);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float mx = fmaxf(m[g], ml[g].x), ref = mx == -INFINITY ? 0.f : mx;
              const float w0 = exp2f(m[g] - ref), w1 = exp2f(ml[g].x - ref);
              o[g0 + g] = o[g0 + g] * w0 + op[g] * w1;
              l_thr[g0 + g] = r == 0 ? l_thr[g0 + g] * w0 + ml[g].y * w1 : 0.f;
              m[g] = mx;
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (r == 0) sm.mrun[cur][g0 + g] = m[g];
        }
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
        // The maxima move only if a score is above one by more than 8 (log2
        // units: p stays below 256, exact in the fp32 sums), and in a piece's
        // first chunk: the reduction over the tokens is for those chunks alone.
        bool move = c == w.c0;
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float s = valid ? __uint_as_float(sr[g]) * a.scale_log2 : -INFINITY;
          sr[g] = __float_as_uint(s);
          move |= g < G && c > w.c0 && s > sm.mrun[cur][g] + 8.f;
        }
        if (c > w.c0) {
          move = sync_softmax_or(move);
          if ((stop = *give_up)) break;  // the same in every softmax thread: written only outside this pair of barriers
        }
        if (move) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float cmax = warp_max(__uint_as_float(sr[g]));
            if (lane == 0) sm.red_max[quarter][g] = cmax;
          }
          sync_softmax();
          if (c == w.c0 && (stop = *give_up)) break;  // (as above)
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float mx =
                fmaxf(fmaxf(sm.red_max[0][g], sm.red_max[1][g]), fmaxf(sm.red_max[2][g], sm.red_max[3][g]));
            const float m_old = sm.mrun[cur][g], m_new = fmaxf(m_old, mx);
            const float alpha = exp2f(m_old - (m_new == -INFINITY ? 0.f : m_new));
            if (r == 0) sm.mrun[cur ^ 1][g] = m_new;
            sr[g] = __float_as_uint(__uint_as_float(sr[g]) - (m_new == -INFINITY ? 0.f : m_new));
            l_thr[g] *= alpha;
            o[g] *= alpha;
          }
          cur ^= 1;
        } else {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float m = sm.mrun[cur][g];
            sr[g] = __float_as_uint(__uint_as_float(sr[g]) - (m == -INFINITY ? 0.f : m));
          }
        }
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float p = exp2f(__uint_as_float(sr[g]));
          l_thr[g] += p;
          if (g < G) *reinterpret_cast<bf16*>(sm.p + qp_offset(g, r)) = f2bf(p);
        }
        bool late = false;
        if (!valid) {
          // The P V product reads all 128 rows of V: those that no token is
          // visible in hold stale or never-written memory, and 0 * NaN = NaN,
          // so they are zeroed once this chunk's V copies have landed. (Each
          // lane from its own 16 bytes on: a warp's lanes in different banks.)
          late = !mbar_wait(&sm.vfull, cc & 1, FB_KERR_TIMEOUT_FULL);
          uint8_t* vrow = sm.v + r * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint4*>(vrow + h * HALF_STRIDE)[i ^ (r & 7)] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        sync_softmax();
        if (lane == 0) mbar_arrive(&sm.p_full);
        if (c + 1 == w.c1) {  // the heads' sums over the token lanes, while P V is on its way
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float ls = warp_sum(l_thr[g]);
            if (lane == 0) sm.red_sum[quarter][g] = ls;
          }
          sync_softmax();
        }
        if (late || !mbar_wait(&sm.o_full, cc & 1, FB_KERR_TIMEOUT_TMEM)) *give_up = 1;
        tc_fence_after();
        uint32_t orr[GP];
        tmem_ld_cols<GP>(t_o + lane_base, orr);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty);
#pragma unroll
        for (int g = 0; g < GP; ++g) o[g] += __uint_as_float(orr[g]);
      }
      if (stop) break;
      auto sum = [&](int g) {
        return (sm.red_sum[0][g] + sm.red_sum[1][g]) + (sm.red_sum[2][g] + sm.red_sum[3][g]);
      };
      if (w.c0 == 0 && w.c1 == w.s.chunks) {
        bf16* to = a.out + w.b * a.ld_o + w.kvh * G * D;
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float l = sum(g);
          if (g < G) to[g * D + r] = f2bf(l == 0.f ? 0.f : o[g] / l);
        }
      } else {
        const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (w.at == begin ? 0 : 1);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          __stcg(a.ws_o + (slot * GP + g) * D + r, o[g]);
          if (r == 0) __stcg(reinterpret_cast<float2*>(a.ws_ml) + slot * GP + g, make_float2(sm.mrun[cur][g], sum(g)));
        }
        if (r == 0) {
          // The item starts at flat position `at0` and lies in the shares of CTAs f, f + 1, ..;
          // odd: its first piece is its CTA's last.
          const int at0 = w.at - w.c0, f = at0 / share;
          sm.cut[cuts] = {f, (at0 + w.s.chunks - 1) / share - f + 1, at0 % share ? 1 : 0, w.b, w.kvh, 0};
        }
        ++cuts;
      }
    }
    // Cut items, last: by now the first piece's results have long been written, and
    // nothing has had to wait for that.
    sync_softmax();
    if (*give_up) {  // the workspace's tickets are left as they are
      sm.abort = 1;
    } else if (cuts) {
      if (lane == 0 && quarter < cuts) {
        // releases the warps' writes (ordered before it by the barrier), acquires the other pieces'
        auto& cut = sm.cut[quarter];
        const int done = add_acq_rel(a.tickets + cut.f, 1) + 1;
        cut.last = done == cut.pieces;
        if (done == cut.pieces) a.tickets[cut.f] = 0;
      }
      sync_softmax();
      for (int i = 0; i < cuts; ++i) {
        const auto cut = sm.cut[i];
        if (!cut.last) continue;
#pragma unroll 1
        for (int g = quarter; g < G; g += 4) {
          auto at = [&](int k) { return (2 * static_cast<size_t>(cut.f + k) + (k == 0 ? cut.odd : 0)) * GP + g; };
          const float4 v = join_pieces(
              cut.pieces, [&](int k) { return reinterpret_cast<const float2*>(a.ws_ml) + at(k); },
              [&](int k) { return a.ws_o + at(k) * D; });
          uint2 packed;
          *reinterpret_cast<bf162*>(&packed.x) = __floats2bfloat162_rn(v.x, v.y);
          *reinterpret_cast<bf162*>(&packed.y) = __floats2bfloat162_rn(v.z, v.w);
          *reinterpret_cast<uint2*>(a.out + cut.b * a.ld_o + (cut.kvh * G + g) * D + lane * 4) = packed;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 32);
}

}  // namespace

#define FB_SPAN_INSTANCE(GP, CTAS)                                                                                \
  extern "C" __global__ void __launch_bounds__(THREADS, CTAS) fb_span_attn_g##GP(                                 \
      const __grid_constant__ SpanMaps maps, const int* block_tables, int max_blocks, int blocks,                 \
      const int* seq_lens, bf16* out, long long ld_o, int B, int Hkv, int G, int window, int sinks,               \
      const int* row_prefix, const float* prefix_o, const float* prefix_ml, int parts, float* ws_o, float* ws_ml, \
      int* tickets, float scale_log2) {                                                                           \
    const Params a{block_tables, seq_lens, row_prefix, out, prefix_o, prefix_ml, ws_o,   ws_ml,                   \
                   tickets,      ld_o,     max_blocks, blocks, B,     Hkv,       G,      parts, window,           \
                   sinks,        scale_log2};                                                                     \
    span_body<GP>(maps, a);                                                                                       \
  }

FB_SPAN_INSTANCE(4, 3)
FB_SPAN_INSTANCE(8, 3)
FB_SPAN_INSTANCE(16, 2)
