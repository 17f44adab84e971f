// Log probability of a given token, entropy and the k most probable tokens of
// each row of logits [T, V] (bf16, fp16 or fp32), in one pass over the logits.
//
// With y = (x - max) log2(e), Z = sum 2^y, U = sum 2^y y:
//   log p(t) = x_t - max - ln Z        H = ln Z - U ln 2 / Z
// (both terms of H are >= 0, so nothing cancels). Each thread keeps its own
// running max and rescales (Z, U) when it moves, once per 64 bytes at most; Z
// and U are fp32 sums: of the 64 bytes, of those, then a tree over the threads.
//
// The k largest (ties: lowest token) come from the same pass: each thread also
// knows the max of what it has read. The block's 256 threads make 64 groups,
// and the k-th largest of the groups' maxima bounds the k-th largest logit from
// below. Only the parts of threads whose max reaches that bound - about k of
// them, but for ties - are read again (from L2, by the whole block), and what
// reaches the bound is listed; the list, rarely longer than 2 k, is ranked by
// counting. Two ways out keep that exact for any input: with more than 256 on the
// list, those above the bound are listed alone, and of the equal ones at it the
// first in token order are taken, 256 logits at a time until enough are found (a
// constant row, or one masked but for a few tokens, ends in its first step); more
// logits above the bound than the list holds (few threads' parts hold many of the
// largest) are found by k passes.
//
// With k = 0 the kernel is bound by reading the logits (2000 x 151936: fp32 all of a
// plain copy's rate, bf16 85%: one 2^x per 2 bytes takes 72% of what the
// special-function units give at that rate). The choice of the k largest comes at a
// row's end, while its CTA reads nothing: 2000 rows in bf16, k = 0 / 1 / 20 109 / 127 /
// 159 us. Each thread
// copies its next 128 bytes into its own slots of shared memory while it works on
// 64, which takes neither registers nor barriers. (Slower: loads ahead into
// registers, which spill; a ring of bulk copies for the block, whose barriers cost
// as many instructions as the sums do.) Up to as many rows as CTAs, a row has a
// whole number of CTAs, so that no CTA ends two rows; beyond, the flat sequence of
// all logits is cut into one equal share per CTA. A row that a cut falls into is
// joined by the CTA that finishes its last piece, through a workspace of two pieces
// per CTA and one ticket per cut (zero before and after every launch). The join is
// in piece order, so results do not depend on which CTA comes last.
//
// Measured (B200): 2000 x 151936, k = 1: fp32 185 us in a graph, 197 call by call (94%
// of the 6545 GB/s of a plain copy), bf16 127 us (73%), fp16 125 us; 256 x 128256 bf16, k = 0 / 5 / 20 16.7 / 19.2 / 21.3 us
// (3.9 / 3.4 / 3.1 TB/s: two rows on most SMs, 1.73 on average), of which constant
// rows 27 us and rows masked but for three tokens 42 us; one row, k = 5 8.7 us.
#include <cuda_fp16.h>

#include "fb_common.cuh"

FB_DEFINE_STATUS

using namespace fbk;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_K = 32;
constexpr int LIST = 1024;   // logits that reach the bound
constexpr int PLAIN = 256;   // so many are ranked as they are; of more, first those above the bound
constexpr int MAX_PIECES = 1024;  // of a row: at most the grid, and two
constexpr int GROUPS = 64;            // of THREADS / GROUPS neighbouring threads
constexpr int U = 4;          // vectors that a thread works on at a time
constexpr int SLOTS = 3;      // as many of these are on their way, less the one in work
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453094;

// Order of candidates: larger logit first, then the lower token. 0 = none.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 -> +0: equal logits tie
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned up) {
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ unsigned long long make_key(float x, int token) {
  return static_cast<unsigned long long>(ordered(x)) << 32 | static_cast<unsigned>(~token);
}
__device__ __forceinline__ int key_token(unsigned long long k) { return static_cast<int>(~static_cast<unsigned>(k)); }
__device__ __forceinline__ float key_value(unsigned long long k) { return from_ordered(static_cast<unsigned>(k >> 32)); }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

template <class T>
struct Pair {
  using type = bf162;
};
template <>
struct Pair<__half> {
  using type = __half2;
};

// The logits of one 16-byte vector; the largest of U of them, NaN ignored.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  __device__ __forceinline__ static void unpack(const uint4& u, float (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(u.x);
      f[1] = __uint_as_float(u.y);
      f[2] = __uint_as_float(u.z);
      f[3] = __uint_as_float(u.w);
    } else {
      const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_float(h[i]);
    }
  }
  __device__ __forceinline__ static float max_of(const uint4 (&u)[U]) {
    if constexpr (sizeof(T) == 4) {
      float mx = -INFINITY;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float f[N];
        unpack(u[q], f);
        mx = fmaxf(mx, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
      }
      return mx;
    } else {
      using T2 = typename Pair<T>::type;
      const T2* h = reinterpret_cast<const T2*>(u);
      T2 hi = h[0];
#pragma unroll
      for (int i = 1; i < 4 * U; ++i) hi = __hmax2(hi, h[i]);
      return fmaxf(to_float(hi.x), to_float(hi.y));
    }
  }
};

// Softmax sums relative to the logit `ref`: z = sum 2^y, u = sum 2^y y with
// y = (x - ref) log2(e). Nothing read yet: ref is fp32's lowest value, so that a
// row masked with its type's lowest value still has a distribution; a row of
// -inf alone has z = 0.
struct Sums {
  float ref, z, u;
  __device__ __forceinline__ void clear() {
    ref = -3.402823466e38f;
    z = u = 0.f;
  }
  __device__ __forceinline__ void move(float to) {  // to >= ref
    const float d = (to - ref) * LOG2E, f = exp2f(-d);
    u = f > 0.f ? f * (u - d * z) : 0.f;
    z *= f;
    ref = to;
  }
  __device__ __forceinline__ void add(float x) {
    // a logit of -inf has p = 0 and no share of u; NaN passes through
    const float y = max_nan((x - ref) * LOG2E, -200.f);
    const float e = exp2f(y);
    z += e;
    u = fmaf(e, y, u);
  }
  // Four logits as packed pairs; where one is so low that y = -inf, u2 becomes NaN.
  __device__ __forceinline__ void add4(const float (&x)[4], float2& z2, float2& u2) const {
    const float2 r = make_float2(-ref, -ref), l = make_float2(LOG2E, LOG2E);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), r), l);
      const float2 e = make_float2(exp2f(y.x), exp2f(y.y));
      z2 = __fadd2_rn(z2, e);
      u2 = __ffma2_rn(e, y, u2);
    }
  }
  __device__ __forceinline__ void join(Sums o) {
    const float to = fmaxf(ref, o.ref);
    move(to);
    o.move(to);
    z += o.z;
    u += o.u;
  }
};

__device__ __noinline__ Sums join_warp(Sums s) {
  s.move(warp_max(s.ref));
  s.z = warp_sum(s.z);
  s.u = warp_sum(s.u);
  return s;
}

struct Smem {
  uint4 ring[SLOTS][U][THREADS];  // each thread's own slots
  unsigned long long list[LIST], heads[MAX_PIECES];
  int2 hit[LIST];  // (vector, its place in the ring) of vectors that reach the bound
  unsigned char head_rank[MAX_PIECES];
  float group_max[GROUPS];
  unsigned char listed[THREADS];  // threads whose max reaches the bound
  int n_listed;
  Sums sums[WARPS];
  unsigned long long best[MAX_K];
  unsigned long long key;
  unsigned bound;  // ordered bits
  int n_list, n_hit, last;
  int scan[WARPS];
};
static_assert(sizeof(Smem) <= 75 * 1024, "host requests 75 KB of dynamic shared memory (3 CTAs per SM; 4 would spill)");

// (From its name in every function: passed on as a reference it would be
// accessed through generic addresses.)
__device__ __forceinline__ Smem& smem() {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  return *reinterpret_cast<Smem*>(smem_raw);
}

struct Params {
  const void* logits;
  long long ld;
  const int* ids;
  float *logprobs, *entropy, *top_logprobs;
  int* top_ids;
  float* ws_sums;                 // [2 * gridDim][4]
  unsigned long long* ws_keys;    // [2 * gridDim][MAX_K]
  int* tickets;                   // [gridDim], zero between launches
  // CTA i has the flat positions [i * share, (i + 1) * share); row r's logits
  // begin at r * pitch (V, or rows padded to whole shares)
  long long share, pitch;
  int T, V, k;
};

// 16 bytes from global to shared memory behind the thread's back.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// The largest key of the block below `below`; all threads get it.
__device__ __forceinline__ unsigned long long block_max(Smem& sm, unsigned long long key) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  if (threadIdx.x == 0) sm.key = 0;
  __syncthreads();
  if ((threadIdx.x & 31) == 0 && key) atomicMax(&sm.key, key);
  __syncthreads();
  key = sm.key;
  __syncthreads();
  return key;
}

// The rank of each of `n` keys among them: 8 threads count for one key. Every
// thread of the block calls it; put(i, rank) runs once for each key.
template <class Put>
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int n, Put put) {
  const int part = threadIdx.x & 7;
  for (int i0 = 0; i0 < n; i0 += THREADS / 8) {
    const int i = i0 + (threadIdx.x >> 3);
    const unsigned long long mine = keys[min(i, n - 1)];
    int rank = 0;
#pragma unroll 8
    for (int j = part; j < n; j += 8) rank += keys[j] > mine;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (part == 0 && i < n) put(i, rank);
  }
}

// sm.best[0..k) = the piece's k largest keys (0 where there are fewer), from
// logits x[0..n) that start at token `first`; tmax: the max of this thread's
// part (vectors tid, tid + THREADS, ..; a logit of the head and of the tail).
template <class T>
__device__ __noinline__ void piece_top(const T* x, int n, int head, int vecs, int first, float tmax, int k) {
  Smem& sm = smem();
  constexpr int N = Vec<T>::N, PER = THREADS / GROUPS;
  const int tid = threadIdx.x;
  float gmax = tmax;
#pragma unroll
  for (int o = 1; o < PER; o <<= 1) gmax = fmaxf(gmax, __shfl_xor_sync(0xffffffffu, gmax, o));
  if (tid % PER == 0) sm.group_max[tid / PER] = gmax;
  if (tid == 0) {
    sm.n_list = sm.n_listed = 0;
    sm.bound = ~0u;
  }
  if (tid < MAX_K) sm.best[tid] = 0;
  __syncthreads();
  {
    // The bound is the smallest group max with fewer than k above it; PER threads count for each.
    int more = 0;
    const float4* part = reinterpret_cast<const float4*>(sm.group_max) + tid % PER * (GROUPS / 4 / PER);
#pragma unroll
    for (int j = 0; j < GROUPS / 4 / PER; ++j) {
      const float4 o = part[j];
      more += (o.x > gmax) + (o.y > gmax) + (o.z > gmax) + (o.w > gmax);
    }
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    const unsigned low = __reduce_min_sync(0xffffffffu, more < k ? ordered(gmax) : ~0u);
    if ((tid & 31) == 0) atomicMin(&sm.bound, low);
  }
  __syncthreads();
  const float bound = from_ordered(sm.bound);
  if (tmax >= bound) sm.listed[atomicAdd(&sm.n_listed, 1)] = static_cast<unsigned char>(tid);
  __syncthreads();
  // Lists what reaches the bound (or, with `above`, passes it): the listed
  // threads' vectors come back into the ring, as many as it holds at a time.
  // Ends as soon as there is more than the list holds.
  auto collect = [&](bool above) {
    auto look = [&](float f, int i) {
      if (f > bound || (f == bound && !above)) {
        const int at = atomicAdd(&sm.n_list, 1);
        if (at < LIST) sm.list[at] = make_key(f, first + i);
      }
    };
    if (tid < head) look(to_float(x[tid]), tid);
    const int tail = head + vecs * N;
    if (tid < n - tail) look(to_float(x[tail + tid]), tail + tid);
    constexpr int ROOM = SLOTS * U * THREADS;
    uint4* ring = &sm.ring[0][0][0];
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    const int threads = sm.n_listed, lane = tid & 31, warp = tid >> 5, all = (vecs + THREADS - 1) / THREADS;
    for (int j0 = 0; j0 < all; j0 += ROOM) {  // vectors j0 .. j0 + len of `take` listed threads at a time
      const int len = min(ROOM, all - j0), take = ROOM / len;
      for (int l0 = 0; l0 < threads; l0 += take) {
        const int l1 = min(l0 + take, threads);
        auto each = [&](auto f) {
#pragma unroll 1
          for (int l = l0 + warp; l < l1; l += WARPS)
#pragma unroll 1
            for (int j = lane; j < len; j += 32)
              if (const int at = sm.listed[l] + (j0 + j) * THREADS; at < vecs) f(at, (l - l0) * len + j);
        };
        each([&](int at, int slot) { copy16(ring + slot, v + at); });
        copy_commit();
        if (tid == 0) sm.n_hit = 0;
        copy_wait<0>();
        __syncthreads();
        each([&](int at, int slot) {  // vectors that reach (pass) the bound ..
          float f[N];
          Vec<T>::unpack(ring[slot], f);
          float mx = f[0];
#pragma unroll
          for (int e = 1; e < N; ++e) mx = fmaxf(mx, f[e]);
          if (above ? mx > bound : mx >= bound)
            if (const int i = atomicAdd(&sm.n_hit, 1); i < LIST) sm.hit[i] = make_int2(at, slot);
        });
        __syncthreads();
        const int hits = sm.n_hit;
        if (hits > LIST && tid == 0) atomicAdd(&sm.n_list, LIST + 1);  // more logits than that, too
        for (int i = tid; i < min(hits, LIST) * N; i += THREADS) {  // .. and their logits, one to a thread
          const int2 h = sm.hit[i / N];
          look(to_float(reinterpret_cast<const T*>(ring + h.y)[i % N]), head + h.x * N + i % N);
        }
        __syncthreads();
        if (sm.n_list > LIST) return;  // (the same in all threads: written again behind the next barrier)
      }
    }
    __syncthreads();
  };
  auto keep = [&](int i, int rank) {
    if (rank < k) sm.best[rank] = sm.list[i];
  };
  collect(false);
  const int listed = sm.n_list;
  bool ties = listed > LIST;
  if (listed > PLAIN && !ties) {  // ties at the bound, or many different logits above it?
    unsigned long long mine[LIST / THREADS];
    int more = 0;
    const unsigned long long at_bound = static_cast<unsigned long long>(ordered(bound)) << 32 | 0xffffffffu;
#pragma unroll
    for (int q = 0; q < LIST / THREADS; ++q) {
      mine[q] = tid + q * THREADS < listed ? sm.list[tid + q * THREADS] : 0;
      more += __syncthreads_count(mine[q] > at_bound);
    }
    ties = more <= PLAIN;
    if (ties) {
      if (tid == 0) sm.n_list = 0;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < LIST / THREADS; ++q)
        if (mine[q] > at_bound) sm.list[atomicAdd(&sm.n_list, 1)] = mine[q];
      __syncthreads();
    }
  } else if (ties) {
    // Ties, or masked logits where fewer than k groups have others: only what is
    // above the bound is worth listing.
    __syncthreads();
    if (tid == 0) sm.n_list = sm.n_listed = 0;
    __syncthreads();
    if (tmax > bound) sm.listed[atomicAdd(&sm.n_listed, 1)] = static_cast<unsigned char>(tid);
    __syncthreads();
    collect(true);
  }
  if (!ties) {
    rank_keys(sm.list, listed, keep);
    __syncthreads();
    return;
  }
  if (sm.n_list <= LIST) {
    int found = sm.n_list;
    rank_keys(sm.list, found, keep);
    // then the first logits at the bound, in token order
    for (int i0 = 0; i0 < n && found < k; i0 += THREADS) {
      const bool hit = i0 + tid < n && to_float(x[i0 + tid]) == bound;
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      if ((tid & 31) == 0) sm.scan[tid >> 5] = __popc(hits);
      __syncthreads();
      int at = found + __popc(hits & ((1u << (tid & 31)) - 1u));
      for (int w = 0; w < WARPS; ++w) {
        if (w < (tid >> 5)) at += sm.scan[w];
        found += sm.scan[w];
      }
      if (hit && at < k) sm.best[at] = make_key(bound, first + i0 + tid);
      __syncthreads();
    }
  } else {
    unsigned long long below = ~0ull;
    for (int r = 0; r < k; ++r) {
      unsigned long long mine = 0;
      for (int i = tid; i < n; i += THREADS) {
        const float f = to_float(x[i]);
        if (!(f >= bound)) continue;
        const unsigned long long key = make_key(f, first + i);
        if (key < below && key > mine) mine = key;
      }
      below = block_max(sm, mine);
      if (tid == 0) sm.best[r] = below;
      if (!below) break;
    }
  }
  __syncthreads();
}

// Where the partial results of piece p of the row that begins in CTA f are: a
// CTA's first slot is for the piece it begins with, so p = 0 is in the second
// one if the row begins inside the share (odd).
__device__ __forceinline__ size_t piece_slot(int f, int p, int odd) {
  return 2 * static_cast<size_t>(f + p) + (p == 0 ? odd : 0);
}

// sm.best = the k largest keys of a row's pieces, each piece's in order at its slot of ws.
// Both are calls, so that the registers they need are not taken from the loop over the logits.
__device__ __noinline__ void join_tops(int pieces, int k, const unsigned long long* ws, int f, int odd) {
  Smem& sm = smem();
  auto keys = [&](int p) { return ws + piece_slot(f, p, odd) * MAX_K; };
  // Only keys not below the k-th largest of the pieces' largest can be among the
  // k largest, and of the piece with the h-th of those only the first k - h: at
  // most k (k + 1) / 2 in all, usually fewer than 2 k.
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int AHEAD = 4;
  unsigned long long ahead[AHEAD];  // a lane's key of the first pieces, while the heads are ranked
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    const int p = warp + q * WARPS;
    ahead[q] = p < pieces && lane < k ? __ldcg(keys(p) + lane) : 0;
  }
  for (int p = tid; p < pieces; p += THREADS) sm.heads[p] = __ldcg(keys(p));
  if (tid < MAX_K) sm.best[tid] = 0;
  if (tid == 0) {
    sm.n_list = 0;
    sm.key = 1;
  }
  __syncthreads();
  rank_keys(sm.heads, pieces, [&](int p, int rank) {
    sm.head_rank[p] = static_cast<unsigned char>(min(rank, 255));
    if (rank == k - 1) sm.key = max(sm.heads[p], 1ull);
  });
  __syncthreads();
  const unsigned long long least = sm.key;
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    const int p = warp + q * WARPS;
    if (ahead[q] >= least && lane + sm.head_rank[p] < k) sm.list[atomicAdd(&sm.n_list, 1)] = ahead[q];
  }
  for (int p = warp + AHEAD * WARPS; p < pieces; p += WARPS) {
    if (lane + sm.head_rank[p] >= k) continue;
    const unsigned long long key = __ldcg(keys(p) + lane);
    if (key >= least) sm.list[atomicAdd(&sm.n_list, 1)] = key;
  }
  __syncthreads();
  rank_keys(sm.list, sm.n_list, [&](int i, int rank) {
    if (rank < k) sm.best[rank] = sm.list[i];
  });
}

__device__ __forceinline__ int add_acq_rel(int* p, int v) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// A CTA's pieces: the part of each row in its share.
template <class T>
struct Piece {
  static constexpr int N = Vec<T>::N;
  long long at;
  const T* x;
  int row, c0, n, head, vecs;  // [head logits up to a 16-byte boundary | vectors | tail logits]
  __device__ __forceinline__ Piece(const Params& a, long long from, long long end) : at(from) {
    row = static_cast<int>(at / a.pitch);
    c0 = static_cast<int>(at - row * a.pitch);
    n = static_cast<int>(min(static_cast<long long>(a.V - c0), end - at));
    x = reinterpret_cast<const T*>(a.logits) + row * a.ld + c0;
    head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    vecs = (n - head) / N;
  }
};

template <class T>
__device__ __forceinline__ void logprobs_body(const Params& a) {
  Smem& sm = smem();
  pdl_entry();
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, k = a.k;
  const long long all = a.T * a.pitch;
  const long long begin = min(blockIdx.x * a.share, all), end = min(begin + a.share, all);
  for (long long at = begin; at < end;) {
    const Piece<T> pc(a, at, end);
    if (pc.n <= 0) break;  // a padded row's end
    // The given token's logit: read here, its way is long and the row's is longer.
    int id = -1;
    float chosen = 0.f;
    if (tid == 0 && a.logprobs) {
      id = a.ids[pc.row];
      if (id >= 0 && id < a.V) chosen = to_float(reinterpret_cast<const T*>(a.logits)[pc.row * a.ld + id]);
    }
    const int row = pc.row, c0 = pc.c0, n = pc.n, head = pc.head, vecs = pc.vecs, tail = head + vecs * N;
    const T* x = pc.x;
    Sums s;
    s.clear();
    float tmax = -INFINITY;
    auto edge = [&](float f) {
      if (f > s.ref) s.move(f);
      s.add(f);
      tmax = fmaxf(tmax, f);
    };
    if (tid < head) edge(to_float(x[tid]));
    if (tid < n - tail) edge(to_float(x[tail + tid]));
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    constexpr int STRIDE = U * THREADS;
    auto fetch = [&](int c) {  // chunk c of this thread's vectors (none behind the end) into its slot
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int j = c * STRIDE + q * THREADS + tid;
        if (j < vecs) copy16(&sm.ring[c % SLOTS][q][tid], v + j);
      }
      copy_commit();
    };
    auto sum = [&](const uint4 (&raw)[U], int count) {
      const float mx = Vec<T>::max_of(raw);
      tmax = fmaxf(tmax, mx);
      if (mx > s.ref) s.move(mx);
      // (Sums of their own: a term far below Z is not lost one by one in rounding Z.)
      float2 z2 = make_float2(0.f, 0.f), u2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int q = 0; q < U; ++q) {
        if (q >= count) break;
        float f[N];
        Vec<T>::unpack(raw[q], f);
#pragma unroll
        for (int e = 0; e < N; e += 4) s.add4({f[e], f[e + 1], f[e + 2], f[e + 3]}, z2, u2);
      }
      const float u = u2.x + u2.y;
      if (u == u) {
        s.z += z2.x + z2.y;
        s.u += u;
        return;
      }
#pragma unroll 1
      for (int q = 0; q < count; ++q) {  // masked logits (or NaN) among them: one by one
        float f[N];
        uint4 w = raw[0];
#pragma unroll
        for (int i = 1; i < U; ++i) w = q == i ? raw[i] : w;
        Vec<T>::unpack(w, f);
#pragma unroll
        for (int e = 0; e < N; ++e) s.add(f[e]);
      }
    };
#pragma unroll
    for (int c = 0; c < SLOTS - 1; ++c) fetch(c);
    const int whole = vecs / STRIDE;
    uint4 raw[U];
#pragma unroll 1
    for (int c = 0; c < whole; ++c) {
      copy_wait<SLOTS - 2>();
#pragma unroll
      for (int q = 0; q < U; ++q) raw[q] = sm.ring[c % SLOTS][q][tid];
      fetch(c + SLOTS - 1);  // into the slot of chunk c - 1, whose logits are in the sums
      sum(raw, U);
    }
    copy_wait<0>();
    if (const int left = vecs - whole * STRIDE - tid; left > 0) {
      const int count = (left + THREADS - 1) / THREADS;
#pragma unroll
      for (int q = 0; q < U; ++q) raw[q] = sm.ring[whole % SLOTS][q < count ? q : 0][tid];
      sum(raw, count);
    }
    // ---- the block's sums, and its k largest ----
    s = join_warp(s);
    if ((tid & 31) == 0) sm.sums[tid >> 5] = s;
    if (k > 0) piece_top<T>(x, n, head, vecs, c0, tmax, k);
    else __syncthreads();
    auto block_sums = [&]() {  // warp 0, after a barrier
      s.clear();
      if (tid < WARPS) s = sm.sums[tid];
      s = join_warp(s);
    };

    // ---- a row cut into pieces: CTAs f .. f + pieces - 1 hold them ----
    const long long row0 = at - c0;
    const int f = static_cast<int>(row0 / a.share);
    const int pieces = static_cast<int>((row0 + a.V - 1) / a.share) - f + 1;
    bool finish = true;
    if (pieces > 1) {
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (at == begin ? 0 : 1);
      if (tid < k) __stcg(a.ws_keys + slot * MAX_K + tid, sm.best[tid]);
      if (tid < 32) {
        block_sums();
        if (tid == 0) __stcg(reinterpret_cast<float4*>(a.ws_sums) + slot, make_float4(s.ref, s.z, s.u, 0.f));
      }
      __syncthreads();
      if (tid == 0) {
        // releases the block's writes (ordered before it by the barrier), acquires the other pieces'
        const int done = add_acq_rel(a.tickets + f, 1) + 1;
        sm.last = done == pieces;
        if (done == pieces) a.tickets[f] = 0;
      }
      __syncthreads();
      finish = sm.last;
      if (finish) {
        const int odd = row0 % a.share ? 1 : 0;  // the first piece begins inside its CTA's share
        s.clear();
        for (int p = tid; p < pieces; p += THREADS) {
          const float4 o = __ldcg(reinterpret_cast<const float4*>(a.ws_sums) + piece_slot(f, p, odd));
          Sums part;
          part.ref = o.x;
          part.z = o.y;
          part.u = o.z;
          s.join(part);
        }
        if (k > 0) join_tops(pieces, k, a.ws_keys, f, odd);
        s = join_warp(s);
        if ((tid & 31) == 0) sm.sums[tid >> 5] = s;
        __syncthreads();
      }
    }
    if (finish && tid < 32) {
      block_sums();
      // In 64 bits: next to a certain token it is the small difference that counts.
      const double lz = s.z > 0.f ? log(static_cast<double>(s.z)) : static_cast<double>(NAN);
      auto logprob = [&](float x) {
        return static_cast<float>(static_cast<double>(x) - static_cast<double>(s.ref) - lz);
      };
      if (tid == 0 && a.logprobs) {
        if (id >= a.V) set_status(FB_KERR_BAD_ARG);
        a.logprobs[row] = id < 0 ? 0.f : id < a.V ? logprob(chosen) : NAN;  // a negative id: no token
      }
      if (tid == 31 && a.entropy)
        a.entropy[row] = static_cast<float>(lz - LN2 * static_cast<double>(s.u) / static_cast<double>(s.z));
      if (tid < k) {
        const unsigned long long key = sm.best[tid];
        a.top_ids[static_cast<size_t>(row) * k + tid] = key ? key_token(key) : -1;
        a.top_logprobs[static_cast<size_t>(row) * k + tid] = key ? logprob(key_value(key)) : NAN;
      }
    }
    __syncthreads();
    at += n;
  }
}

}  // namespace

// Row r at logits + r * ld. ids, logprobs / entropy / top_* may be null (then
// not read / written; k = 0 with null top_*). top_* are [T, k].
#define FB_LOGPROBS(NAME, TYPE)                                                                                    \
  extern "C" __global__ void __launch_bounds__(THREADS, 3) fb_logprobs_##NAME(                                     \
      const TYPE* logits, long long ld, const int* ids, float* logprobs, float* entropy, float* top_logprobs,      \
      int* top_ids, float* ws_sums, unsigned long long* ws_keys, int* tickets, long long share, long long pitch, \
      int T, int V, int k) {                                                                                                     \
    const Params a{logits,  ld,      ids,   logprobs, entropy, top_logprobs, top_ids,                              \
                   ws_sums, ws_keys, tickets, share, pitch,  T,      V,            k};                                   \
    logprobs_body<TYPE>(a);                                                                                        \
  }
FB_LOGPROBS(bf16, bf16)
FB_LOGPROBS(f16, __half)
FB_LOGPROBS(f32, float)
