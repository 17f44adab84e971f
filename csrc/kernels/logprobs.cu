// Log probability of a given token, entropy and the k most probable tokens of
// each row of logits [T, V] (bf16, fp16 or fp32), in one pass over the logits.
//
// With y = (x - max) log2(e), Z = sum 2^y, U = sum 2^y y:
//   log p(t) = x_t - max - ln Z        H = ln Z - U ln 2 / Z
// (both terms of H are >= 0, so nothing cancels). Each thread keeps its own
// running max and rescales (Z, U) when it moves, once per 64 bytes at most; Z
// and U are fp32 sums of at most a few hundred terms each, joined as a tree.
//
// The k largest (ties: lowest token) come from the same pass: each thread also
// knows the max of what it has read, and the k-th largest of the block's 256
// maxima bounds the k-th largest logit from below. Only threads whose max
// reaches that bound - k of them, but for ties - read their logits again (from
// L2) and list what reaches it; the list, rarely longer than 2 k, is ranked by
// counting. Two ways out keep that exact for any input: more equal logits at
// the bound than the list holds are taken in token order, 256 at a time until
// enough are found (a constant row ends in its first step); more logits above
// the bound than the list holds (one thread's share holds many of the largest)
// are found by k passes.
//
// The kernel is bound by reading the logits. The flat sequence of all logits
// is cut into one equal share per CTA, whatever T and V are; a row that a cut
// falls into is joined by the CTA that finishes its last piece, through a
// workspace of two pieces per CTA and one ticket per cut (zero before and
// after every launch). The join is in piece order, so results do not depend
// on which CTA comes last.
#include <cuda_fp16.h>

#include "fb_common.cuh"

FB_DEFINE_STATUS

using namespace fbk;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_K = 32;
constexpr int LIST = 512;    // logits above the bound, and as many at it
constexpr int MAX_PIECES = 1024;
constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453094;

// Order of candidates: larger logit first, then the lower token. 0 = none.
__device__ __forceinline__ unsigned long long make_key(float x, int token) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 -> +0: equal logits tie
  const unsigned up = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(up) << 32 | static_cast<unsigned>(~token);
}
__device__ __forceinline__ int key_token(unsigned long long k) { return static_cast<int>(~static_cast<unsigned>(k)); }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned up = static_cast<unsigned>(k >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

// The logits of one 16-byte vector.
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
  __device__ __forceinline__ void join(Sums o) {
    const float to = fmaxf(ref, o.ref);
    move(to);
    o.move(to);
    z += o.z;
    u += o.u;
  }
  __device__ __forceinline__ void join_warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Sums other;
      other.ref = __shfl_xor_sync(0xffffffffu, ref, o);
      other.z = __shfl_xor_sync(0xffffffffu, z, o);
      other.u = __shfl_xor_sync(0xffffffffu, u, o);
      join(other);
    }
  }
};

struct Smem {
  float tmax[THREADS];
  Sums sums[WARPS];
  unsigned long long above[LIST], equal[LIST], best[MAX_K];
  unsigned long long cand[MAX_K * (MAX_K + 1) / 2];
  unsigned long long key;
  float bound;
  int n_above, n_equal, n_cand, last;
  int scan[WARPS];
  unsigned char head_rank[MAX_PIECES];
};

struct Params {
  const void* logits;
  long long ld;
  const int* ids;
  float *logprobs, *entropy, *top_logprobs;
  int* top_ids;
  float* ws_sums;                 // [2 * gridDim][4]
  unsigned long long* ws_keys;    // [2 * gridDim][MAX_K]
  int* tickets;                   // [gridDim], zero between launches
  long long share;                // logits per CTA
  int T, V, k;
};

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

// best[0..k) = the k largest of `n` distinct keys at list(i), in order.
template <class List>
__device__ __forceinline__ void rank_keys(Smem& sm, int n, int k, List list) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long mine = list(i);
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list(j) > mine;
    if (rank < k) sm.best[rank] = mine;
  }
}

// sm.best[0..k) = the piece's k largest keys (0 where there are fewer), from
// logits x[0..n) that start at token `first`; tmax: the max of what this
// thread's part of the vectors (and its head and tail logit) holds.
template <class T>
__device__ __forceinline__ void piece_top(Smem& sm, const T* x, int n, int head, int vecs, int first, float tmax,
                                          int k) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x;
  sm.tmax[tid] = tmax;
  if (tid == 0) {
    sm.n_above = sm.n_equal = 0;
    sm.bound = -INFINITY;
  }
  if (tid < MAX_K) sm.best[tid] = 0;
  __syncthreads();
  {
    int more = 0, same = 0;
    const float4* all = reinterpret_cast<const float4*>(sm.tmax);
#pragma unroll 4
    for (int j = 0; j < THREADS / 4; ++j) {
      const float4 o = all[j];
      more += (o.x > tmax) + (o.y > tmax) + (o.z > tmax) + (o.w > tmax);
      same += (o.x == tmax) + (o.y == tmax) + (o.z == tmax) + (o.w == tmax);
    }
    if (more < k && more + same >= k) sm.bound = tmax;  // one value: every writer's is the same
  }
  __syncthreads();
  const float bound = sm.bound;
  auto look = [&](float f, int i) {
    if (f > bound) {
      const int at = atomicAdd(&sm.n_above, 1);
      if (at < LIST) sm.above[at] = make_key(f, first + i);
    } else if (f == bound) {
      const int at = atomicAdd(&sm.n_equal, 1);
      if (at < LIST) sm.equal[at] = make_key(f, first + i);
    }
  };
  if (tmax >= bound) {
    if (tid < head) look(to_float(x[tid]), tid);
    const int tail = head + vecs * N;
    if (tid < n - tail) look(to_float(x[tail + tid]), tail + tid);
    const uint4* v = reinterpret_cast<const uint4*>(x + head);
    for (int j = tid; j < vecs; j += THREADS) {
      float f[N];
      Vec<T>::unpack(__ldg(v + j), f);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (f[e] >= bound) look(f[e], head + j * N + e);
    }
  }
  __syncthreads();
  const int above = sm.n_above, equal = sm.n_equal;
  if (above <= LIST && equal <= LIST) {
    rank_keys(sm, above + equal, k,
              [&](int i) { return i < above ? sm.above[i] : sm.equal[i - above]; });
  } else if (above <= LIST) {
    rank_keys(sm, above, k, [&](int i) { return sm.above[i]; });
    int found = above;  // then the first logits at the bound, in token order
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

template <class T>
__device__ __forceinline__ void logprobs_body(const Params& a) {
  __shared__ __align__(16) Smem sm;
  pdl_entry();
  constexpr int N = Vec<T>::N, U = 4;  // U vectors per thread in flight
  const int tid = threadIdx.x, k = a.k;
  const long long all = static_cast<long long>(a.T) * a.V;
  const long long begin = min(blockIdx.x * a.share, all), end = min(begin + a.share, all);
  for (long long at = begin; at < end;) {
    const int row = static_cast<int>(at / a.V), c0 = static_cast<int>(at - static_cast<long long>(row) * a.V);
    const int n = static_cast<int>(min(static_cast<long long>(a.V - c0), end - at));
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld + c0;
    // [head logits up to a 16-byte boundary | vectors | tail logits]
    const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    const int vecs = (n - head) / N, tail = head + vecs * N;
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
    for (int j = tid; j < vecs; j += U * THREADS) {
      uint4 raw[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int i = j + q * THREADS;
        raw[q] = i < vecs ? __ldg(v + i) : raw[0];
      }
      float f[U][N];
      float mx = -INFINITY;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        Vec<T>::unpack(raw[q], f[q]);
#pragma unroll
        for (int e = 0; e < N; ++e) mx = fmaxf(mx, f[q][e]);
      }
      tmax = fmaxf(tmax, mx);
      if (mx > s.ref) s.move(mx);
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (j + q * THREADS < vecs) {
#pragma unroll
          for (int e = 0; e < N; ++e) s.add(f[q][e]);
        }
    }
    // ---- the block's sums, and its k largest ----
    s.join_warp();
    if ((tid & 31) == 0) sm.sums[tid >> 5] = s;
    __syncthreads();
    s = sm.sums[0];
    for (int w = 1; w < WARPS; ++w) s.join(sm.sums[w]);
    if (k > 0) piece_top<T>(sm, x, n, head, vecs, c0, tmax, k);

    // ---- a row cut into pieces: CTAs f .. f + pieces - 1 hold them ----
    const long long row0 = at - c0;
    const int f = static_cast<int>(row0 / a.share);
    const int pieces = static_cast<int>((row0 + a.V - 1) / a.share) - f + 1;
    bool finish = true;
    if (pieces > 1) {
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (at == begin ? 0 : 1);
      if (tid < k) __stcg(a.ws_keys + slot * MAX_K + tid, sm.best[tid]);
      if (tid == 0) __stcg(reinterpret_cast<float4*>(a.ws_sums) + slot, make_float4(s.ref, s.z, s.u, 0.f));
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        const int done = atomicAdd(a.tickets + f, 1) + 1;
        sm.last = done == pieces;
        if (done == pieces) a.tickets[f] = 0;
        sm.n_cand = 0;
        __threadfence();
      }
      __syncthreads();
      finish = sm.last;
      if (finish) {
        const int odd = row0 % a.share ? 1 : 0;  // the first piece begins inside its CTA's share
        auto slot_of = [&](int p) { return 2 * static_cast<size_t>(f + p) + (p == 0 ? odd : 0); };
        Sums part;
        s.clear();
        for (int p = tid; p < pieces; p += THREADS) {
          const float4 o = __ldcg(reinterpret_cast<const float4*>(a.ws_sums) + slot_of(p));
          part.ref = o.x;
          part.z = o.y;
          part.u = o.z;
          s.join(part);
        }
        s.join_warp();
        if ((tid & 31) == 0) sm.sums[tid >> 5] = s;
        // Of a list whose largest key ranks h-th among the lists' largest keys,
        // only the first k - h keys can be among the k largest.
        if (k > 0) {
          if (tid < MAX_K) sm.best[tid] = 0;
          for (int p = tid; p < pieces; p += THREADS) {
            const unsigned long long mine = __ldcg(a.ws_keys + slot_of(p) * MAX_K);
            int rank = 0;
            for (int o = 0; o < pieces; ++o) rank += __ldcg(a.ws_keys + slot_of(o) * MAX_K) > mine;
            sm.head_rank[p] = static_cast<unsigned char>(min(rank, 255));
          }
          __syncthreads();
          for (int i = tid; i < pieces * k; i += THREADS) {
            const int p = i / k, e = i - p * k;
            if (e + sm.head_rank[p] >= k) continue;
            const unsigned long long key = __ldcg(a.ws_keys + slot_of(p) * MAX_K + e);
            if (key) sm.cand[atomicAdd(&sm.n_cand, 1)] = key;
          }
          __syncthreads();
          rank_keys(sm, sm.n_cand, k, [&](int i) { return sm.cand[i]; });
        }
        __syncthreads();
        s = sm.sums[0];
        for (int w = 1; w < WARPS; ++w) s.join(sm.sums[w]);
      }
    }
    if (finish) {
      // In 64 bits: next to a certain token it is the small difference that counts.
      const double lz = s.z > 0.f ? log(static_cast<double>(s.z)) : static_cast<double>(NAN);
      auto logprob = [&](float x) {
        return static_cast<float>(static_cast<double>(x) - static_cast<double>(s.ref) - lz);
      };
      if (tid == 0 && a.logprobs) {
        const int id = a.ids[row];
        float lp = 0.f;  // a negative id: no token
        if (id >= a.V) {
          set_status(FB_KERR_BAD_ARG);
          lp = NAN;
        } else if (id >= 0) {
          lp = logprob(to_float(reinterpret_cast<const T*>(a.logits)[row * a.ld + id]));
        }
        a.logprobs[row] = lp;
      }
      if (tid == 32 && a.entropy)
        a.entropy[row] = static_cast<float>(lz - LN2 * static_cast<double>(s.u) / static_cast<double>(s.z));
      if (tid >= 64 && tid < 64 + k) {
        const unsigned long long key = sm.best[tid - 64];
        a.top_ids[static_cast<size_t>(row) * k + tid - 64] = key ? key_token(key) : -1;
        a.top_logprobs[static_cast<size_t>(row) * k + tid - 64] = key ? logprob(key_value(key)) : NAN;
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
  extern "C" __global__ void __launch_bounds__(THREADS, 4) fb_logprobs_##NAME(                                     \
      const TYPE* logits, long long ld, const int* ids, float* logprobs, float* entropy, float* top_logprobs,      \
      int* top_ids, float* ws_sums, unsigned long long* ws_keys, int* tickets, long long share, int T, int V,      \
      int k) {                                                                                                     \
    const Params a{logits,  ld,      ids,   logprobs, entropy, top_logprobs, top_ids,                              \
                   ws_sums, ws_keys, tickets, share,  T,       V,            k};                                   \
    logprobs_body<TYPE>(a);                                                                                        \
  }
FB_LOGPROBS(bf16, bf16)
FB_LOGPROBS(f16, __half)
FB_LOGPROBS(f32, float)
