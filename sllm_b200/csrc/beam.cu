// Beam search on the device: the best continuations of every search over its beams and the whole vocabulary, and what of them goes on or is finished.
// The reference decodes one sequence by sampling alone (runtime/sampler.py:36-88); it has no search.
//
// Candidates.  With m_b the largest logit of beam b, the continuation of beam b by token v scores
//   s(b, v) = score_b + ((x_bv - m_b) - log sum_u exp(x_bu - m_b)),
// and the `keep` largest of a search are wanted, in order: s descending, then the beam, then the logit descending, then the token.  Within a beam s grows with the
// logit, so a beam's own best are those of the largest logits, and no candidate of the search lies outside the `keep` best of its beam:
//   beam_rows_kernel    a part of a row a block: the part's maximum, its sum of exponentials and its `keep` largest logits, from one pass over the logits;
//   beam_merge_kernel   a block a search, a warp a beam: the beam's parts joined, then the beams.
// Exponentials and a batch's sum of them (16 terms) are float32; the sums over batches, threads and parts, the logarithm and s are of 48 bits and more, because continuations of different beams
// are compared with each other (those of one beam by their logits alone).  Where two beams' lie closer than those float32 steps can tell, their sums are made again in float64 (see `beam_close`).
// s is rounded to float32 once, when it is stored.
// Measured, both kernels, us (reading the logits at the measured copy rate): 4 rows of 151,936 float32 10.3 (0.4), 35 of 32,001 13.3 (0.7), 512 of 152,064 float32 63 (47.6) and
// bfloat16 53.6 (23.8).  Few rows are bound by the chain load, first bound, list, sums, join, about a microsecond each; many by HBM through the long runs, and by the same chain, which their blocks go
// through side by side.
#include <float.h>

#include "common.cuh"

namespace sllm {

constexpr int BEAM_THREADS = 256, BEAM_KEEP = 128, BEAM_MAX = 32;
constexpr int BEAM_VALUES = 16;                                 // logits of a thread and batch
constexpr uint32_t BEAM_MINUS_INFINITY = 0x007fffffu;           // the key of minus infinity: what is not above it offers nothing

// Keys: the logit's bits so that unsigned order is float order, then the token turned around, so that of equal logits the first is the largest key.  0: no key.
__device__ __forceinline__ uint32_t beam_order(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float beam_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ unsigned long long beam_key(float f, int token) { return (unsigned long long)beam_order(f) << 32 | ~(uint32_t)token; }
__device__ __forceinline__ unsigned long long order_double(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double double_of(unsigned long long k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (unsigned long long)hi << 32 | lo;
}

// log2 e as the kernels multiply with it: 2^(x BEAM_LOG2E) is e^x but for 1.34e-8 |x| of it, and for 1.34e-8 |x - max| once the maximum is taken out in the same way.
constexpr float BEAM_LOG2E = 1.4426950408889634f;

// A sum of exponentials, Sum 2^(x BEAM_LOG2E), is held over 2^r.  r goes by the largest logit m alone: a whole number at m BEAM_LOG2E or just above it where float32 holds one to the unit
// with room to spare (`beam_whole`; not a number elsewhere: infinite m, rows of 10^6 and more), so that sums of other maxima are brought to it by a change of exponent, exactly; m BEAM_LOG2E itself elsewhere.
__device__ __forceinline__ float beam_whole(float m) {
  const float to = m * BEAM_LOG2E;
  return fabsf(to) < 4194304.f ? ceilf(to) : __uint_as_float(0x7fffffffu);
}
__device__ __forceinline__ double beam_reference(float m, float whole) { return whole == whole ? (double)whole : (double)m * (double)BEAM_LOG2E; }
// 2^(r of m - r of top), m <= top; whole: theirs (minus infinity: nothing summed yet)
__device__ __forceinline__ double beam_moved(float m, float whole, float top, float top_whole) {
  if (whole <= top_whole) {
    const float d = whole - top_whole;
    return d > -1022.f ? __hiloint2double((1023 + (int)d) << 20, 0) : 0.0;
  }
  return exp2(beam_reference(m, whole) - beam_reference(top, top_whole));
}

// a part of a row: its sum of exponentials, and its largest logit
struct BeamPart {
  double sum;
  float max;
};

// 16 bytes of logits: how many, their values, their largest (a number where there is one), one that is missing, one alone
template <typename T> struct BeamLoad;
template <> struct BeamLoad<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& raw, float* x) {
    x[0] = __uint_as_float(raw.x);
    x[1] = __uint_as_float(raw.y);
    x[2] = __uint_as_float(raw.z);
    x[3] = __uint_as_float(raw.w);
  }
  static __device__ __forceinline__ float largest(const uint4& raw) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
  }
  template <class F> static __device__ __forceinline__ uint4 gather(const float* p, F there) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = there(i) ? __float_as_uint(p[i]) : 0xff800000u;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct BeamLoad<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& raw, float* x) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float largest(const uint4& raw) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  template <class F> static __device__ __forceinline__ uint4 gather(const __nv_bfloat16* p, F there) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (there(2 * i) ? (uint32_t)__bfloat16_as_ushort(p[2 * i]) : 0xff80u) | (there(2 * i + 1) ? (uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) : 0xff80u) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// LIST: keys that may belong to the best, what a batch can add (see beam_rows_kernel) beside the `keep` already held at the least; OTHER: the other half of a filter's ping-pong, what
// a pass over a full list can leave.
constexpr int BEAM_LIST = BEAM_KEEP * BEAM_VALUES + BEAM_KEEP, BEAM_OTHER = BEAM_LIST / 2 + BEAM_KEEP;

constexpr int BEAM_SEEN = 256;                                  // threads' batches a warp can note in a run

struct BeamShared {
  unsigned long long list[BEAM_LIST], other[BEAM_OTHER];
  unsigned long long group[BEAM_THREADS];
  int seen[BEAM_THREADS / 32][BEAM_SEEN];
  unsigned long long bound;
  double red_s[BEAM_THREADS / 32];
  float red_m[BEAM_THREADS / 32];
  int n;
};

// The keep-th largest of the groups' largest keys, known to all threads: `keep` keys at least are no smaller.  0 where fewer than `keep` groups have a key.
// `mine`: this thread's largest; a group is 1 << log2_lanes threads side by side.
__device__ unsigned long long beam_group_bound(unsigned long long mine, int log2_lanes, int keep, BeamShared& sh) {
  for (int o = 1; o < (1 << log2_lanes); o <<= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
    mine = mine > other ? mine : other;
  }
  const int groups = BEAM_THREADS >> log2_lanes;
  if ((threadIdx.x & ((1 << log2_lanes) - 1)) == 0) sh.group[threadIdx.x >> log2_lanes] = mine;
  if (threadIdx.x == 0) sh.bound = 0;
  __syncthreads();
  // a group's threads share the comparisons of its rank
  {
    const int lanes = 1 << log2_lanes, mine_at = threadIdx.x >> log2_lanes;
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x & (lanes - 1); j < groups; j += lanes) rank += sh.group[j] > mine || (sh.group[j] == mine && j < mine_at);
    for (int o = 1; o < lanes; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (rank == keep - 1) sh.bound = mine;
  }
  __syncthreads();
  const unsigned long long b = sh.bound;
  __syncthreads();
  return b;
}

// The keys sh.list[0, sh.n) become their `keep` largest, sorted; returns how many there are.  Filters by the groups' bound until no more than the threads are left (each pass
// leaves at most (keep - 1) groups' keys and one, about half of them), then every key finds its place.
__device__ int beam_compact(int keep, int log2_lanes, BeamShared& sh) {
  __syncthreads();
  int n = sh.n;
  unsigned long long *from = sh.list, *to = sh.other;
  while (n > BEAM_THREADS) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS) best = best > from[i] ? best : from[i];
    const unsigned long long b = beam_group_bound(best, log2_lanes, keep, sh);
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += BEAM_THREADS)
      if (from[i] >= b) to[atomicAdd(&sh.n, 1)] = from[i];
    __syncthreads();
    n = sh.n;
    unsigned long long* t = from;
    from = to;
    to = t;
    __syncthreads();
  }
  unsigned long long me = 0;
  int rank = 0;
  if ((int)threadIdx.x < n) {
    me = from[threadIdx.x];
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += from[j] > me;
  }
  __syncthreads();
  if ((int)threadIdx.x < n && rank < keep) sh.list[rank] = me;
  n = n < keep ? n : keep;
  if (threadIdx.x == 0) sh.n = n;
  __syncthreads();
  return n;
}

// 2^t, within 2^-22 of it (the hardware's; denormal results are zero)
__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// two float32 operations an instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r)) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
  return r;
}

// One part of one row: blockIdx.x = row * splits + part.  What bounds it: reading the logits once.  A batch is BEAM_VALUES logits a thread in 16-byte loads, all in flight
// together, the next batch's under the arithmetic of this one.
// An exponential is 2^(x log2 e - c) in one rounding of the exponent, c a whole number; what it is off by: `beam_close`.
// Of a batch only keys that reach the bound, a key that `keep` others are known to reach, can be among the best.  The first batch's bound comes from the threads' largest.  A run of
// 6, then 36, ... batches is read without a barrier; a thread whose largest logit of a batch reaches the bound notes the batch (a vote of its warp, no atomics), and behind the run the noted
// ones are read again (from L1 or L2), their keys join the list, and the list, cut to its `keep` largest, gives the next bound: of logits in no particular order five or six
// times `keep` a run.  Where a run has more than the lists hold (logits that rise through the row, or are equal), its batches are read again one by one, each with a bound of its own.
// (512 rows of 152,064 bfloat16 logits, keep 16, us: reading them and their maxima 30, with the exponentials 37, with the list 48; 50 where every thread put its
// keys into the list at once.)
template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 1024 / BEAM_THREADS) beam_rows_kernel(const T* logits, int V, int keep, int log2_lanes, int splits, int part_vecs, BeamPart* parts, unsigned long long* keys) {
  constexpr int N = BeamLoad<T>::N, LOADS = BEAM_VALUES / N, BATCH = LOADS * BEAM_THREADS;
  extern __shared__ __align__(16) unsigned char beam_smem[];
  BeamShared& sh = *reinterpret_cast<BeamShared*>(beam_smem);
  const int row = blockIdx.x / splits, part = blockIdx.x - row * splits;
  const T* x_row = logits + (size_t)row * V;
  // Pieces of 16 bytes of tokens.  Which thread takes which tokens goes by their numbers and not by where the row lies, so that equal rows give equal sums; a row that does not begin
  // on 16 bytes is read an element at a time (from L1 but for the first of a piece; 512 rows of 152,063: float32 76 us for 62, bfloat16 83 for 53).
  const int pieces = (V + N - 1) / N;
  const int v0 = part * part_vecs, v1 = min(v0 + part_vecs, pieces);
  const int whole = (reinterpret_cast<uintptr_t>(x_row) & 15) == 0 ? min(v1, V / N) : 0;          // pieces that are read as they lie
  if (threadIdx.x == 0) sh.n = 0;
  unsigned long long bound = (unsigned long long)(BEAM_MINUS_INFINITY + 1) << 32;
  float bound_logit = beam_value(BEAM_MINUS_INFINITY + 1);
  float m = -INFINITY, s = 0.f, s_low = 0.f;
  // the pieces of one thread's batch: first, first + BEAM_THREADS, ...
  auto fetch = [&](int first, bool all, uint4* raw) {
    if (all) {
      const uint4* p = reinterpret_cast<const uint4*>(x_row) + first;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) raw[u] = p[u * BEAM_THREADS];
    } else {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int v = first + u * BEAM_THREADS, token = v * N;
        if (v < whole) raw[u] = *reinterpret_cast<const uint4*>(x_row + token);
        else raw[u] = BeamLoad<T>::gather(x_row + token, [&](int i) { return v < v1 && token + i < V; });
      }
    }
  };
  // values and the largest of them (a number where there is one)
  auto open = [&](const uint4* raw, float* x) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      BeamLoad<T>::unpack(raw[u], x + u * N);
      top = fmaxf(top, BeamLoad<T>::largest(raw[u]));
    }
    return top;
  };
  // s + s_low: the sum of 2^(x log2 e - c), c the whole number of m; every batch's own sum is float32, what adding it to s rounds away goes into s_low (one float64 in their place: 512 rows
  // of bfloat16 55.3 us for 54.5).  Where m has no such number c is none either and every batch goes the long way.
  float c = -INFINITY;
  auto split = [&](double sum) {
    s = (float)sum;
    s_low = (float)(sum - (double)s);
  };
  auto add_up = [&](const float* x, float top) {
    if (top > m) {
      const float to = beam_whole(top);
      if (c <= to) {
        const float d = c - to, by = d > -126.f ? __uint_as_float((uint32_t)(127 + (int)d) << 23) : 0.f;
        s *= by;
        s_low *= by;
      } else {
        split(((double)s + (double)s_low) * beam_moved(m, c, top, to));
      }
      m = top;
      c = to;
    }
    if (m > -INFINITY) {
      const float2 by = make_float2(-c, -c), factor = make_float2(BEAM_LOG2E, BEAM_LOG2E);
      float2 p[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int i = 0; i < BEAM_VALUES; i += 2) {
        const float2 t = fma2(make_float2(x[i], x[i + 1]), factor, by);
        p[(i >> 1) & 1] = add2(p[(i >> 1) & 1], make_float2(exp2_fast(t.x), exp2_fast(t.y)));
      }
      const float add = (p[0].x + p[0].y) + (p[1].x + p[1].y);
      // (asked of the bits: the compiler takes what the exponential's asm gives for numbers and leaves `add != add` out)
      if ((__float_as_uint(add) & 0x7fffffffu) >= 0x7f800000u) {
        // a logit that is none, which counts for nothing, or an m without a whole number: differences from it are exact where they count (those of an infinite m: all of the mass lies on the infinities)
        const bool whole = (__float_as_uint(c) & 0x7fffffffu) < 0x7f800000u;
        double sum = (double)s + (double)s_low;
#pragma unroll
        for (int i = 0; i < BEAM_VALUES; ++i) {
          if (whole) sum += x[i] <= m ? (double)exp2_fast(fmaf(x[i], BEAM_LOG2E, -c)) : 0.0;
          else if (x[i] == m) sum += 1.0;
          else if (x[i] < m && m < INFINITY) sum += (double)exp2_fast((x[i] - m) * BEAM_LOG2E);
        }
        split(sum);
      } else {
        const float sum = s + add, z = sum - s;
        s_low += (s - (sum - z)) + (add - z);
        s = sum;
      }
    }
  };
  // a logit's key, 0 where it offers nothing; minus zero is zero
  auto key_of = [&](float f, int first, int i) {
    f += 0.0f;
    return f > -INFINITY ? beam_key(f, (first + (i / N) * BEAM_THREADS) * N + i % N) : 0ull;
  };
  auto append = [&](const float* x, float top, int first) {
    if (top >= bound_logit) {
#pragma unroll
      for (int i = 0; i < BEAM_VALUES; ++i)
        if (x[i] >= bound_logit) {
          const unsigned long long k = key_of(x[i], first, i);
          if (k >= bound) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < BEAM_LIST) sh.list[at] = k;
          }
        }
    }
  };
  auto raise = [&](unsigned long long b) {
    bound = bound > b ? bound : b;
    bound_logit = beam_value((uint32_t)(bound >> 32));
  };
  int held = 0;                                    // keys in the list behind a cut
  auto cut = [&]() {
    held = beam_compact(keep, log2_lanes, sh);
    if (held == keep) raise(sh.list[keep - 1]);
    __syncthreads();
  };
  // The bound of one batch: the keep-th largest of the groups' largest keys.  The keys that reach it are those of fewer than `keep` groups and one more.
  auto bound_of = [&](const float* x, float top, int first) {
    int at = 0;
#pragma unroll
    for (int i = BEAM_VALUES - 1; i >= 0; --i) at = x[i] == top ? i : at;          // the first of the largest
    raise(beam_group_bound(key_of(top, first, at), log2_lanes, keep, sh));
  };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4 next[LOADS];
  float x[BEAM_VALUES];
  __syncthreads();
  pdl_wait();
  fetch(v0 + threadIdx.x, v0 + BATCH <= whole, next);
  for (int vb = v0, batches = 6; vb < v1; batches = min(6 * batches, 1 << 20)) {
    const int run = vb, end = min(vb + batches * BATCH, v1);
    int noted = 0;
    for (; vb < end; vb += BATCH) {
      const float top = open(next, x);
      if (vb + BATCH < v1) fetch(vb + BATCH + threadIdx.x, vb + 2 * BATCH <= whole, next);
      add_up(x, top);
      if (vb == v0) bound_of(x, top, vb + threadIdx.x);
      const unsigned votes = __ballot_sync(0xffffffffu, top >= bound_logit);
      if (votes) {
        const int at = noted + __popc(votes & ((1u << lane) - 1));
        if (top >= bound_logit && at < BEAM_SEEN) sh.seen[warp][at] = vb + threadIdx.x;
        noted += __popc(votes);
      }
    }
    __syncwarp();
    uint4 raw[LOADS];
    if (noted <= BEAM_SEEN) {
      for (int j = lane; j < noted; j += 32) {
        const int first = sh.seen[warp][j];
        fetch(first, false, raw);
        const float top = open(raw, x);
        append(x, top, first);
      }
    } else if (lane == 0) {
      atomicAdd(&sh.n, BEAM_LIST + 1);
    }
    __syncthreads();
    if (sh.n <= BEAM_LIST) {
      cut();
    } else {
      __syncthreads();
      if (threadIdx.x == 0) sh.n = held;
      for (int again = run; again < end; again += BATCH) {
        fetch(again + threadIdx.x, false, raw);
        const float top = open(raw, x);
        bound_of(x, top, again + threadIdx.x);     // (the list holds `keep` keys at most: it has room)
        append(x, top, again + threadIdx.x);
        cut();
      }
    }
  }
  pdl_launch_dependents();
  // the part's maximum and sum: the threads' sums, brought to its maximum
  const float warp_top = warp_max(m);
  if (lane == 0) sh.red_m[warp] = warp_top;
  __syncthreads();
  const float all = warp_max(lane < BEAM_THREADS / 32 ? sh.red_m[lane] : -INFINITY);
  double sum = (double)s + (double)s_low;
  if (m != all) sum = m > -INFINITY && all < INFINITY ? sum * beam_moved(m, c, all, beam_whole(all)) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.red_s[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < BEAM_THREADS / 32; ++w) sum += sh.red_s[w];
    parts[blockIdx.x] = BeamPart{sum, all};
  }
  for (int i = threadIdx.x; i < keep; i += BEAM_THREADS) keys[(size_t)blockIdx.x * keep + i] = i < held ? sh.list[i] : 0ull;
}

// A search: warp b joins the parts of beam b's row, then the first warp joins the beams.  Every step of a join takes the largest of the lists' heads, one a lane; the key behind a head
// is loaded before the head goes.  About 0.15 us a step of a chain that nothing hides: 5 us for 16 kept, 20 for 64.
struct BeamHead {
  const unsigned long long* list;
  int at, n;
  unsigned long long head, behind;
  __device__ __forceinline__ BeamHead(const unsigned long long* l, int length) : list(l), at(2), n(length) {
    head = n > 0 ? list[0] : 0ull;
    behind = n > 1 ? list[1] : 0ull;
  }
  __device__ __forceinline__ void pop() {
    head = behind;
    behind = at < n ? list[at] : 0ull;
    ++at;
  }
};

// Neighbours in the order that are two beams' and lie closer than `close` are told apart by the beams' sums in 64 bits throughout, which the block makes from the rows then.  `close` is twice what the
// logarithm of a sum of the rows' kernel may be off by, in units of u = 2^-24, with means under the softmax itself, under which |t| of 2^t is log2 V + 1 at the most:
//   the rounding of t = x log2 e - c         ln 2 (log2 V + 1)
//   log2 e's own                             0.23 ln V
//   the exponential (2^-22)                  4
//   the float32 sum of a batch, 5 additions  5
// together less than 0.86 log2 V + 9.8; the sums of batches, threads and parts change their reference exactly and lose nothing of that size.  (Of 152,064 logits: 24.9 u, 1.5e-6.)
// Of 400 calls of 64 searches of 8 beams over 152,064 normal logits ten made sums again, two of them each, which took them 150 us more.
static double beam_close(int V) { return 2.0 * (0.86 * log2((double)V) + 10.0) / 16777216.0; }

// e^d, d <= 0, but for some (1 + |d| / 8) 2^-51 of it (d below -690: e^-690): d = n ln 2 / 64 + r, the Taylor polynomial of degree 5 of r (|r| <= ln 2 / 128 leaves 4e-17), 2^((n mod 64) / 64) from a table and the
// rest of n into the exponent (Tang's table-driven method).  A sum of a row is bound by float64 instructions, half as many as without a table; and no branch, so that a thread's run side by side.
constexpr int BEAM_POWERS = 64;
__device__ __forceinline__ double exp_double(double d, const double* powers) {
  const double e = fmax(d, -690.0);
  const double shifted = fma(e, 64 / 0.69314718055994531, 6755399441055744.0);                // + 1.5 * 2^52: n in the low bits
  const double n = shifted - 6755399441055744.0;
  const double r = fma(n, -0.69314718055994531 / 64, e);
  const double r2 = r * r;
  const double tail = fma(fma(fma(r, 1.0 / 120, 1.0 / 24), r2, fma(r, 1.0 / 6, 0.5)), r2, r);      // e^r - 1
  const int k = __double2loint(shifted);
  const double p = powers[k & (BEAM_POWERS - 1)], v = fma(p, tail, p);
  return __hiloint2double(__double2hiint(v) + ((k >> 6) << 20), __double2loint(v));
}

// What a beam's scores are made of: s + (x - top), less the logarithm of its sum.
struct BeamRow {
  float score, top;
};
__device__ __forceinline__ double beam_score(const BeamRow& r, float x, double lse) { return (double)r.score + ((x == r.top ? 0.0 : (double)x - (double)r.top) - lse); }

// The beams in `close` of a search: their sums again, by the whole block, and their scores: 52 us a row of 152,064 that L2 holds.  (A function of its own, so that the join's instructions lie together;
// within the join it took 8 rows of 4 beams 0.1 us more that made no sum again.)
template <typename T>
__device__ __noinline__ void beam_sums_again(const T* logits, int V, int B, int keep, unsigned close, const BeamRow* rows, const float* best_logit, unsigned long long* merged) {
  __shared__ double red[BEAM_MAX], powers[BEAM_POWERS];
  const int width = blockDim.x;
  const T* search = logits + (size_t)blockIdx.x * B * V;
  // the rows from HBM into L2, all at once: what a block's own loads have in flight would take as long again
  for (unsigned left = close; left; left &= left - 1) {
    const char* x_row = reinterpret_cast<const char*>(search + (size_t)(__ffs(left) - 1) * V);
    for (size_t at = (size_t)threadIdx.x * 128; at < V * sizeof(T); at += (size_t)width * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(x_row + at));
  }
  for (int i = threadIdx.x; i < BEAM_POWERS; i += width) powers[i] = exp2((double)i / BEAM_POWERS);
  __syncthreads();
  for (unsigned left = close; left; left &= left - 1) {
    const int c = __ffs(left) - 1;
    const BeamRow row = rows[c];
    if (!(row.top < INFINITY)) continue;            // (an infinite maximum: a count, which is exact)
    const T* x_row = search + (size_t)c * V;
    // eight logits of a thread a step, the next step's loaded under this one's exponentials
    const double top = row.top;
    double each[4] = {0.0, 0.0, 0.0, 0.0};
    float next[8];
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < 8; ++u) next[u] = i0 + u * width < V ? to_f32(x_row[i0 + u * width]) : -INFINITY;
    };
    load(threadIdx.x);
    for (int i0 = threadIdx.x; i0 < V; i0 += 8 * width) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = fmaxf(next[u], -INFINITY);                // (not a number: minus infinity)
      load(i0 + 8 * width);
#pragma unroll
      for (int u = 0; u < 8; ++u) each[u & 3] += exp_double((double)x[u] - top, powers);
    }
    double all = (each[0] + each[1]) + (each[2] + each[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = all;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < width / 32; ++w) total += red[w];
    const double exact = fmax(log(total), 0.0);
    for (int i = threadIdx.x; i < keep; i += width)
      if (merged[c * keep + i] != 0) merged[c * keep + i] = order_double(beam_score(row, best_logit[c * keep + i], exact));
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * BEAM_MAX) beam_merge_kernel(const T* logits, int V, const float* scores, const BeamPart* parts, const unsigned long long* keys, int B, int keep, int splits, double close_by,
                                  float* out_score, int* out_parent, int* out_token) {
  extern __shared__ __align__(16) unsigned char beam_smem[];
  unsigned long long* lists = reinterpret_cast<unsigned long long*>(beam_smem);        // [B][splits][keep]: a beam's parts
  unsigned long long* merged = lists + (size_t)B * splits * keep;                      // [B][keep]: a beam's keys joined, then its scores
  int* best_token = reinterpret_cast<int*>(merged + B * keep);                         // [B][keep]
  float* best_logit = reinterpret_cast<float*>(best_token + B * keep);                 // [B][keep]
  __shared__ int picked[BEAM_KEEP];                                                    // beam << 8 | place
  __shared__ unsigned close_s;
  __shared__ BeamRow rows[BEAM_MAX];
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x, b = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (b < B) {                                      // (warps behind the beams' are there for sums that are made again)
    const size_t row = (size_t)g * B + b;
    const float score = scores[row];
    unsigned long long *mine = lists + (size_t)b * splits * keep, *joined = merged + b * keep;
    const unsigned long long* src = keys + row * splits * keep;
    const BeamPart part = lane < splits ? parts[row * splits + lane] : BeamPart{0.0, -INFINITY};
#pragma unroll 4
    for (int i = lane; i < splits * keep; i += 32) mine[i] = src[i];
    const float top = warp_max(part.max), whole = beam_whole(top);
    const BeamRow about = {score, top};
    if (lane == 0) rows[b] = about;
    double sum = 0.0;
    if (part.max > -INFINITY && (top < INFINITY || part.max == top)) sum = part.max == top ? part.sum : part.sum * beam_moved(part.max, beam_whole(part.max), top, whole);
    if (splits > 1) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    } else {
      sum = __shfl_sync(0xffffffffu, sum, 0);
    }
    __syncwarp();
    int found = 0;
    if (splits > 1) {                               // lane l walks the l-th part's list
      BeamHead h(mine + lane * keep, lane < splits ? keep : 0);
      for (; found < keep; ++found) {
        const unsigned long long best = warp_max_key(h.head);
        if (best == 0) break;
        if (h.head == best) {
          joined[found] = best;
          h.pop();
        }
      }
      __syncwarp();
    } else {
      joined = mine;
      found = keep;
    }
    const bool alive = score > -INFINITY && top > -INFINITY;
    // (the maximum's own term is 1, so the logarithm is never below 0)
    const double lse = fmax(whole == whole ? log(sum) + ((double)whole - (double)top * (double)BEAM_LOG2E) * 0.69314718055994531 : log(sum), 0.0);
    for (int i = lane; i < keep; i += 32) {
      const unsigned long long k = i < found && alive ? joined[i] : 0ull;
      const float x = beam_value((uint32_t)(k >> 32));
      const double v = beam_score(about, x, lse);
      merged[b * keep + i] = k != 0 && v > -INFINITY ? order_double(v) : 0ull;
      best_token[b * keep + i] = (int)~(uint32_t)k;
      best_logit[b * keep + i] = x;
    }
  }
  // (a step of 64-bit scores beside it: what is far from 0 has few bits left behind the point)
  auto close_to = [&](double v, double w) { return v - w < close_by + fabs(v) * 8.8817841970012523e-16; };       // 2^-50
  int n = 0;
  for (bool again = false;; again = true) {
    __syncthreads();
    if (b == 0) {
      // (what is picked is noted and written out by all lanes afterwards: a step of the join is a chain that nothing hides)
      BeamHead h(merged + lane * keep, lane < B ? keep : 0);
      for (n = 0; n < keep; ++n) {
        const unsigned long long best = warp_max_key(h.head);
        if (best == 0) break;
        const unsigned here = __ballot_sync(0xffffffffu, h.head == best);
        if ((here & ((2u << lane) - 1)) == 1u << lane) {                       // of equal scores the first beam's
          picked[n] = lane << 8 | (h.at - 2);
          h.pop();
        }
      }
      __syncwarp();
      // the beams with one that is left out as close to the last that is not
      const double last = n > 0 ? double_of(merged[(picked[n - 1] >> 8) * keep + (picked[n - 1] & 255)]) : 0.0;
      const unsigned behind = __ballot_sync(0xffffffffu, n > 0 && h.head != 0 && close_to(last, double_of(h.head)));
      unsigned close = 0;
      for (int i = lane; i < n; i += 32) {
        const int a = picked[i] >> 8;
        const double v = double_of(merged[a * keep + (picked[i] & 255)]);
        if (i + 1 < n) {
          const int c = picked[i + 1] >> 8;
          if (a != c && close_to(v, double_of(merged[c * keep + (picked[i + 1] & 255)]))) close |= 1u << a | 1u << c;
        } else if (behind & ~(1u << a)) {
          close |= 1u << a | behind;
        }
      }
      close = __reduce_or_sync(0xffffffffu, close);
      if (lane == 0) close_s = again ? 0u : close;
    }
    __syncthreads();
    const unsigned close = close_s;
    if (close == 0) break;
    beam_sums_again(logits, V, B, keep, close, rows, best_logit, merged);
  }
  if (b != 0) return;
  for (int i = lane; i < keep; i += 32) {
    const size_t o = (size_t)g * keep + i;
    const int which = i < n ? picked[i] : 0, from = (which >> 8) * keep + (which & 255);
    out_score[o] = i < n ? (float)double_of(merged[from]) : -INFINITY;
    out_parent[o] = i < n ? which >> 8 : -1;
    out_token[o] = i < n ? best_token[from] : -1;
  }
}

// ---- what goes on and what is finished ------------------------------------------------------------------------------------
//
// A warp a search.  The candidates come in their order; stop tokens among the first `beams` of them are finished continuations, scored s / n^power with n the tokens
// so far; the first `beams` that are none go on.  At n = max_new what would go on is finished too.  The pool holds the W best finished ones in order (of equal
// scores the earlier), lane w the w-th.  The search is over when nothing goes on, at max_new, or when the pool is full and the best that goes on cannot
// get above its last: log-probabilities only fall, so it ends at best at best / max_new^power (power >= 0) or best / (n + 1)^power (power < 0).
// A launch and its dependent loads bound it: 4 us for one search, 6.5 for 64 of 24 beams and 96 candidates (19 with a power an insertion; it is the same power for all of a step).
struct BeamPool {
  float* score;
  int *length, *parent, *token;
};

__global__ void __launch_bounds__(32) beam_advance_kernel(const float* c_score, const int* c_parent, const int* c_token, int keep, int beams, int W, const float* p_score,
                                                          const int* p_length, const int* p_parent, const int* p_token, const int* lengths, const int* done, const int* stop_ids,
                                                          int stops, int max_new, double power, float* out_score, int* out_parent, int* out_token, BeamPool pool,
                                                          int* out_lengths, int* out_done) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x, lane = threadIdx.x;
  const unsigned full = 0xffffffffu;
  float ps = -INFINITY;
  int pl = 0, pp = 0, pt = 0;
  if (lane < W) {
    ps = p_score[(size_t)g * W + lane];
    if (ps > -INFINITY) {
      pl = p_length[(size_t)g * W + lane];
      pp = p_parent[(size_t)g * W + lane];
      pt = p_token[(size_t)g * W + lane];
    } else {
      ps = -INFINITY;
    }
  }
  const bool was_done = done[g] != 0;
  const int before = lengths[g], n = before + 1;
  bool over = was_done;
  constexpr int PER = BEAM_KEEP / 32;
  float cs[PER], norm[PER];
  int cp[PER], ct[PER], place[PER];              // place: among those that go on, -1: not one of them
  int live = 0;
  float lead = -INFINITY;
  if (!was_done) {
    unsigned stop_mask[PER];
    const double length = pow((double)n, power), reach = pow((double)(power >= 0.0 ? max_new : n + 1), power);
    auto enter = [&](float v, int parent, int token) {        // uniform
      const int at = __popc(__ballot_sync(full, lane < W && ps >= v));
      const float us = __shfl_up_sync(full, ps, 1);
      const int ul = __shfl_up_sync(full, pl, 1), up = __shfl_up_sync(full, pp, 1), ut = __shfl_up_sync(full, pt, 1);
      if (lane < W && lane >= at && v > -INFINITY) {
        ps = lane == at ? v : us;
        pl = lane == at ? n : ul;
        pp = lane == at ? parent : up;
        pt = lane == at ? token : ut;
      }
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int r = 32 * j + lane;
      const bool in = r < keep;
      cs[j] = in ? c_score[(size_t)g * keep + r] : -INFINITY;
      cp[j] = in ? c_parent[(size_t)g * keep + r] : -1;
      ct[j] = in ? c_token[(size_t)g * keep + r] : -1;
      norm[j] = fmaxf((float)((double)cs[j] / length), cs[j] > -INFINITY ? -FLT_MAX : -INFINITY);         // (a finite score's: minus infinity is an empty place)
      bool stop = false;
      for (int k = 0; k < stops; ++k) stop |= stop_ids[k] == ct[j];
      const bool there = cs[j] > -INFINITY;
      stop_mask[j] = __ballot_sync(full, there && stop && r < beams);
      const unsigned goes = __ballot_sync(full, there && !stop);
      const int mine = live + __popc(goes & ((1u << lane) - 1));
      place[j] = (there && !stop && mine < beams) ? mine : -1;
      const unsigned first = __ballot_sync(full, place[j] == 0);
      if (first) lead = __shfl_sync(full, cs[j], __ffs(first) - 1);
      live += __popc(goes);
    }
    live = live < beams ? live : beams;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      for (unsigned mask = stop_mask[j]; mask; mask &= mask - 1) {
        const int l = __ffs(mask) - 1;
        enter(__shfl_sync(full, norm[j], l), __shfl_sync(full, cp[j], l), __shfl_sync(full, ct[j], l));
      }
    if (n >= max_new) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        for (unsigned mask = __ballot_sync(full, place[j] >= 0); mask; mask &= mask - 1) {
          const int l = __ffs(mask) - 1;
          enter(__shfl_sync(full, norm[j], l), __shfl_sync(full, cp[j], l), __shfl_sync(full, ct[j], l));
        }
      over = true;
    }
    const float last = __shfl_sync(full, ps, W - 1);
    if (live == 0) over = true;
    else if (last > -INFINITY && (float)((double)lead / reach) <= last) over = true;
  }
  // the next beams: those that go on, in order; the others of them idle (parent -1), or all of them where the search is over
  if (lane < beams && (over || lane >= live)) {
    out_score[(size_t)g * beams + lane] = -INFINITY;
    out_parent[(size_t)g * beams + lane] = over ? lane : -1;
    out_token[(size_t)g * beams + lane] = 0;
  }
  if (!over) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (place[j] >= 0) {
        out_score[(size_t)g * beams + place[j]] = cs[j];
        out_parent[(size_t)g * beams + place[j]] = cp[j];
        out_token[(size_t)g * beams + place[j]] = ct[j];
      }
  }
  if (lane < W) {
    pool.score[(size_t)g * W + lane] = ps;
    pool.length[(size_t)g * W + lane] = pl;
    pool.parent[(size_t)g * W + lane] = pp;
    pool.token[(size_t)g * W + lane] = pt;
  }
  if (lane == 0) {
    out_lengths[g] = was_done ? before : n;
    out_done[g] = over ? 1 : 0;
  }
}

static size_t beam_merge_smem(int B, int splits, int keep) { return (size_t)B * keep * (8 * splits + 16); }

static int beam_log2_lanes(int keep) {             // four groups a wanted key, where the threads suffice
  int lg = 5;
  while (lg > 0 && (BEAM_THREADS >> lg) < 4 * keep) --lg;
  return lg;
}

template <typename T>
static bool beam_both(const T* logits, const float* scores, int G, int B, int V, int keep, int splits, BeamPart* parts, unsigned long long* keys, float* out_score, int* out_parent,
                      int* out_token, cudaStream_t stream) {
  static SharedLimit rows_limit, merge_limit;
  constexpr int N = BeamLoad<T>::N;
  const size_t merge_smem = beam_merge_smem(B, splits, keep);
  if (!rows_limit.raise(beam_rows_kernel<T>, sizeof(BeamShared)) || !merge_limit.raise(beam_merge_kernel<T>, merge_smem)) return false;
  launch_kernel(beam_rows_kernel<T>, dim3((unsigned)(G * B * splits)), BEAM_THREADS, sizeof(BeamShared), stream, logits, V, keep, beam_log2_lanes(keep), splits,
                ((V + N - 1) / N + splits - 1) / splits, parts, keys);
  launch_kernel(beam_merge_kernel<T>, G, 32 * (B > 8 ? B : 8), merge_smem, stream, logits, V, scores, (const BeamPart*)parts, (const unsigned long long*)keys, B, keep, splits, beam_close(V),
                out_score, out_parent, out_token);
  return true;
}

}  // namespace sllm

using namespace sllm;

// Parts a row is cut into: as many as the SMs hold blocks (four an SM) for all rows, none shorter than a batch, at most 32 (a lane of the merging warp each) and 64 lists a search, beyond which
// the join costs what the parts save.  (us by parts, 152,064 float32 logits: 4 rows: 1 23, 8 11, 16 9.4, 32 8.7; 32 rows: 1 27, 4 18, 8 15, 16 16, 32 21; 128 rows: 1 39, 4 28, 8 30;
// 256 rows: 1 45, 2 38, 4 46; 512 rows: 1 61, 2 67.)
SLLM_EXPORT int sllm_beam_splits(int G, int B, int V) {
  const long long rows = (long long)G * B;
  long long n = rows > 0 ? 4ll * num_sms() / rows : 1;
  const long long batches = (V + BEAM_VALUES * BEAM_THREADS - 1) / (BEAM_VALUES * BEAM_THREADS);
  if (n > batches) n = batches;
  if (n > 64 / B) n = 64 / B;
  if (n > 32) n = 32;
  return n < 1 ? 1 : (int)n;
}

// scratch: G * B * splits * (8 * keep + 16) bytes, every part's keys, then its sum and maximum
SLLM_EXPORT int sllm_beam_candidates(const void* logits, int dtype, const float* scores, int G, int B, int V, int keep, int splits, void* scratch, float* out_score, int* out_parent,
                                     int* out_token, cudaStream_t stream) {
  SLLM_REQUIRE(G >= 0 && B >= 1 && B <= BEAM_MAX && V >= 1 && keep >= 1 && keep <= BEAM_KEEP && (long long)G * B < (1ll << 24), "beam_candidates: %d searches of %d beams, %d logits, %d kept", G, B, V,
               keep);
  SLLM_REQUIRE(V <= (1 << 30), "beam_candidates: rows of %d logits", V);
  SLLM_REQUIRE(dtype == SLLM_F32 || dtype == SLLM_BF16, "beam_candidates: unknown dtype %d", dtype);
  SLLM_REQUIRE(splits >= 1 && splits <= 32 && (long long)G * B * splits < (1ll << 31), "beam_candidates: %d parts a row", splits);
  if (G == 0) return SLLM_OK;
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(scratch);
  BeamPart* parts = reinterpret_cast<BeamPart*>(keys + (size_t)G * B * splits * keep);
  const bool there = dtype == SLLM_F32 ? beam_both((const float*)logits, scores, G, B, V, keep, splits, parts, keys, out_score, out_parent, out_token, stream)
                                       : beam_both((const __nv_bfloat16*)logits, scores, G, B, V, keep, splits, parts, keys, out_score, out_parent, out_token, stream);
  if (!there) {
    set_error("beam_candidates: cannot raise the shared memory limit");
    return SLLM_ERR_LAUNCH;
  }
  return launch_status("beam_candidates");
}

// `power` (on the host): the length penalty.  What is read may be what is written.
SLLM_EXPORT int sllm_beam_advance(const float* c_score, const int* c_parent, const int* c_token, int G, int keep, int beams, int W, const float* p_score, const int* p_length,
                                  const int* p_parent, const int* p_token, const int* lengths, const int* done, const int* stop_ids, int stops, int max_new, const double* power,
                                  float* out_score, int* out_parent, int* out_token, float* out_p_score, int* out_p_length, int* out_p_parent, int* out_p_token, int* out_lengths,
                                  int* out_done, cudaStream_t stream) {
  SLLM_REQUIRE(G >= 0 && keep >= 1 && keep <= BEAM_KEEP && beams >= 1 && beams <= BEAM_MAX && W >= 1 && W <= 32 && stops >= 0 && max_new >= 1,
               "beam_advance: %d searches, %d candidates, %d beams, a pool of %d, %d stops, max_new %d", G, keep, beams, W, stops, max_new);
  if (G == 0) return SLLM_OK;
  launch_kernel(beam_advance_kernel, G, 32, 0, stream, c_score, c_parent, c_token, keep, beams, W, p_score, p_length, p_parent, p_token, lengths, done, stop_ids, stops, max_new, *power,
                out_score, out_parent, out_token, BeamPool{out_p_score, out_p_length, out_p_parent, out_p_token}, out_lengths, out_done);
  return launch_status("beam_advance");
}
