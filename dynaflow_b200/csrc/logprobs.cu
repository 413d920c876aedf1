// Log probability of a given token, entropy and the most likely tokens of rows of logits, in one pass over them.
//
// In powers of two, with y = (x - m) log2(e) for a reference m, the largest logit, S = sum 2^y, U = sum 2^y y:
//   log2 p(t) = y_t - log2 S,      entropy (bits) = log2 S - U / S
// Every thread keeps (m, S, U) of what it has seen, in fp32 (two logits an instruction), relative to its own maximum;
// they are joined by moving to the larger reference. Logits at or below -2^123 are lifted to -2^123 on the way, so that
// 2^y y is 0 and not a NaN for the forbidden ones (-inf, or the type's lowest value); a slice that has nothing else is
// gone through again with subtractions. They are no candidates either: what is missing from the k largest at the end
// is filled with them, the lower index first.
//
// The k largest: a key of 64 bits, the logit made sortable in the upper half and the complement of its index in
// the lower, is unique, so equal logits come out with the lower index first. The pass itself only leaves every
// thread's maximum of each of at most 16 stretches of its part (as bf16, rounded up) in shared memory. With
// r = ceil(k / 8) the smallest of the eight warps' r-th largest lane maxima is a threshold that at least k logits of
// the block's part reach and few more do: the threads with a stretch that reaches it read that stretch again and put
// what reaches it into a list, which is ranked by comparing all pairs. If it does not fit (a great many equal logits),
// the k largest keys are selected by bisection instead.
//
// Bound: HBM, each logit is read once (2048 x 128256 bf16, sums alone: 84.8 us = 6.2 TB/s), then the exponentials (16 a
// clock and SM). With the most likely tokens the end of a block (threshold, reading again, ranking, 6 to 8 us) is in the
// way of few rows: 256 x 128256, 20 tokens: 25 us, sums alone 17 us. The next chunk is fetched while one
// is worked on. When there are few rows, a row is cut into slices: up to eight are one thread-block cluster, whose
// first CTA joins them through distributed shared memory; more of them (a very long row) leave records in the
// workspace for a second launch, which also joins the shards of a vocabulary that is split over ranks.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_util.h"
#include "ptx.cuh"

namespace df {
namespace logprobs {

constexpr int THREADS = 256;
constexpr int VECS = 4;                              // 16-byte vectors of a chunk a thread: 8192 bf16 or 4096 fp32 logits a block
constexpr int CHUNK = THREADS * VECS * 8;
constexpr int MAX_TOP = 32;
constexpr int LIST = 512;                            // candidates of a block
constexpr int MAX_SLICES = 64;
constexpr int CLUSTER_SLICES = 8;
constexpr int LONG_SLICE = 16;                       // chunks of a slice above which a row is cut into more than a cluster
constexpr int TARGET_BLOCKS = 296;                   // two a SM of 148 (64 x 128256, top 20: 12.1 us; four a SM: 14.8 us)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -0x1p123f;                  // a number of both types; (LOWEST - 2e38) log2(e) is still finite

typedef unsigned long long u64;

struct Stats {
  float m, s, u, x;  // reference logit (-inf: none so far), sum 2^y and sum 2^y y of y = (logit - m) log2(e), the given token's logit (-inf: not here)
};

struct Params {
  const void* logits;
  const void* ids;
  uint8_t* record;            // [parts] of (Stats [rows], u64 [rows][top])
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
  long long ld;
  int id_bytes, rows, vocab, vocab_start, top, slices, parts;
  int finish;                 // 1: the results, 0: one record of the parts
  int cluster;                // whether the slices of a row are one cluster
  size_t part_bytes;
  const uint8_t* parts_in;
};

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t sortable(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return b ^ ((b >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_sortable(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) != 0u ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 make_key(float x, uint32_t index) { return (static_cast<u64>(sortable(x)) << 32) | (0xffffffffu - index); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ u64 pack2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void join(Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {  // neither has a logit; NaN sums stay
    a.s += b.s;
    a.u += b.u;
  } else {
    const float da = fmaxf((a.m - m) * LOG2E, -1e30f), db = fmaxf((b.m - m) * LOG2E, -1e30f);
    const float fa = ex2f(da), fb = ex2f(db);
    a.u = fa * fmaf(da, a.s, a.u) + fb * fmaf(db, b.s, b.u);
    a.s = fa * a.s + fb * b.s;
  }
  a.m = m;
  a.x = fmaxf(a.x, b.x);
}

__device__ __forceinline__ Stats shuffle(const Stats& v, int o) {
  Stats r;
  r.m = __shfl_xor_sync(0xffffffffu, v.m, o);
  r.s = __shfl_xor_sync(0xffffffffu, v.s, o);
  r.u = __shfl_xor_sync(0xffffffffu, v.u, o);
  r.x = __shfl_xor_sync(0xffffffffu, v.x, o);
  return r;
}

constexpr int STRETCHES = 16;
struct Shared {
  __nv_bfloat16 stretch[STRETCHES][THREADS];
  u64 list[LIST];
  u64 kept[MAX_TOP];
  uint32_t warp_value[THREADS / 32];
  float warp_high[THREADS / 32];
  Stats stats[THREADS / 32];
  alignas(8) Stats total;
  uint32_t items[LIST];  // (stretch << 8 | thread) with a candidate
  int count, item_count, sum[2];
};

// The r-th largest of the lanes' values (equal ones count as often as they occur).
__device__ __forceinline__ uint32_t rth_of_lanes(uint32_t v, int r, int lane) {
  uint32_t top = 0u;
  for (int i = 0; i < r; ++i) {
    top = __reduce_max_sync(0xffffffffu, v);
    const unsigned at = __ballot_sync(0xffffffffu, v == top);
    if (lane == __ffs(at) - 1) v = 0u;
  }
  return top;
}

// The largest number of the logits' type below t.
__device__ __forceinline__ float just_below(float t, uint32_t ulp) {
  const uint32_t b = __float_as_uint(t);
  return __uint_as_float(t > 0.0f ? b - ulp : (t < 0.0f ? b + ulp : 0x80000000u | ulp));
}

// Keeps the `top` largest of the list, largest first, in sm.kept (0: fewer than that): a key's place is the number of
// larger ones, counted by four threads. All threads; ends with a barrier.
__device__ __forceinline__ void keep_largest(Shared& sm, int count, int top) {
  if (threadIdx.x < MAX_TOP) sm.kept[threadIdx.x] = 0ull;
  __syncthreads();
  const unsigned quad = 0xfu << (threadIdx.x & 28);
  for (int i = threadIdx.x >> 2; i < count; i += THREADS / 4) {
    const u64 key = sm.list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 3; j < count; j += 4) rank += sm.list[j] > key ? 1 : 0;
    rank += __shfl_xor_sync(quad, rank, 1);
    rank += __shfl_xor_sync(quad, rank, 2);
    if (rank < top && (threadIdx.x & 3) == 0) sm.kept[rank] = key;
  }
  __syncthreads();
}

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t FORBIDDEN = 0xff80ff80u;  // -inf, twice
  static constexpr uint32_t ULP = 0x10000u;           // of the fp32 bits of a logit
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ float get(const uint4& v, int j) {
    const uint32_t w = j < 4 ? (j < 2 ? v.x : v.y) : (j < 6 ? v.z : v.w);
    return __uint_as_float((j & 1) != 0 ? w & 0xffff0000u : w << 16);
  }
  // bit j of the result: whether logit j of the vector exceeds thr
  static __device__ __forceinline__ uint32_t exceeding(const uint4& v, float thr) {
    const __nv_bfloat162 t = __float2bfloat162_rn(thr);
    const uint32_t a = __hgt2_mask(reinterpret_cast<const __nv_bfloat162&>(v.x), t), b = __hgt2_mask(reinterpret_cast<const __nv_bfloat162&>(v.y), t);
    const uint32_t c = __hgt2_mask(reinterpret_cast<const __nv_bfloat162&>(v.z), t), d = __hgt2_mask(reinterpret_cast<const __nv_bfloat162&>(v.w), t);
    const uint32_t m = (a & 0x00010001u) | (b & 0x00040004u) | (c & 0x00100010u) | (d & 0x00400040u);  // 2 i and 16 + 2 i
    return (m | m >> 15) & 0xffu;
  }
  // largest of the vectors' logits (NaN does not count)
  template <int COUNT>
  static __device__ __forceinline__ float highest(const uint4 (&v)[COUNT]) {
    __nv_bfloat162 m = __float2bfloat162_rn(-INFINITY);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const __nv_bfloat162 a = __hmax2(reinterpret_cast<const __nv_bfloat162&>(v[i].x), reinterpret_cast<const __nv_bfloat162&>(v[i].y));
      const __nv_bfloat162 b = __hmax2(reinterpret_cast<const __nv_bfloat162&>(v[i].z), reinterpret_cast<const __nv_bfloat162&>(v[i].w));
      m = __hmax2(m, __hmax2(a, b));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
  // pair i of the vector, no lower than LOWEST (NaN stays)
  static __device__ __forceinline__ u64 pair(const uint4& v, int i) {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    const __nv_bfloat162 low = __float2bfloat162_rn(LOWEST);
    const __nv_bfloat162 h = __hmax2_nan(reinterpret_cast<const __nv_bfloat162&>(w), low);
    const uint32_t c = reinterpret_cast<const uint32_t&>(h);
    return pack2(__uint_as_float(c << 16), __uint_as_float(c & 0xffff0000u));
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t FORBIDDEN = 0xff800000u;
  static constexpr uint32_t ULP = 1u;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float get(const uint4& v, int j) { return __uint_as_float(j < 2 ? (j == 0 ? v.x : v.y) : (j == 2 ? v.z : v.w)); }
  static __device__ __forceinline__ uint32_t exceeding(const uint4& v, float thr) {
    return (get(v, 0) > thr ? 1u : 0u) | (get(v, 1) > thr ? 2u : 0u) | (get(v, 2) > thr ? 4u : 0u) | (get(v, 3) > thr ? 8u : 0u);
  }
  template <int COUNT>
  static __device__ __forceinline__ float highest(const uint4 (&v)[COUNT]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) m = fmaxf(m, fmaxf(fmaxf(get(v[i], 0), get(v[i], 1)), fmaxf(get(v[i], 2), get(v[i], 3))));
    return m;
  }
  static __device__ __forceinline__ float lift(float x) {  // max that keeps NaN
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(LOWEST));
    return r;
  }
  static __device__ __forceinline__ u64 pair(const uint4& v, int i) { return pack2(lift(get(v, 2 * i)), lift(get(v, 2 * i + 1))); }
};

// From base 2 with the fp32 constant LOG2E, whose powers are those of e to 2^-26 of the exponent.
__device__ __forceinline__ float to_nats(double bits) { return static_cast<float>(bits * (1.0 / static_cast<double>(LOG2E))); }
__device__ __forceinline__ float logprob_of(float x, const Stats& s, float log_s) {
  return to_nats((static_cast<double>(x) - static_cast<double>(s.m)) * static_cast<double>(LOG2E) - static_cast<double>(log_s));
}
__device__ __forceinline__ void write_results(const Params& p, int row, const Stats& s, const u64* kept) {
  const bool empty = s.m == -INFINITY && s.s == 0.0f;  // no token is allowed: no distribution
  const float log_s = log2f(s.s);
  if (threadIdx.x == 0) {
    p.logprob[row] = empty ? -INFINITY : logprob_of(s.x, s, log_s);
    p.entropy[row] = empty ? 0.0f : to_nats(static_cast<double>(log_s) - static_cast<double>(s.u / s.s));
  }
  if (static_cast<int>(threadIdx.x) < p.top) {
    const u64 key = kept[threadIdx.x];
    p.top_ids[static_cast<size_t>(row) * p.top + threadIdx.x] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    p.top_logprobs[static_cast<size_t>(row) * p.top + threadIdx.x] = empty ? -INFINITY : logprob_of(from_sortable(static_cast<uint32_t>(key >> 32)), s, log_s);
  }
}

__device__ __forceinline__ void write_record(const Params& p, int part, int row, const Stats& s, const u64* kept) {
  uint8_t* base = p.record + static_cast<size_t>(part) * p.part_bytes;
  if (threadIdx.x == 0) reinterpret_cast<Stats*>(base)[row] = s;
  if (static_cast<int>(threadIdx.x) < p.top)
    reinterpret_cast<u64*>(base + static_cast<size_t>(p.rows) * sizeof(Stats))[static_cast<size_t>(row) * p.top + threadIdx.x] = kept[threadIdx.x];
}

// A chunk of this thread's logits: vectors `at`, at + THREADS, ... of `vectors`; behind the last one -inf.
template <typename T>
__device__ __forceinline__ void load_chunk(uint4 (&v)[VECS], const uint4* src, int at, int vectors, bool full) {
  if (full) {  // the whole block's chunk
#pragma unroll
    for (int i = 0; i < VECS; ++i) v[i] = __ldg(src + at + i * THREADS);
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      v[i] = make_uint4(Vec<T>::FORBIDDEN, Vec<T>::FORBIDDEN, Vec<T>::FORBIDDEN, Vec<T>::FORBIDDEN);
      if (at + i * THREADS < vectors) v[i] = __ldg(src + at + i * THREADS);
    }
  }
}

// More candidates among elements [e0, e1) of the row than the list holds: the `top` largest keys, exactly, by bisection;
// they replace the list. (Goes through the elements 64 times: rows of equal logits come here, others do not.) All threads.
template <typename T>
__device__ __noinline__ void select_exactly(Shared& sm, const T* x0, int e0, int e1, int top) {
  const int tid = threadIdx.x;
  u64 found = 0ull;
  for (int bit = 63; bit >= 0; --bit) {
    const u64 mid = found | (1ull << bit);
    int n = 0;
#pragma unroll 1
    for (int e = e0 + tid; e < e1; e += THREADS) n += make_key(Vec<T>::one(x0 + e), static_cast<uint32_t>(e)) >= mid ? 1 : 0;
    if (tid == 0) sm.sum[bit & 1] = 0;
    __syncthreads();
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0) atomicAdd(&sm.sum[bit & 1], n);
    __syncthreads();
    if (sm.sum[bit & 1] >= top) found = mid;
  }
  if (tid == 0) sm.count = 0;
  __syncthreads();
  for (int e = e0 + tid; e < e1; e += THREADS) {
    const u64 key = make_key(Vec<T>::one(x0 + e), static_cast<uint32_t>(e));
    if (key >= found) sm.list[atomicAdd(&sm.count, 1)] = key;
  }
  __syncthreads();
}

// The list has fewer than `top` keys because the other logits of elements [e0, e1) are forbidden (at or below LOWEST):
// adds those, larger values first, of equal ones the lower index. All threads.
template <typename T>
__device__ __noinline__ void fill_forbidden(Shared& sm, const T* x0, int e0, int e1, int top) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t below = sortable(LOWEST) + 1u;  // values under it are still to be added
  while (true) {
    uint32_t value = 0u;                   // the largest of them; 0: none is left
    for (int e = e0 + tid; e < e1; e += THREADS) {
      const uint32_t o = sortable(Vec<T>::one(x0 + e));
      if (o < below) value = max(value, o);
    }
    __syncthreads();
    value = __reduce_max_sync(0xffffffffu, value);
    if (lane == 0) sm.warp_value[warp] = value;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) value = max(value, sm.warp_value[i]);
    int count = sm.count;
    if (value == 0u || count >= top) return;
    for (int e = e0; e < e1 && count < top; e += THREADS) {  // in order of the index
      const bool here = e + tid < e1 && sortable(Vec<T>::one(x0 + e + tid)) == value;
      const unsigned votes = __ballot_sync(0xffffffffu, here);
      __syncthreads();
      if (lane == 0) sm.warp_value[warp] = __popc(votes);
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) before += sm.warp_value[i];
        all += sm.warp_value[i];
      }
      const int at = count + before + __popc(votes & ((1u << lane) - 1u));
      if (here && at < top) sm.list[at] = static_cast<u64>(value) << 32 | (0xffffffffu - static_cast<uint32_t>(e + tid));
      count = min(count + all, top);
    }
    __syncthreads();
    if (tid == 0) sm.count = count;
    __syncthreads();
    below = value;
  }
}

__device__ __forceinline__ u64 read_remote(const u64* p, unsigned rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const Params p) {
  constexpr int N = Vec<T>::N;
  __shared__ Shared sm;
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x0 = static_cast<const T*>(p.logits) + row * p.ld;
  // whole vectors on 16-byte boundaries from element `head`; the few logits before and behind them are a thread's each
  const int head = min(static_cast<int>((16u - (reinterpret_cast<uintptr_t>(x0) & 15u)) % 16u / sizeof(T)), p.vocab);
  const int vectors = (p.vocab - head) / N;
  const uint4* src = reinterpret_cast<const uint4*>(x0 + head);
  const int chunks = (vectors + THREADS * VECS - 1) / (THREADS * VECS);
  const int c0 = chunks * slice / p.slices, c1 = chunks * (slice + 1) / p.slices;
  float extra = -INFINITY;
  int extra_at = 0;
  if (tid < 16 && slice == (tid < 8 ? 0 : p.slices - 1)) {
    extra_at = tid < 8 ? tid : head + vectors * N + tid - 8;
    if (extra_at < (tid < 8 ? head : p.vocab)) extra = Vec<T>::one(x0 + extra_at);
  }
  float given = -INFINITY;
  if (slice == 0 && tid == 0) {
    const long long id = (p.id_bytes == 8 ? static_cast<const long long*>(p.ids)[row] : static_cast<const int*>(p.ids)[row]) - p.vocab_start;
    if (id >= 0 && id < p.vocab) given = Vec<T>::one(x0 + id);
  }
  if (TOP && tid == 0) sm.count = sm.item_count = 0;
  float high = -INFINITY;  // largest logit of this thread
  u64 s2 = pack2(0.f, 0.f), u2 = s2;
  const u64 scale = pack2(LOG2E, LOG2E);
  auto load = [&](uint4 (&v)[VECS], int ch) { load_chunk<T>(v, src, ch * (THREADS * VECS) + tid, vectors, (ch + 1) * (THREADS * VECS) <= vectors); };
  const int per_stretch = max((c1 - c0 + STRETCHES - 1) / STRETCHES, 1);  // chunks
  float stretch_high = -INFINITY;
  int in_stretch = 0;
  auto work = [&](const uint4 (&v)[VECS], int ch) {
    const float now = Vec<T>::highest(v);
    if (TOP) {
      stretch_high = fmaxf(stretch_high, now);
      if (++in_stretch == per_stretch || ch + 1 == c1) {
        sm.stretch[(ch - c0) / per_stretch][tid] = __float2bfloat16_ru(stretch_high);
        stretch_high = -INFINITY;
        in_stretch = 0;
      }
    }
    if (now > high) {
      if (high > LOWEST) {
        const float d = (high - now) * LOG2E, f = ex2f(d);
        const float2 s = unpack2(s2), u = unpack2(u2);
        s2 = pack2(f * s.x, f * s.y);
        u2 = pack2(f * fmaf(d, s.x, u.x), f * fmaf(d, s.y, u.y));
      }
      high = now;
    }
    const float ref = high > LOWEST ? -high : 0.0f;  // without a reference 2^(LOWEST) is 0, too
    const u64 minus = pack2(ref, ref);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const u64 y = mul2(add2(Vec<T>::pair(v[i], j), minus), scale);
        const float2 yy = unpack2(y);
        const u64 e = pack2(ex2f(yy.x), ex2f(yy.y));
        s2 = add2(s2, e);
        u2 = fma2(e, y, u2);
      }
  };
  uint4 va[VECS], vb[VECS];  // one chunk is on its way while the other is worked on
  if (c0 < c1) load(va, c0);
#pragma unroll 1
  for (int ch = c0; ch < c1; ch += 2) {
    if (ch + 1 < c1) load(vb, ch + 1);
    work(va, ch);
    if (ch + 1 < c1) {
      if (ch + 2 < c1) load(va, ch + 2);
      work(vb, ch + 1);
    }
  }
  // ---- the block's sums
  const float2 s = unpack2(s2), u = unpack2(u2);
  Stats st{-INFINITY, 0.0f, 0.0f, given};
  if (high > LOWEST) {
    st.m = high;
    st.s = s.x + s.y;
    st.u = u.x + u.y;
  } else if (s.x + s.y != s.x + s.y) {
    st.s = NAN;  // a NaN among forbidden tokens
  }
  if (extra > LOWEST) join(st, Stats{extra, 1.0f, 0.0f, -INFINITY});
  if (extra != extra) st.s = NAN;
  high = fmaxf(high, extra);
  const float mine = high;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    join(st, shuffle(st, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  // The threshold is the least of the r-th largest thread maxima of `ranked` warps, ranked * r >= top: so many logits reach
  // it. Only warps whose threads all have a vector are asked (at least the first): one without logits would let everything
  // through (2000 rows of 1000 bf16 logits, top 20: 165 us instead of 24). Fewer vectors than that have no threshold.
  const int in_block = min(c1 * (THREADS * VECS), vectors) - c0 * (THREADS * VECS);  // vectors
  const int ranked = max(min(in_block, THREADS) / 32, 1), r = (p.top + ranked - 1) / ranked;
  uint32_t rth = 0u;
  if (TOP && in_block >= r) rth = warp < ranked ? rth_of_lanes(sortable(mine), r, lane) : 0xffffffffu;
  if (lane == 0) {
    sm.stats[warp] = st;
    sm.warp_high[warp] = high;
    sm.warp_value[warp] = rth;
  }
  __syncthreads();
  // this block's logits; the first slice has those before the first vector, the last one those behind the last
  const int e0 = slice == 0 ? 0 : head + c0 * (THREADS * VECS * N), e1 = slice == p.slices - 1 ? p.vocab : head + c1 * (THREADS * VECS * N);
  if (TOP) {
    uint32_t reach = sm.warp_value[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) reach = min(reach, sm.warp_value[i]);
    const float least = from_sortable(reach), past = least > LOWEST ? just_below(least, Vec<T>::ULP) : LOWEST;  // a candidate exceeds it
    auto append = [&](float x, int e) {
      const int at = atomicAdd(&sm.count, 1);
      if (at < LIST) sm.list[at] = make_key(x, static_cast<uint32_t>(e));
    };
    if (mine > past) {
      if (extra > past) append(extra, extra_at);
      const int stretches = (c1 - c0 + per_stretch - 1) / per_stretch;
#pragma unroll 4
      for (int i = 0; i < stretches; ++i)
        if (__bfloat162float(sm.stretch[i][tid]) > past) {  // (or only seems so when rounded up)
          const int at = atomicAdd(&sm.item_count, 1);
          if (at < LIST) sm.items[at] = static_cast<uint32_t>(i << 8 | tid);
        }
    }
    __syncthreads();
    const int items = sm.item_count;
    if (items > LIST) {
      if (tid == 0) sm.count = LIST + 1;
    } else {
      for (int w = tid; w < items * VECS * per_stretch; w += THREADS) {
        const int item = w / (VECS * per_stretch), rest = w - item * (VECS * per_stretch);
        const int i = static_cast<int>(sm.items[item] >> 8), thread = static_cast<int>(sm.items[item] & 255u);
        const int ch = c0 + i * per_stretch + rest / VECS, at = ch * (THREADS * VECS) + rest % VECS * THREADS + thread;
        if (ch >= c1 || at >= vectors) continue;
        const uint4 v = __ldg(src + at);
#pragma unroll 1
        for (uint32_t bits = Vec<T>::exceeding(v, past); bits != 0u; bits &= bits - 1u) {
          const int j = __ffs(bits) - 1;
          append(Vec<T>::get(v, j), head + at * N + j);
        }
      }
    }
  }
  if (warp == 0) {
    st = sm.stats[lane & 7];
    high = sm.warp_high[lane & 7];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      join(st, shuffle(st, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if (high <= LOWEST) {
      // nothing above LOWEST: forbidden tokens only, or finite logits that low, which are summed with subtractions
      const bool nan = st.s != st.s;
      float sum = 0.0f, moment = 0.0f;
      if (high > -INFINITY)
#pragma unroll 1
        for (int e = e0 + lane; e < e1; e += 32) {
          const float y = (Vec<T>::one(x0 + e) - high) * LOG2E, w = ex2f(y);
          sum += w;
          if (w > 0.0f) moment = fmaf(w, y, moment);
        }
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        moment += __shfl_xor_sync(0xffffffffu, moment, o);
      }
      st.m = high;
      st.s = nan ? NAN : sum;
      st.u = moment;
    }
    if (lane == 0) sm.total = st;
  }
  if (TOP) {
    __syncthreads();
    if (sm.count > LIST) select_exactly(sm, x0, e0, e1, p.top);
    if (sm.count < p.top) fill_forbidden(sm, x0, e0, e1, p.top);
    keep_largest(sm, min(sm.count, LIST), p.top);
  } else {
    __syncthreads();
  }
  if (TOP && p.vocab_start != 0 && tid < p.top && sm.kept[tid] != 0ull) sm.kept[tid] -= static_cast<u64>(p.vocab_start);
  if (p.cluster) {
    cluster_sync();  // every slice's sums and keys are in its shared memory
    if (slice == 0) {
      if (warp == 0) {
        st = sm.total;
        if (lane < p.slices) {
          const u64 a = read_remote(reinterpret_cast<const u64*>(&sm.total), lane), b = read_remote(reinterpret_cast<const u64*>(&sm.total) + 1, lane);
          const float2 ms = unpack2(a), ux = unpack2(b);
          st = Stats{ms.x, ms.y, ux.x, ux.y};
        } else {
          st = Stats{-INFINITY, 0.0f, 0.0f, -INFINITY};
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) join(st, shuffle(st, o));
        __syncwarp();
        if (lane == 0) sm.stats[0] = st;
      }
      if (TOP) {
        const int n = p.slices * p.top;  // at most 8 * 32, a key a thread
        const u64 key = tid < n ? read_remote(&sm.kept[tid % p.top], tid / p.top) : 0ull;
        if (tid < n) sm.list[tid] = key;
        __syncthreads();
        keep_largest(sm, n, p.top);
      } else {
        __syncthreads();
      }
      st = sm.stats[0];
    }
    cluster_sync();  // nobody leaves while its shared memory is read
    if (slice != 0) return;
  } else {
    st = sm.total;
  }
  if (p.finish && (p.cluster || p.slices == 1))
    write_results(p, row, st, sm.kept);
  else
    write_record(p, p.cluster ? 0 : slice, row, st, sm.kept);
}

// Joins the parts of a row: sums in the order of the parts, the k largest of their keys.
__global__ void __launch_bounds__(THREADS) token_logprobs_join_kernel(const Params p) {
  extern __shared__ u64 keys[];
  __shared__ u64 kept[MAX_TOP];
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x, tid = threadIdx.x;
  const int n = p.parts * p.top;
  for (int i = tid; i < n; i += THREADS) {
    const int part = i / p.top;
    keys[i] = reinterpret_cast<const u64*>(p.parts_in + part * p.part_bytes + static_cast<size_t>(p.rows) * sizeof(Stats))[static_cast<size_t>(row) * p.top + (i - part * p.top)];
  }
  if (tid < MAX_TOP) kept[tid] = 0ull;
  __syncthreads();
  for (int i = tid; i < n; i += THREADS) {
    const u64 key = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > key ? 1 : 0;
    if (rank < p.top && key != 0ull) kept[rank] = key;
  }
  __syncthreads();
  Stats st = reinterpret_cast<const Stats*>(p.parts_in)[row];
  for (int i = 1; i < p.parts; ++i) join(st, reinterpret_cast<const Stats*>(p.parts_in + i * p.part_bytes)[row]);
  if (p.finish)
    write_results(p, row, st, kept);
  else
    write_record(p, 0, row, st, kept);
}

// Slices a row is cut into: enough blocks to fill the device and no slice shorter than a chunk, at most a cluster of
// them unless that leaves long slices to few rows.
int slices_of(int rows, int vocab) {
  const int chunks = (vocab + CHUNK - 1) / CHUNK;
  int want = (TARGET_BLOCKS + rows - 1) / rows;
  if (want > chunks) want = chunks;
  if (want > CLUSTER_SLICES && (chunks + CLUSTER_SLICES - 1) / CLUSTER_SLICES > LONG_SLICE) return want < MAX_SLICES ? want : MAX_SLICES;
  int s = 1;
  while (s < CLUSTER_SLICES && 2 * s <= want) s *= 2;
  return s;
}
size_t record_bytes(int rows, int top) { return static_cast<size_t>(rows) * (sizeof(Stats) + static_cast<size_t>(top) * sizeof(u64)); }

template <typename Kernel>
int launch(Kernel kernel, unsigned blocks, unsigned cluster, size_t smem, const Params& p, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  cfg.numAttrs = dependent_launch_attr(&attrs[0]);
  if (cluster > 1) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = cluster;
    attrs[cfg.numAttrs].val.clusterDim.y = 1;
    attrs[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(DF_ECUDA, "log probability launch: %s", cudaGetErrorString(e));
  }
  return DF_OK;
}

int check_logits(const void* logits, int fp32, long long ld, const void* ids, int id_bytes, int rows, int vocab, int top) {
  if (logits == nullptr || ids == nullptr) return fail(DF_EINVAL, "NULL pointer argument");
  if (rows <= 0 || vocab <= 0) return fail(DF_EINVAL, "rows and vocab must be positive");
  if (fp32 != 0 && fp32 != 1) return fail(DF_EINVAL, "fp32 must be 0 (bf16 logits) or 1");
  if (id_bytes != 4 && id_bytes != 8) return fail(DF_EINVAL, "ids are 4- or 8-byte integers");
  if (ld < vocab) return fail(DF_EINVAL, "the row stride (%lld) must cover the vocabulary (%d)", ld, vocab);
  if (top < 0 || top > MAX_TOP || top > vocab) return fail(DF_EUNSUPPORTED, "top must be 0 to %d and no more than the vocabulary (got %d)", MAX_TOP, top);
  if (vocab > (1 << 30)) return fail(DF_EUNSUPPORTED, "at most 2^30 logits a row");
  if (static_cast<long long>(rows) * MAX_SLICES > 0x7fffffffLL) return fail(DF_EUNSUPPORTED, "too many rows");
  if ((reinterpret_cast<uintptr_t>(logits) % (fp32 ? 4 : 2)) != 0) return fail(DF_EINVAL, "logits must be aligned to their elements");
  return DF_OK;
}

}  // namespace logprobs
}  // namespace df

extern "C" size_t df_token_logprobs_record_bytes(int rows, int top) {
  if (rows <= 0 || top < 0 || top > df::logprobs::MAX_TOP) return 0;
  return df::logprobs::record_bytes(rows, top);
}

extern "C" size_t df_token_logprobs_workspace_bytes(int rows, int vocab, int top) {
  using namespace df::logprobs;
  if (rows <= 0 || vocab <= 0 || top < 0 || top > MAX_TOP) return 0;
  const int slices = slices_of(rows, vocab);
  return slices > CLUSTER_SLICES ? slices * record_bytes(rows, top) : 16;  // a cluster needs none
}

static int run_logprobs(df::logprobs::Params& p, int fp32, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace df;
  using namespace df::logprobs;
  p.slices = slices_of(p.rows, p.vocab);
  p.cluster = p.slices > 1 && p.slices <= CLUSTER_SLICES;
  p.part_bytes = record_bytes(p.rows, p.top);
  uint8_t* result = p.record;
  if (p.slices > CLUSTER_SLICES) {
    const size_t need = p.slices * p.part_bytes;
    if (workspace == nullptr || workspace_bytes < need) return fail(DF_EINVAL, "workspace of %zu bytes is too small (need %zu)", workspace_bytes, need);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(DF_EINVAL, "the workspace must be 16-byte aligned");
    p.record = static_cast<uint8_t*>(workspace);
  }
  const unsigned blocks = static_cast<unsigned>(p.rows) * static_cast<unsigned>(p.slices), cluster = p.cluster ? p.slices : 1;
  auto kernel = fp32 ? (p.top > 0 ? token_logprobs_kernel<float, true> : token_logprobs_kernel<float, false>)
                     : (p.top > 0 ? token_logprobs_kernel<__nv_bfloat16, true> : token_logprobs_kernel<__nv_bfloat16, false>);
  const int rc = launch(kernel, blocks, cluster, 0, p, stream);
  if (rc != DF_OK || p.slices <= CLUSTER_SLICES) return rc;
  p.parts = p.slices;
  p.parts_in = static_cast<const uint8_t*>(workspace);
  p.record = result;
  return launch(token_logprobs_join_kernel, static_cast<unsigned>(p.rows), 1, static_cast<size_t>(p.parts) * p.top * sizeof(u64), p, stream);
}

extern "C" int df_token_logprobs(const void* logits, int fp32, long long ld, const void* ids_dev, int id_bytes, int rows, int vocab,
                                 int top, float* logprob_dev, float* entropy_dev, int* top_ids_dev, float* top_logprobs_dev,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace df;
  using namespace df::logprobs;
  const int rc = check_logits(logits, fp32, ld, ids_dev, id_bytes, rows, vocab, top);
  if (rc != DF_OK) return rc;
  if (logprob_dev == nullptr || entropy_dev == nullptr || (top > 0 && (top_ids_dev == nullptr || top_logprobs_dev == nullptr)))
    return fail(DF_EINVAL, "NULL pointer argument");
  Params p = {};
  p.logits = logits;
  p.ids = ids_dev;
  p.ld = ld;
  p.id_bytes = id_bytes;
  p.rows = rows;
  p.vocab = vocab;
  p.top = top;
  p.finish = 1;
  p.logprob = logprob_dev;
  p.entropy = entropy_dev;
  p.top_ids = top_ids_dev;
  p.top_logprobs = top_logprobs_dev;
  return run_logprobs(p, fp32, workspace, workspace_bytes, stream);
}

extern "C" int df_token_logprobs_shard(const void* logits, int fp32, long long ld, const void* ids_dev, int id_bytes, int rows, int vocab,
                                       int vocab_start, int top, void* record_dev, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace df;
  using namespace df::logprobs;
  const int rc = check_logits(logits, fp32, ld, ids_dev, id_bytes, rows, vocab, top);
  if (rc != DF_OK) return rc;
  if (record_dev == nullptr) return fail(DF_EINVAL, "NULL pointer argument");
  if (vocab_start < 0 || vocab_start > (1 << 30)) return fail(DF_EINVAL, "vocab_start must be 0 to 2^30");
  if ((reinterpret_cast<uintptr_t>(record_dev) & 15u) != 0) return fail(DF_EINVAL, "the record must be 16-byte aligned");
  Params p = {};
  p.logits = logits;
  p.ids = ids_dev;
  p.ld = ld;
  p.id_bytes = id_bytes;
  p.rows = rows;
  p.vocab = vocab;
  p.vocab_start = vocab_start;
  p.top = top;
  p.record = static_cast<uint8_t*>(record_dev);
  return run_logprobs(p, fp32, workspace, workspace_bytes, stream);
}

extern "C" int df_token_logprobs_join(const void* records_dev, int parts, int rows, int top, float* logprob_dev, float* entropy_dev,
                                      int* top_ids_dev, float* top_logprobs_dev, void* stream) {
  using namespace df;
  using namespace df::logprobs;
  if (records_dev == nullptr || logprob_dev == nullptr || entropy_dev == nullptr || (top > 0 && (top_ids_dev == nullptr || top_logprobs_dev == nullptr)))
    return fail(DF_EINVAL, "NULL pointer argument");
  if (parts <= 0 || parts > MAX_SLICES || rows <= 0) return fail(DF_EINVAL, "rows must be positive, parts 1 to %d", MAX_SLICES);
  if (top < 0 || top > MAX_TOP) return fail(DF_EUNSUPPORTED, "top must be 0 to %d (got %d)", MAX_TOP, top);
  if ((reinterpret_cast<uintptr_t>(records_dev) & 15u) != 0) return fail(DF_EINVAL, "the records must be 16-byte aligned");
  Params p = {};
  p.rows = rows;
  p.top = top;
  p.parts = parts;
  p.finish = 1;
  p.part_bytes = record_bytes(rows, top);
  p.parts_in = static_cast<const uint8_t*>(records_dev);
  p.logprob = logprob_dev;
  p.entropy = entropy_dev;
  p.top_ids = top_ids_dev;
  p.top_logprobs = top_logprobs_dev;
  return launch(token_logprobs_join_kernel, static_cast<unsigned>(rows), 1, static_cast<size_t>(parts) * top * sizeof(u64), p, stream);
}
