// Log probability of a given token, entropy and the most likely tokens of rows of logits, in one pass over them.
//
// With m the largest logit of a row, S = sum exp(x - m) and U = sum exp(x - m) (x - m):
//   log p(t) = (x_t - m) - log S,      entropy = log S - U / S
// Every thread keeps (m, S, U) of what it has seen, in fp32, relative to its own maximum; they are joined by
// rescaling to the larger one. exp(-inf) (x - m) counts as 0, so forbidden tokens (-inf) take no part.
//
// The k largest: a key of 64 bits, the logit made sortable in the upper half and the complement of its index in
// the lower, is unique, so equal logits come out with the lower index first. A block goes through its part of the
// row in chunks of 8192 logits. The first chunk gives a threshold: the k-th largest of the 256 threads' maxima is
// reached by at least k logits and by few more; logits above it are put into a list (their order does not matter,
// the keys decide), and a list that gets long is cut to its k largest, which raises the threshold. A chunk that
// brings more than the list can hold (logits that grow along the row, or a great many equal ones) is selected
// exactly by bisection over the keys instead.
//
// Bound: HBM, each logit is read once. A row is cut into slices when there are few rows, and a second launch joins
// the slices (the same launch joins the shards of a vocabulary that is split over ranks).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_util.h"
#include "ptx.cuh"

namespace df {
namespace logprobs {

constexpr int THREADS = 256;
constexpr int PER_THREAD = 32;                       // logits of a chunk a thread
constexpr int CHUNK = THREADS * PER_THREAD;
constexpr int MAX_TOP = 32;
constexpr int LIST = 512;                            // candidates of a block
constexpr int MAX_SLICES = 64;
constexpr int TARGET_BLOCKS = 592;                   // four a SM of 148
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

struct Stats {
  float m, s, u, x;  // maximum, sum exp, sum exp * (x - m), the given token's logit (-inf: not here)
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

__device__ __forceinline__ void join(Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {  // neither has a distribution; NaN sums stay
    a.s += b.s;
    a.u += b.u;
  } else {
    const float da = fmaxf(a.m - m, -1e30f), db = fmaxf(b.m - m, -1e30f);
    const float fa = ex2f(da * LOG2E), fb = ex2f(db * LOG2E);
    a.u = fa * (a.u + da * a.s) + fb * (b.u + db * b.s);
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

struct Shared {
  u64 list[LIST];
  u64 kept[MAX_TOP];
  uint32_t thread_max[THREADS];
  Stats stats[THREADS / 32];
  int count, sum[2];
  uint32_t threshold;
};

// The sortable value that exactly `k` or more of the 256 thread maxima reach and k - 1 or fewer exceed (by the first warp).
__device__ __forceinline__ uint32_t kth_of_threads(const uint32_t* v, int k, int lane) {
  uint32_t x[THREADS / 32];
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) x[i] = v[i * 32 + lane];
  uint32_t found = 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t mid = found | (1u << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) n += x[i] >= mid ? 1 : 0;
    if (__reduce_add_sync(0xffffffffu, n) >= k) found = mid;
  }
  return found;
}

// Keeps the `top` largest of the list, largest first, in sm.kept (0: fewer than that). All threads; ends with a barrier.
__device__ __forceinline__ void keep_largest(Shared& sm, int count, int top) {
  if (threadIdx.x < MAX_TOP) sm.kept[threadIdx.x] = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += THREADS) {
    const u64 key = sm.list[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += sm.list[j] > key ? 1 : 0;
    if (rank < top) sm.kept[rank] = key;
  }
  __syncthreads();
}

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};

__device__ __forceinline__ void write_results(const Params& p, int row, const Stats& s, const u64* kept) {
  const bool empty = s.m == -INFINITY && s.s == 0.0f;  // no token is allowed: no distribution
  const float log_s = logf(s.s);
  if (threadIdx.x == 0) {
    p.logprob[row] = empty ? -INFINITY : (s.x - s.m) - log_s;
    p.entropy[row] = empty ? 0.0f : log_s - s.u / s.s;
  }
  if (static_cast<int>(threadIdx.x) < p.top) {
    const u64 key = kept[threadIdx.x];
    p.top_ids[static_cast<size_t>(row) * p.top + threadIdx.x] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    p.top_logprobs[static_cast<size_t>(row) * p.top + threadIdx.x] =
        empty ? -INFINITY : (from_sortable(static_cast<uint32_t>(key >> 32)) - s.m) - log_s;
  }
}

__device__ __forceinline__ void write_record(const Params& p, int part, int row, const Stats& s, const u64* kept) {
  uint8_t* base = p.record + static_cast<size_t>(part) * p.part_bytes;
  if (threadIdx.x == 0) reinterpret_cast<Stats*>(base)[row] = s;
  if (static_cast<int>(threadIdx.x) < p.top)
    reinterpret_cast<u64*>(base + static_cast<size_t>(p.rows) * sizeof(Stats))[static_cast<size_t>(row) * p.top + threadIdx.x] = kept[threadIdx.x];
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 3) token_logprobs_kernel(const Params p) {
  constexpr int N = Vec<T>::N, VECS = PER_THREAD / N;
  __shared__ Shared sm;
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x0 = static_cast<const T*>(p.logits) + row * p.ld;
  // vectors lie on 16-byte boundaries; the row begins `lead` elements into its first one
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x0) & 15u) / sizeof(T));
  const int vectors = (p.vocab + lead + N - 1) / N;
  const int chunks = (vectors + THREADS * VECS - 1) / (THREADS * VECS);
  const int c0 = static_cast<int>(static_cast<long long>(chunks) * slice / p.slices), c1 = static_cast<int>(static_cast<long long>(chunks) * (slice + 1) / p.slices);
  if (tid == 0) {
    sm.count = 0;
    sm.threshold = 0u;
  }
  if (tid < MAX_TOP) sm.kept[tid] = 0ull;
  Stats st{-INFINITY, 0.0f, 0.0f, -INFINITY};
  bool first = true;
  for (int c = c0; c < c1; ++c) {
    float x[PER_THREAD];
    const int v0 = c * THREADS * VECS + tid;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int e = (v0 + i * THREADS) * N - lead;  // first element of the vector
      if (e >= 0 && e + N <= p.vocab) {
        Vec<T>::unpack(*reinterpret_cast<const uint4*>(x0 + e), x + i * N);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[i * N + j] = e + j >= 0 && e + j < p.vocab ? Vec<T>::one(x0 + e + j) : -INFINITY;
      }
    }
    float high = x[0];
#pragma unroll
    for (int i = 1; i < PER_THREAD; ++i) high = fmaxf(high, x[i]);
    // ---- sums
    if (high > st.m) {
      if (st.m != -INFINITY) {
        const float d = st.m - high, f = ex2f(d * LOG2E);
        st.u = f * (st.u + d * st.s);
        st.s *= f;
      }
      st.m = high;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const float d = x[i] - ref, e = ex2f(d * LOG2E);
      st.s += e;
      st.u = fmaf(e, fmaxf(d, -1e30f), st.u);
    }
    // ---- candidates
    if (p.top > 0) {
      auto index_of = [&](int i) { return (v0 + (i / N) * THREADS) * N - lead + i % N; };
      auto valid = [&](int i) { const int e = index_of(i); return e >= 0 && e < p.vocab; };
      if (first) {
        sm.thread_max[tid] = sortable(high);
        __syncthreads();
        if (warp == 0) {
          const uint32_t t = kth_of_threads(sm.thread_max, p.top, lane);
          if (lane == 0) sm.threshold = t - 1u;  // the first chunk takes what reaches it
        }
        __syncthreads();
      }
      const uint32_t above = sm.threshold;
      const int before = sm.count;
      __syncthreads();
      if (sortable(high) > above) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i)
          if (sortable(x[i]) > above && valid(i)) {
            const int at = atomicAdd(&sm.count, 1);
            if (at < LIST) sm.list[at] = make_key(x[i], static_cast<uint32_t>(index_of(i)));
          }
      }
      __syncthreads();
      const int count = sm.count;
      if (count > LIST) {
        // too many: the k-th largest key of the list so far and this chunk by bisection, then exactly those that reach it
        u64 found = 0ull;
        for (int bit = 63; bit >= 0; --bit) {
          const u64 mid = found | (1ull << bit);
          int n = 0;
#pragma unroll
          for (int i = 0; i < PER_THREAD; ++i) n += valid(i) && make_key(x[i], static_cast<uint32_t>(index_of(i))) >= mid ? 1 : 0;
          for (int i = tid; i < before; i += THREADS) n += sm.list[i] >= mid ? 1 : 0;
          if (tid == 0) sm.sum[bit & 1] = 0;
          __syncthreads();
          n = __reduce_add_sync(0xffffffffu, n);
          if (lane == 0) atomicAdd(&sm.sum[bit & 1], n);
          __syncthreads();
          if (sm.sum[bit & 1] >= p.top) found = mid;
        }
        if (tid == 0) sm.count = 0;
        __syncthreads();
        for (int i = tid; i < before; i += THREADS)
          if (sm.list[i] >= found) sm.kept[atomicAdd(&sm.count, 1)] = sm.list[i];
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
          const u64 key = make_key(x[i], static_cast<uint32_t>(index_of(i)));
          if (valid(i) && key >= found) sm.kept[atomicAdd(&sm.count, 1)] = key;
        }
        __syncthreads();
        if (tid < p.top) sm.list[tid] = sm.kept[tid];
        if (tid == 0) sm.threshold = static_cast<uint32_t>(found >> 32);
      } else if (count > LIST / 2) {
        keep_largest(sm, count, p.top);
        if (tid < p.top) sm.list[tid] = sm.kept[tid];
        if (tid == 0) {
          sm.count = p.top;
          sm.threshold = static_cast<uint32_t>(sm.kept[p.top - 1] >> 32);
        }
      } else if (first && tid == 0 && count >= p.top) {
        sm.threshold = above + 1u;  // later logits have higher indices: those equal to it lose
      }
      __syncthreads();
      first = false;
    }
  }
  // ---- the block's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(st, shuffle(st, o));
  if (lane == 0) sm.stats[warp] = st;
  __syncthreads();
  st = sm.stats[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) join(st, sm.stats[w]);
  if (slice == 0) {
    const long long id = (p.id_bytes == 8 ? static_cast<const long long*>(p.ids)[row] : static_cast<const int*>(p.ids)[row]) - p.vocab_start;
    if (id >= 0 && id < p.vocab) st.x = Vec<T>::one(x0 + id);
  }
  if (p.top > 0) keep_largest(sm, min(sm.count, LIST), p.top);
  if (p.vocab_start != 0 && static_cast<int>(threadIdx.x) < p.top && sm.kept[tid] != 0ull) sm.kept[tid] -= static_cast<u64>(p.vocab_start);
  if (p.finish && p.slices == 1)
    write_results(p, row, st, sm.kept);
  else
    write_record(p, slice, row, st, sm.kept);
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

// Slices a row is cut into: enough blocks to fill the device, no slice shorter than a chunk.
int slices_of(int rows, int vocab) {
  const int chunks = (vocab + CHUNK - 1) / CHUNK;
  int s = (TARGET_BLOCKS + rows - 1) / rows;
  if (s > chunks) s = chunks;
  return s < 1 ? 1 : (s > MAX_SLICES ? MAX_SLICES : s);
}
size_t record_bytes(int rows, int top) { return static_cast<size_t>(rows) * (sizeof(Stats) + static_cast<size_t>(top) * sizeof(u64)); }

template <typename Kernel>
int launch(Kernel kernel, unsigned blocks, size_t smem, const Params& p, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;
  cfg.numAttrs = dependent_launch_attr(&attr);
  cfg.attrs = &attr;
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
  return static_cast<size_t>(slices_of(rows, vocab)) * record_bytes(rows, top);
}

static int run_logprobs(df::logprobs::Params& p, int fp32, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace df;
  using namespace df::logprobs;
  p.slices = slices_of(p.rows, p.vocab);
  p.part_bytes = record_bytes(p.rows, p.top);
  uint8_t* result = p.record;
  if (p.slices > 1) {
    const size_t need = p.slices * p.part_bytes;
    if (workspace == nullptr || workspace_bytes < need) return fail(DF_EINVAL, "workspace of %zu bytes is too small (need %zu)", workspace_bytes, need);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(DF_EINVAL, "the workspace must be 16-byte aligned");
    p.record = static_cast<uint8_t*>(workspace);
  }
  const unsigned blocks = static_cast<unsigned>(p.rows) * static_cast<unsigned>(p.slices);
  int rc = fp32 ? launch(token_logprobs_kernel<float>, blocks, 0, p, stream) : launch(token_logprobs_kernel<__nv_bfloat16>, blocks, 0, p, stream);
  if (rc != DF_OK || p.slices == 1) return rc;
  p.parts = p.slices;
  p.parts_in = static_cast<const uint8_t*>(workspace);
  p.record = result;
  return launch(token_logprobs_join_kernel, static_cast<unsigned>(p.rows), static_cast<size_t>(p.parts) * p.top * sizeof(u64), p, stream);
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
  return launch(token_logprobs_join_kernel, static_cast<unsigned>(rows), static_cast<size_t>(parts) * top * sizeof(u64), p, stream);
}
