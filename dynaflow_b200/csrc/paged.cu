// The bookkeeping of a key/value cache held in pages of 4-bit codes: the page plan of a step, and the
// launch that rotates a step's new tokens, quantises their keys and values and puts them into their slots.
//
// Cache layout (uint8 [pages, kv_heads, page_size * 136]): granules of 16 tokens, 2176 bytes each, so that
// any run of granules of one page and head is one contiguous copy for the attention launch:
//   [0, 1024)     key codes, 64 bytes a token; byte i holds dimensions 2i (low four bits) and 2i + 1
//   [1024, 1088)  key parameters, (scale, minimum) in bf16 a token
//   [1088, 2176)  the same for the values
// The four 16-byte chunks of token r are stored at places c ^ ((r >> 1) & 3): eight rows read at one chunk
// (the transposed matrix loads of the value product) then fall into eight different bank groups.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_util.h"
#include "paged_layout.cuh"
#include "ptx.cuh"

namespace df {
namespace paged {

// ------------------------------------------------------------------ page plan
//
// Request b needs need_b = ceil(len_b / page_size) pages and holds held_b. With exclusive prefix sums over
// the requests of the pages given back (back_b) and taken (more_b),
//   free'  = free list with the returned pages on top, the first of them uppermost
//   the i-th taken page = free'[count + returned - 1 - i]
// so a step that is taken back leaves the free list exactly as it was. Everything is whole numbers and
// depends on nothing but the inputs: no atomics, the same tables on every run.
//
// What bounds it: latency. One cluster of CTAs does it all in one launch (a few KB to some hundred KB of
// integers); every CTA repeats the prefix sums over the requests in its own shared memory, and the cluster
// barrier separates "everyone has read the old state" from "the new state is written". One CTA up to 4096 rows (256
// requests, a step and its return: 10.4 us), eight above (61 prompts, 125000 rows, and their return: 16.5 us).
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_REQUESTS = 8192;
constexpr int plan_smem(int requests) { return 3 * (requests + 1) * static_cast<int>(sizeof(int)); }  // the prefix sums

struct PlanParams {
  const int* lens;
  const int* fresh;
  int* table;
  int* held;
  int* free_pages;
  int* free_count;
  int* row_starts;
  int* slots;
  int* positions;
  int requests, max_pages, num_pages, rows, page_size, rows_per_request;
  Status* status;
};

// Prefix sums saturate: what lies past the last row of the caller's buffers only has to stay past it.
constexpr int PLAN_SUM_MAX = 1 << 30;
__device__ __forceinline__ int add_sat(int a, int b) { return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), static_cast<unsigned>(PLAN_SUM_MAX))); }

struct Request {
  int len, fresh, held, need;  // need: limited to what the table's row can hold
  bool too_long;
};

__device__ __forceinline__ Request load_request(const PlanParams& p, int b) {
  Request r;
  r.len = max(p.lens[b], 0);
  r.fresh = min(max(p.fresh[b], 0), r.len);
  r.held = min(max(p.held[b], 0), p.max_pages);
  const int need = r.len / p.page_size + (r.len % p.page_size != 0 ? 1 : 0);
  r.too_long = need > p.max_pages;
  r.need = r.too_long ? r.held : need;  // a request that outgrows its row keeps what it has
  return r;
}

// Largest i in [0, n) with start[i] <= x (start is non-decreasing, start[0] == 0).
__device__ __forceinline__ int find_last(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PlanParams p) {
  extern __shared__ int sums[];  // exclusive prefix sums: rows, pages taken, pages given back; requests + 1 each
  int* row_at = sums;
  int* more_at = row_at + p.requests + 1;
  int* back_at = more_at + p.requests + 1;
  __shared__ int warp_sum[3][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int worker = blockIdx.x * PLAN_THREADS + tid, workers = gridDim.x * PLAN_THREADS;
  const int count = min(max(p.free_count[0], 0), p.num_pages);
  auto everyone = [&]() {  // one cluster, or one CTA
    if (gridDim.x > 1) cluster_sync();
    else __syncthreads();
  };

  int carry[3] = {0, 0, 0};
  for (int b0 = 0; b0 < p.requests; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    int v[3] = {0, 0, 0};
    if (b < p.requests) {
      const Request r = load_request(p, b);
      v[0] = p.rows_per_request > 0 ? p.rows_per_request : min(r.fresh, PLAN_SUM_MAX);
      v[1] = max(r.need - r.held, 0);
      v[2] = max(r.held - r.need, 0);
      if (blockIdx.x == 0 && r.too_long) report(p.status, DF_ERR_PLAN, DF_WHERE_PLAN_TABLE, b);
      if (blockIdx.x == 0 && p.rows_per_request > 0 && r.fresh > p.rows_per_request) report(p.status, DF_ERR_PLAN, DF_WHERE_PLAN_ROWS, b);
    }
    int before[3];  // sum over the lanes before this one
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int inc = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc = add_sat(inc, up);
      }
      before[k] = __shfl_up_sync(0xffffffffu, inc, 1);
      if (lane == 0) before[k] = 0;
      if (lane == 31) warp_sum[k][warp] = inc;
    }
    __syncthreads();
    if (warp < 3) {
      int s = warp_sum[warp][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s = add_sat(s, up);
      }
      warp_sum[warp][lane] = s;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (b < p.requests) sums[k * (p.requests + 1) + b] = add_sat(carry[k], add_sat(warp > 0 ? warp_sum[k][warp - 1] : 0, before[k]));
      carry[k] = add_sat(carry[k], warp_sum[k][31]);
    }
    __syncthreads();
  }
  if (tid < 3) sums[tid * (p.requests + 1) + p.requests] = carry[tid];
  __syncthreads();
  const int taken = carry[1], returned = carry[2];
  const int top = count + returned;
  const bool enough = taken <= top;

  // pages given back: onto the free list
  for (int i = worker; i < returned; i += workers) {
    const int b = find_last(back_at, p.requests, i);
    const Request r = load_request(p, b);
    int* entry = p.table + static_cast<size_t>(b) * p.max_pages + r.need + (i - back_at[b]);
    const int to = top - 1 - i;
    if (to < p.num_pages) p.free_pages[to] = *entry;
    *entry = -1;
  }
  if (returned > 0) everyone();  // the list is complete

  // pages taken: into the tables
  if (enough)
    for (int i = worker; i < taken; i += workers) {
      const int b = find_last(more_at, p.requests, i);
      const Request r = load_request(p, b);
      const int from = top - 1 - i;
      p.table[static_cast<size_t>(b) * p.max_pages + r.held + (i - more_at[b])] = from < p.num_pages ? p.free_pages[from] : -1;
    }
  // Rows, four a thread: the request of the first one from the prefix sums, the others from there. A page that this launch
  // hands out is read from the list, not from the table (another thread may be writing that entry).
  const bool whole = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15u) == 0;
  for (int row0 = 4 * worker; row0 < p.rows; row0 += 4 * workers) {
    int b = p.rows_per_request > 0 ? min(row0 / p.rows_per_request, p.requests - 1) : find_last(row_at, p.requests, row0);
    Request r = load_request(p, b);
    int4 slot4, position4;
    int* slots = &slot4.x;
    int* positions = &position4.x;
    int column = -1, page = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = row0 + k;
      while (b + 1 < p.requests && row >= row_at[b + 1]) {
        r = load_request(p, ++b);
        column = -1;
      }
      const int i = row - row_at[b];
      int slot = -1, position = 0;
      if (i < (p.rows_per_request > 0 ? min(r.fresh, p.rows_per_request) : r.fresh)) {
        position = r.len - r.fresh + i;
        const int c = position / p.page_size;
        if (c != column) {
          column = c;
          page = -1;
          if (c < min(r.held, r.need)) {
            page = p.table[static_cast<size_t>(b) * p.max_pages + c];
          } else if (enough && c < r.need) {
            const int from = top - 1 - (more_at[b] + c - r.held);
            page = from < p.num_pages ? p.free_pages[from] : -1;
          }
        }
        if (page >= 0 && page < p.num_pages) slot = page * p.page_size + (position - c * p.page_size);
      }
      slots[k] = slot;
      positions[k] = position;
    }
    if (whole && row0 + 4 <= p.rows) {
      *reinterpret_cast<int4*>(p.slots + row0) = slot4;
      *reinterpret_cast<int4*>(p.positions + row0) = position4;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (row0 + k < p.rows) {
          p.slots[row0 + k] = slots[k];
          p.positions[row0 + k] = positions[k];
        }
    }
  }
  for (int b = worker; b <= p.requests; b += workers) p.row_starts[b] = row_at[b];
  everyone();  // every thread is done with the old state
  for (int b = worker; b < p.requests; b += workers) {
    const Request r = load_request(p, b);
    if (r.need <= r.held || enough) p.held[b] = r.need;
  }
  if (worker == 0) {
    p.free_count[0] = min(top, p.num_pages) - (enough ? taken : 0);
    if (!enough) report(p.status, DF_ERR_PLAN, DF_WHERE_PLAN_PAGES, static_cast<unsigned>(taken - top));
    if (carry[0] > p.rows && p.rows > 0) report(p.status, DF_ERR_PLAN, DF_WHERE_PLAN_ROWS, static_cast<unsigned>(carry[0] - p.rows));
  }
}

// ------------------------------------------------- rotary + quantise + append
//
// A row of the fused activation is [q heads | k heads | v heads] of 128 dimensions. Eight lanes share a head:
// lane l holds dimensions 8l..8l+7 and 64+8l..64+8l+7, so both elements of every rotated pair are in one
// thread, the row's minimum and maximum are three shuffle steps, and a thread's codes are two 32-bit words.
// A group of eight lanes goes through HEADS heads of one token with the angles in registers.
//
// Rounding points: the rotated value is rounded to bf16 (it is the bf16 key that is quantised); scale =
// bf16(max / 15 - min / 15); code = (x - min) / scale rounded to nearest even; every operation is the IEEE
// one (no contraction, no approximate division), so the codes are the same on any machine. The quotient is
// Markstein's: with r = 1 / scale correctly rounded and t = d r, t + (d - t scale) r in two fused operations is the
// correctly rounded d / scale (P. Markstein, Computation of elementary functions on the IBM RISC System/6000, 1990);
// scales so small or large that a step could leave the normal numbers take the division itself.
//
// Bound: HBM. Each row is read and written once, 136 bytes a key/value head go to the cache: 16384 rows of 32 + 2 x 8
// heads, 429 MB in 82 us = 5.2 TB/s. Two heads a group, four blocks a SM (one head: 89 us; four, two blocks: 86 us).
// Few rows are bound by the chain slot -> row -> angles: one head a group (256 rows: 3.5 us; two 4.1, four 4.3).
constexpr int APPEND_THREADS = 256;
constexpr int APPEND_FEW = 8;  // blocks a SM

struct AppendParams {
  const __nv_bfloat16* qkv;
  __nv_bfloat16* out;
  const int* positions;
  const int* slots;
  const float* angles;
  uint8_t* cache;
  long long ld_qkv, ld_out;
  int rows, q_heads, kv_heads, page_size, num_slots, num_positions;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void unpack8(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int APPEND_HEADS>
__global__ void __launch_bounds__(APPEND_THREADS, 4) rope_append_paged4_kernel(const AppendParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int l = threadIdx.x & 7;
  const int heads = p.q_heads + 2 * p.kv_heads;
  const int groups = (heads + APPEND_HEADS - 1) / APPEND_HEADS;
  const long long total = static_cast<long long>(p.rows) * groups;
  const long long first = (static_cast<long long>(blockIdx.x) * APPEND_THREADS + threadIdx.x) >> 3;
  const long long step = static_cast<long long>(gridDim.x) * (APPEND_THREADS / 8);
  const unsigned mask = 0xffu << (threadIdx.x & 24);  // the eight lanes of this head go through the loop together
  for (long long w = first; w < total; w += step) {
    const int row = static_cast<int>(w / groups);
    const int h0 = static_cast<int>(w - static_cast<long long>(row) * groups) * APPEND_HEADS;
    const int slot = p.slots[row], pos = p.positions[row];
    if (slot < 0 || slot >= p.num_slots || pos < 0 || pos >= p.num_positions) continue;  // padding: left as it is
    const __nv_bfloat16* src = p.qkv + row * p.ld_qkv;
    __nv_bfloat16* dst = p.out + row * p.ld_out;
    uint4 lo[APPEND_HEADS], hi[APPEND_HEADS];
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i)
      if (h0 + i < heads) {
        lo[i] = *reinterpret_cast<const uint4*>(src + (h0 + i) * 128 + l * 8);
        hi[i] = *reinterpret_cast<const uint4*>(src + (h0 + i) * 128 + 64 + l * 8);
      }
    float cs[8], sn[8];
    if (h0 < p.q_heads + p.kv_heads) {
      const float4* a = reinterpret_cast<const float4*>(p.angles + static_cast<size_t>(pos) * 128 + l * 8);
      *reinterpret_cast<float4*>(cs) = __ldg(a);
      *reinterpret_cast<float4*>(cs + 4) = __ldg(a + 1);
      *reinterpret_cast<float4*>(sn) = __ldg(a + 16);
      *reinterpret_cast<float4*>(sn + 4) = __ldg(a + 17);
    }
    const int page = slot / p.page_size, in_page = slot - page * p.page_size;
    const int r = in_page & (GRANULE - 1);
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i) {
      const int h = h0 + i;
      if (h >= heads) break;
      float x[16];
      unpack8(lo[i], x);
      unpack8(hi[i], x + 8);
      if (h < p.q_heads + p.kv_heads) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = x[j], v = x[j + 8];
          x[j] = __bfloat162float(__float2bfloat16_rn(__fsub_rn(__fmul_rn(u, cs[j]), __fmul_rn(v, sn[j]))));
          x[j + 8] = __bfloat162float(__float2bfloat16_rn(__fadd_rn(__fmul_rn(v, cs[j]), __fmul_rn(u, sn[j]))));
        }
      }
      if (h >= p.q_heads) {
        float low = x[0], high = x[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) {
          low = min_nan(low, x[j]);
          high = max_nan(high, x[j]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          low = min_nan(low, __shfl_xor_sync(mask, low, o));
          high = max_nan(high, __shfl_xor_sync(mask, high, o));
        }
        const __nv_bfloat16 scale_b = __float2bfloat16_rn(__fsub_rn(__fdiv_rn(high, 15.0f), __fdiv_rn(low, 15.0f)));
        const __nv_bfloat16 low_b = __float2bfloat16_rn(low);  // exact: the minimum is one of the bf16 values
        const float scale = __bfloat162float(scale_b);
        uint32_t word[2] = {0u, 0u};
        if (scale > 0x1p-100f && scale < 0x1p100f) {
          constexpr float ROUND = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, which stands in the low bits
          constexpr uint32_t ROUND_BITS = 0x4b400000u;
          const float inv = __frcp_rn(scale);
          word[0] = word[1] = 0u - ROUND_BITS * 0x11111111u;  // what the other bits add up to
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float d = __fsub_rn(x[j], low), t = __fmul_rn(d, inv);
            const float n = __fadd_rn(__fmaf_rn(__fmaf_rn(-t, scale, d), inv, t), ROUND);
            word[j >> 3] += __float_as_uint(n) << (4 * (j & 7));
            x[j] = __fmaf_rn(scale, __fsub_rn(n, ROUND), low);  // scale * code is exact: one rounding
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            // a row of equal values has scale 0 and codes 0; NaN fails the comparison and reaches the reader through the scale
            const float n = scale > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[j], low), scale)), 0.0f), 15.0f) : 0.0f;
            word[j >> 3] |= static_cast<uint32_t>(n) << (4 * (j & 7));
            x[j] = __fadd_rn(__fmul_rn(scale, n), low);
          }
        }
        const bool value = h >= p.q_heads + p.kv_heads;
        const int kvh = value ? h - p.q_heads - p.kv_heads : h - p.q_heads;
        uint8_t* half = p.cache + (static_cast<size_t>(page) * p.kv_heads + kvh) * p.page_size * TOKEN_BYTES +
                        static_cast<size_t>(in_page / GRANULE) * GRANULE_BYTES + (value ? HALF_GRANULE : 0);
        uint8_t* token = half + r * CODE_BYTES;
        *reinterpret_cast<uint32_t*>(token + (chunk_place(l >> 2, r) << 4) + (l & 3) * 4) = word[0];
        *reinterpret_cast<uint32_t*>(token + (chunk_place(2 + (l >> 2), r) << 4) + (l & 3) * 4) = word[1];
        if (l == 0) *reinterpret_cast<__nv_bfloat162*>(half + PARAM_OFFSET + r * 4) = __nv_bfloat162(scale_b, low_b);
      }
      *reinterpret_cast<uint4*>(dst + h * 128 + l * 8) = pack8(x);
      *reinterpret_cast<uint4*>(dst + h * 128 + 64 + l * 8) = pack8(x + 8);
    }
  }
}

}  // namespace paged
}  // namespace df

extern "C" int df_page_plan(const int* seq_lens_dev, const int* new_lens_dev, int* page_table_dev, int* page_counts_dev,
                            int* free_pages_dev, int* free_count_dev, int* row_starts_dev, int* slots_dev, int* positions_dev,
                            int requests, int max_pages, int num_pages, int rows, int page_size, int rows_per_request,
                            df_status_t* dev_status, void* stream) {
  using namespace df;
  using namespace df::paged;
  if (seq_lens_dev == nullptr || new_lens_dev == nullptr || page_table_dev == nullptr || page_counts_dev == nullptr ||
      free_pages_dev == nullptr || free_count_dev == nullptr || row_starts_dev == nullptr || dev_status == nullptr ||
      (rows > 0 && (slots_dev == nullptr || positions_dev == nullptr)))
    return fail(DF_EINVAL, "NULL pointer argument");
  if (requests <= 0 || max_pages <= 0 || num_pages <= 0 || rows < 0 || rows_per_request < 0)
    return fail(DF_EINVAL, "requests, max_pages and num_pages must be positive, rows and rows_per_request not negative");
  if (requests > PLAN_MAX_REQUESTS) return fail(DF_EUNSUPPORTED, "at most %d requests (got %d)", PLAN_MAX_REQUESTS, requests);
  if (page_size <= 0 || page_size % GRANULE != 0) return fail(DF_EINVAL, "page_size must be a positive multiple of %d (got %d)", GRANULE, page_size);
  if (static_cast<long long>(num_pages) * page_size > 0x7fffffffLL) return fail(DF_EUNSUPPORTED, "num_pages * page_size must stay below 2^31");
  if (static_cast<long long>(requests) * rows_per_request >= PLAN_SUM_MAX || rows >= PLAN_SUM_MAX ||
      static_cast<long long>(requests) * max_pages >= PLAN_SUM_MAX)
    return fail(DF_EUNSUPPORTED, "rows, requests * rows_per_request and requests * max_pages must stay below 2^30");
  PlanParams p;
  p.lens = seq_lens_dev;
  p.fresh = new_lens_dev;
  p.table = page_table_dev;
  p.held = page_counts_dev;
  p.free_pages = free_pages_dev;
  p.free_count = free_count_dev;
  p.row_starts = row_starts_dev;
  p.slots = slots_dev;
  p.positions = positions_dev;
  p.requests = requests;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.rows = rows;
  p.page_size = page_size;
  p.rows_per_request = rows_per_request;
  p.status = reinterpret_cast<Status*>(dev_status);
  // More than 48 KB (static part and all) a launch has to ask for: once a device, what the largest call needs.
  static bool attr_set[64] = {false};
  int dev = 0;
  (void)cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, plan_smem(PLAN_MAX_REQUESTS));
    if (e != cudaSuccess) return fail(DF_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int ctas = rows > 4 * PLAN_THREADS || requests > 2 * PLAN_THREADS ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(PLAN_THREADS, 1, 1);
  cfg.dynamicSmemBytes = plan_smem(requests);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = ctas > 1 ? attr : attr + 1;
  cfg.numAttrs = (ctas > 1 ? 1 : 0) + dependent_launch_attr(&attr[1]);
  e = cudaLaunchKernelEx(&cfg, page_plan_kernel, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(DF_ECUDA, "page plan launch: %s", cudaGetErrorString(e));
  }
  return DF_OK;
}

extern "C" int df_rope_append_paged4_bf16(const void* qkv, long long ld_qkv, void* out, long long ld_out, const int* positions_dev,
                                          const int* slots_dev, const float* angles_dev, int num_positions, int rows, int q_heads,
                                          int kv_heads, int head_dim, void* cache, int num_pages, int page_size, void* stream) {
  using namespace df;
  using namespace df::paged;
  if (qkv == nullptr || out == nullptr || positions_dev == nullptr || slots_dev == nullptr || angles_dev == nullptr || cache == nullptr)
    return fail(DF_EINVAL, "NULL pointer argument");
  if (head_dim != HEAD_DIM) return fail(DF_EUNSUPPORTED, "head_dim must be %d (got %d)", HEAD_DIM, head_dim);
  if (rows <= 0 || q_heads < 0 || kv_heads <= 0 || num_pages <= 0 || num_positions <= 0)
    return fail(DF_EINVAL, "rows, kv_heads, num_pages and num_positions must be positive");
  if (page_size <= 0 || page_size % GRANULE != 0) return fail(DF_EINVAL, "page_size must be a positive multiple of %d (got %d)", GRANULE, page_size);
  if (static_cast<long long>(num_pages) * page_size > 0x7fffffffLL) return fail(DF_EUNSUPPORTED, "num_pages * page_size must stay below 2^31");
  const long long cols = (static_cast<long long>(q_heads) + 2LL * kv_heads) * head_dim;
  if (ld_qkv < cols || ld_out < cols || (ld_qkv % 8) != 0 || (ld_out % 8) != 0)
    return fail(DF_EINVAL, "row strides must cover (q_heads + 2 kv_heads) * head_dim elements and be multiples of 8");
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache) |
        reinterpret_cast<uintptr_t>(angles_dev)) & 15u) != 0)
    return fail(DF_EINVAL, "qkv, out, the cache and the angles must be 16-byte aligned");
  const int sms = df_sm_count();
  if (sms <= 0) return fail(DF_ECUDA, "no CUDA device");
  AppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.positions = positions_dev;
  p.slots = slots_dev;
  p.angles = angles_dev;
  p.cache = static_cast<uint8_t*>(cache);
  p.ld_qkv = ld_qkv;
  p.ld_out = ld_out;
  p.rows = rows;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.num_slots = num_pages * page_size;
  p.num_positions = num_positions;
  // heads a group of eight lanes goes through: one when there are few rows
  const long long all = q_heads + 2LL * kv_heads, few = rows * all * 8 / APPEND_THREADS <= APPEND_FEW * sms;
  const long long groups = few ? all : (all + 1) / 2, blocks = (rows * groups * 8 + APPEND_THREADS - 1) / APPEND_THREADS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks < 16LL * sms ? blocks : 16LL * sms), 1, 1);
  cfg.blockDim = dim3(APPEND_THREADS, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;
  cfg.numAttrs = dependent_launch_attr(&attr);
  cfg.attrs = &attr;
  const cudaError_t e = few ? cudaLaunchKernelEx(&cfg, rope_append_paged4_kernel<1>, p) : cudaLaunchKernelEx(&cfg, rope_append_paged4_kernel<2>, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(DF_ECUDA, "paged rope + append launch: %s", cudaGetErrorString(e));
  }
  return DF_OK;
}
