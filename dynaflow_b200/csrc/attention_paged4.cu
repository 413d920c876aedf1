// Attention of a step's new tokens over a key/value cache held in pages of 4-bit codes.
//
// A key is s_k n + m_k (16 code values n, one scale s_k and one minimum m_k a token and head), a value likewise:
//   score(key) = scale * (s_k (q . n) + m_k sum(q))
//   out        = (sum p s_v n_v + sum p m_v) / sum p,       p = exp(score - reference)
// so both products run on the codes themselves and the parameters are two multiplications a score.
//
// The codes feed the matrix instructions without a conversion: a 16-bit half with a code in its low four bits
// is, read as fp16, the subnormal number n * 2^-24 (or 16 n * 2^-24 from the next four bits), which the
// matrix units take exactly. Eight codes cost four ANDs and a shift. The powers of two are put back with the
// scores and the result. Everything is summed in fp32; roundings to fewer bits:
//   * q is scaled by a power of two a row (its largest element to [2^14, 2^15)) and held in fp16: bf16 has 8
//     significant bits, fp16 11, so only elements below 2^-28 of the largest lose any;
//   * p s_v, scaled by a power of two so that it stays below 2^13, is held in fp16 for the value product: 2^-12
//     of its value, against the 2^-9 of the bf16 result.
//
// Both products are transposed, 16 keys on the rows of m16n8k16 and the query columns (new token x head of the
// group) on its 8 columns:  S^T[16 keys, 8] = K[16, 128] Q^T  and  O^T[128 dims, 8] += V^T[128, 16 keys] P^T.
// A thread's 16 bytes of a key row are four k-steps of A fragments whatever the order of the dimensions, as long
// as Q's fragments use the same order; the value fragments come from transposed 8x8 loads (a 16-bit unit is
// four dimensions of one key, its transposed pair the same four of the next key); P^T from the scores' layout by
// two 8x8 transposes in registers. (A decode step has one query row a head; at 8 columns the work is 1/16 of
// what the tensor pipe would do in the time the bytes take, so it stays on the warp-level instructions: operands
// come from registers, where the codes are unpacked, instead of going through shared or tensor memory again.)
//
// Work: the granules (16 tokens of a head) of all requests and heads in one list, cut evenly over all warps of
// the launch, whatever the lengths. A warp walks its part on its own: its lanes issue the copies of its ring
// (one contiguous 2176-byte bulk copy a granule), it keeps its own maximum, sum and O^T and never waits for
// another warp. A request and head that lies inside one warp's part is written to the output at once; one that
// is cut leaves a partial result a warp (at most two a warp), which a second launch merges in order.
//
// Bound: HBM, 136 bytes a key and head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_util.h"
#include "paged_layout.cuh"
#include "ptx.cuh"

namespace df {
namespace paged {

constexpr int WHERE_PAGED_ATTN = 51;
constexpr int ATTN_MIN_PART = 2;       // granules a warp takes at least
constexpr float RESCALE_LIMIT = 8.0f;  // the reference maximum moves when a score exceeds it by 2^8
constexpr int PARTIAL_FLOATS = HEAD_DIM + 2;

struct AttnParams {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const int* table;
  const int* seq_lens;
  const int* row_starts;  // may be null: request b is row b
  const int* new_lens;    // may be null: one row a request
  __nv_bfloat16* out;
  float* partial;         // [workers][2][columns][PARTIAL_FLOATS]
  long long* prefix;      // [requests + 1] granules before a request
  long long ld_q, ld_out;
  int rows, requests, max_pages, num_pages, page_granules;
  int q_heads, kv_heads, group, max_new;
  float scale_log2;
  unsigned long long timeout_ns;
  Status* status;
};

// What a request adds to the list of granules.
struct Weight {
  int len, fresh, granules, blocks;  // blocks: sets of columns (new token x head of the group) of a key/value head
  __device__ __forceinline__ int total(int kv_heads) const { return granules * blocks * kv_heads; }
};

template <int COLS>
__device__ __forceinline__ Weight request_weight(const AttnParams& p, int b) {
  Weight w;
  w.len = static_cast<int>(min(static_cast<long long>(max(p.seq_lens[b], 0)), static_cast<long long>(p.max_pages) * p.page_granules * GRANULE));
  w.fresh = p.new_lens != nullptr ? p.new_lens[b] : 1;
  const int served = min(w.fresh, p.max_new);
  w.granules = max((w.len + GRANULE - 1) / GRANULE, 1);  // a row without keys still has its output (zeros) to be written
  w.blocks = served > 0 ? (served * p.group + COLS - 1) / COLS : 0;
  return w;
}

// Worker w of `workers` takes granules [part_start(w), part_start(w + 1)).
__device__ __forceinline__ long long part_start(long long total, long long workers, long long w) { return total * w / workers; }
__device__ __forceinline__ long long part_of(long long total, long long workers, long long f) { return ((f + 1) * workers - 1) / total; }
__device__ __forceinline__ long long worker_count(long long total, long long most) {
  const long long n = total / ATTN_MIN_PART;
  return n < 1 ? 1 : (n < most ? n : most);
}

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 0xffu) - 127; }

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two pairs of codes of a 32-bit word as fp16 subnormals: n 2^-24 and 16 n 2^-24.
__device__ __forceinline__ uint32_t code_lo(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t code_hi(uint32_t w) { return w & 0x00f000f0u; }

__device__ __forceinline__ float sum_rows(float v) {  // over the 8 lanes that share lane % 4
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float max_rows(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

struct Desc {
  int b, hc, g, page_ok;  // request, key/value head * blocks + block, granule of the request, whether its page exists
};

template <int NT, int WARPS, int STAGES>
struct AttnShared {
  uint8_t ring[WARPS][STAGES][GRANULE_BYTES];
  Desc desc[WARPS][STAGES];
  uint64_t full[WARPS][STAGES];
  uint32_t abort;
};

// NT: sets of 8 columns a warp carries. One CTA an SM; the registers of a warp decide how many warps it has.
template <int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_paged4_kernel(const AttnParams p) {
  constexpr int COLS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<AttnShared<NT, WARPS, STAGES>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (lane < STAGES) mbar_init(&sm.full[warp][lane], 1);
  if (threadIdx.x == 0) sm.abort = 0u;
  mbar_fence_init();
  __syncthreads();
  const Deadline dl{globaltimer_ns() + p.timeout_ns, &sm.abort, p.status};
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- the whole list, and this warp's part of it
  long long total = 0;
  for (int b0 = 0; b0 < p.requests; b0 += 32) {
    const int b = b0 + lane;
    long long w = b < p.requests ? request_weight<COLS>(p, b).total(p.kv_heads) : 0;
    if (blockIdx.x == 0 && warp == 0) {
      long long inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (b < p.requests) p.prefix[b] = total + inc - w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    total += w;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.prefix[p.requests] = total;
  if (total == 0) return;
  const long long workers = worker_count(total, static_cast<long long>(gridDim.x) * WARPS);
  const long long worker = static_cast<long long>(warp) * gridDim.x + blockIdx.x;  // neighbours in the list are on different SMs
  if (worker >= workers) return;
  const long long f0 = part_start(total, workers, worker);
  const int count = static_cast<int>(part_start(total, workers, worker + 1) - f0);

  // first request of the part
  int cur_b = 0;
  long long rel0 = f0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const long long w = b < p.requests ? request_weight<COLS>(p, b).total(p.kv_heads) : 0;
    long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, inc > rel0);  // the request ends behind the start
    if (past != 0u) {
      const int src = __ffs(past) - 1;
      cur_b = b0 + src;
      rel0 -= __shfl_sync(0xffffffffu, inc - w, src);
      break;
    }
    rel0 -= __shfl_sync(0xffffffffu, inc, 31);
    if (b0 + 32 >= p.requests) return;  // cannot be: the part lies inside the list
  }
  int cur_rel = static_cast<int>(rel0);

  // ---- copies: lane i looks up the i-th of the next 32 granules; `issue(n)` starts the copy of granule n of the part
  Desc ahead{0, 0, 0, 0};
  const uint8_t* ahead_src = nullptr;
  auto look_up = [&](int n0) {
    int b = cur_b, rel = cur_rel + lane;
    Weight w = request_weight<COLS>(p, b);
    int all = w.total(p.kv_heads);
    while (rel >= all && b + 1 < p.requests) {
      rel -= all;
      w = request_weight<COLS>(p, ++b);
      all = w.total(p.kv_heads);
    }
    cur_b = __shfl_sync(0xffffffffu, b, 31);
    cur_rel = __shfl_sync(0xffffffffu, rel, 31) + 1;
    ahead.page_ok = 0;
    if (n0 + lane < count) {
      ahead.b = b;
      ahead.hc = rel / w.granules;
      ahead.g = rel - ahead.hc * w.granules;
      const int column = ahead.g / p.page_granules;
      const int page = column < p.max_pages && w.len > 0 ? p.table[static_cast<size_t>(b) * p.max_pages + column] : -1;
      if (page >= 0 && page < p.num_pages) {
        ahead.page_ok = 1;
        ahead_src = p.cache + ((static_cast<size_t>(page) * p.kv_heads + ahead.hc / w.blocks) * p.page_granules + (ahead.g - column * p.page_granules)) * GRANULE_BYTES;
      }
    }
  };
  auto issue = [&](int n) {  // by the lane that looked granule n up
    const int s = n % STAGES;
    sm.desc[warp][s] = ahead;
    if (ahead.page_ok) {
      mbar_expect_tx(&sm.full[warp][s], GRANULE_BYTES);
      bulk_load(sm.ring[warp][s], ahead_src, GRANULE_BYTES, &sm.full[warp][s]);
    } else {
      mbar_arrive(&sm.full[warp][s]);  // nothing to copy: its keys are masked
    }
  };
  look_up(0);
  if (lane < STAGES && lane < count) issue(lane);
  __syncwarp();

  // ---- state of the segment (one request, key/value head and set of columns)
  uint32_t qf[NT][16];                        // Q^T fragments: pair p of the 16 this thread's 32 dimensions make
  float c1[NT][2], c2[NT][2];                 // score = acc * c1 * s_k + m_k * c2, of columns 2t and 2t + 1
  int limit[NT][2];                           // keys a column sees
  float m[NT][2], l[NT][2], pm[NT][2];        // reference maximum (log2), sum p, sum p m_v (this thread's keys)
  float acc[NT][8][4];
  float v_scale = 1.0f, v_limit = -1.0f;      // p s_v is held times v_scale = 2^-v_exp; scales above v_limit move it
  int v_exp = -100;
  int seg_b = -1, seg_hc = -1, seg_first = 0, seg_last = 0, seg_granules = 0, min_limit = 0;

  auto begin = [&](const Desc& d) {
    seg_b = d.b;
    seg_hc = d.hc;
    seg_first = d.g;
    const Weight w = request_weight<COLS>(p, d.b);
    seg_granules = w.granules;
    const int kvh = d.hc / w.blocks, block = d.hc - kvh * w.blocks;
    const int served = min(w.fresh, p.max_new);
    const int row0 = p.row_starts != nullptr ? p.row_starts[d.b] : d.b;
    min_limit = w.len;
    v_scale = 1.0f;
    v_limit = -1.0f;
    v_exp = -100;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = block * COLS + nt * 8 + g;  // this lane's column of the B fragments
      const int j = c / p.group, row = row0 + j;
      const bool here = j < served && row >= 0 && row < p.rows;
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[i] = here ? *reinterpret_cast<const uint4*>(p.q + row * p.ld_q + (kvh * p.group + c - j * p.group) * HEAD_DIM + t * 32 + i * 8)
                      : make_uint4(0u, 0u, 0u, 0u);
      float x[32];
      float sum = 0.f, big = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w4[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[i * 8 + 2 * k] = __uint_as_float(w4[k] << 16);
          x[i * 8 + 2 * k + 1] = __uint_as_float(w4[k] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        sum += x[i];
        big = fmaxf(big, fabsf(x[i]));
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = max(min(exponent_of(big), 127), -100);
      const float up = pow2i(14 - e);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // word i of the 16 bytes, nibbles k and k + 4: dimensions 8i + k and 8i + k + 4 (odd k: 16 times the code)
          const float f = (k & 1) ? up * 0.0625f : up;
          const __half2 h = __floats2half2_rn(x[i * 8 + k] * f, x[i * 8 + k + 4] * f);
          qf[nt][i * 4 + k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      const float a = p.scale_log2 * pow2i(e + 10 > 127 ? 127 : e + 10);  // 2^24 of the codes, 2^(e - 14) of q
      const float b2 = p.scale_log2 * sum;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int cc = 2 * t + k;  // the columns of this thread's scores: held by lane group cc
        c1[nt][k] = __shfl_sync(0xffffffffu, a, cc * 4);
        c2[nt][k] = __shfl_sync(0xffffffffu, b2, cc * 4);
        const int jj = (block * COLS + nt * 8 + cc) / p.group;
        limit[nt][k] = jj < served ? min(w.len - w.fresh + jj + 1, w.len) : w.len;  // a column without a query is computed and dropped
        m[nt][k] = -INFINITY;
        l[nt][k] = 0.f;
        pm[nt][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[nt][i][k] = 0.f;
      min_limit = min(min_limit, min(limit[nt][0], limit[nt][1]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) min_limit = min(min_limit, __shfl_xor_sync(0xffffffffu, min_limit, o));
  };

  auto flush = [&]() {
    const Weight w = request_weight<COLS>(p, seg_b);
    const int kvh = seg_hc / w.blocks, block = seg_hc - kvh * w.blocks;
    const int served = min(w.fresh, p.max_new);
    const int row0 = p.row_starts != nullptr ? p.row_starts[seg_b] : seg_b;
    const bool began = seg_first == 0, whole = began && seg_last == seg_granules - 1;
    const float back = 16777216.0f * pow2i(v_exp);  // 2^24 of the codes
    float* slot = p.partial + (worker * 2 + (began ? 1 : 0)) * COLS * PARTIAL_FLOATS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float sum = sum_rows(l[nt][k]), add = sum_rows(pm[nt][k]);
        const int local = nt * 8 + 2 * t + k, c = block * COLS + local;
        const int j = c / p.group, row = row0 + j;
        const bool any = sum != 0.0f;  // no keys: zeros
        const float inv = whole ? 1.0f / sum : 1.0f;
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          // dimensions 32 c4 + 4 g .. + 3: rows g and g + 8 of m-tiles 2 c4 and 2 c4 + 1
          const float o0 = (acc[nt][2 * c4][k] * back + add) * inv, o1 = (acc[nt][2 * c4][2 + k] * (back * 0.0625f) + add) * inv;
          const float o2 = (acc[nt][2 * c4 + 1][k] * back + add) * inv, o3 = (acc[nt][2 * c4 + 1][2 + k] * (back * 0.0625f) + add) * inv;
          const int dim = 32 * c4 + 4 * g;
          if (whole) {
            if (j < served && row >= 0 && row < p.rows) {
              const __nv_bfloat162 lo = __floats2bfloat162_rn(any ? o0 : 0.f, any ? o1 : 0.f), hi = __floats2bfloat162_rn(any ? o2 : 0.f, any ? o3 : 0.f);
              *reinterpret_cast<uint2*>(p.out + row * p.ld_out + (kvh * p.group + c - j * p.group) * HEAD_DIM + dim) =
                  make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
          } else {
            *reinterpret_cast<float2*>(slot + local * PARTIAL_FLOATS + dim) = make_float2(o0, o1);
            *reinterpret_cast<float2*>(slot + local * PARTIAL_FLOATS + dim + 2) = make_float2(o2, o3);
          }
        }
        if (!whole && g == 0) {
          slot[local * PARTIAL_FLOATS + HEAD_DIM] = m[nt][k];
          slot[local * PARTIAL_FLOATS + HEAD_DIM + 1] = sum;
        }
      }
  };

  // lane's row address of the transposed loads: matrix lane / 8 of four (keys 0-7 / 8-15 of chunks c, c + 1)
  const int lm_row = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t lm_off = HALF_GRANULE + lm_row * CODE_BYTES + (chunk_place(lane >> 4, lm_row) << 4);
  const uint32_t k_off = g * CODE_BYTES + (chunk_place(t, g) << 4);

  bool ok = true;
  for (int n = 0; n < count; ++n) {
    const int s = n % STAGES;
    ok = mbar_wait(&sm.full[warp][s], (n / STAGES) & 1, dl, WHERE_PAGED_ATTN, static_cast<unsigned>(worker));
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const Desc d = sm.desc[warp][s];
    if (d.b != seg_b || d.hc != seg_hc) {
      if (seg_b >= 0) flush();
      begin(d);
    }
    seg_last = d.g;
    const uint8_t* st = sm.ring[warp][s];
    const uint32_t st_addr = smem_u32(st);
    const int key0 = d.g * GRANULE + g;  // this thread's keys: key0 and key0 + 8
    const bool edge = d.page_ok == 0 || (d.g + 1) * GRANULE > min_limit;

    // ---- S^T = K Q^T
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) sc[nt][k] = 0.f;
    {
      const uint4 ka = *reinterpret_cast<const uint4*>(st + k_off), kb = *reinterpret_cast<const uint4*>(st + k_off + 8 * CODE_BYTES);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a8 = wa[i] >> 8, b8 = wb[i] >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(sc[nt], code_lo(wa[i]), code_lo(wb[i]), code_hi(wa[i]), code_hi(wb[i]), qf[nt][4 * i], qf[nt][4 * i + 1]);
          mma_f16(sc[nt], code_lo(a8), code_lo(b8), code_hi(a8), code_hi(b8), qf[nt][4 * i + 2], qf[nt][4 * i + 3]);
        }
      }
    }
    // ---- parameters of the two keys
    float ks[2], km[2], vs[2], vm[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(st + PARAM_OFFSET + (g + 8 * r) * 4);
      const uint32_t vp = *reinterpret_cast<const uint32_t*>(st + HALF_GRANULE + PARAM_OFFSET + (g + 8 * r) * 4);
      ks[r] = __uint_as_float(kp << 16);
      km[r] = __uint_as_float(kp & 0xffff0000u);
      vs[r] = __uint_as_float(vp << 16);
      vm[r] = __uint_as_float(vp & 0xffff0000u);
    }
    bool seen[NT][4];
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = k >> 1, c = k & 1;
        sc[nt][k] = fmaf(sc[nt][k], c1[nt][c] * ks[r], c2[nt][c] * km[r]);
        seen[nt][k] = true;
        if (edge) {
          seen[nt][k] = d.page_ok != 0 && key0 + 8 * r < limit[nt][c];
          if (!seen[nt][k]) sc[nt][k] = -INFINITY;
        }
        move = move || sc[nt][k] > m[nt][c] + RESCALE_LIMIT;
      }
    float vmax = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      bool any = seen[0][2 * r] || seen[0][2 * r + 1];
      if (NT == 2) any = any || seen[NT - 1][2 * r] || seen[NT - 1][2 * r + 1];
      if (any) vmax = fmaxf(vmax, vs[r]);
    }
    move = move || vmax > v_limit;
    if (__any_sync(0xffffffffu, move)) {
      // new references: the largest score of each column so far, the power of two above the largest scale so far
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
      const int e_new = max(v_exp, min(max(exponent_of(vmax) + 1, -100), 126));
      const float beta = e_new == v_exp ? 1.0f : pow2i(max(v_exp - e_new, -126));
      v_exp = e_new;
      v_scale = pow2i(-e_new);
      v_limit = pow2i(min(e_new + 4, 127));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float top = fmaxf(m[nt][c], max_rows(fmaxf(sc[nt][c], sc[nt][2 + c])));
          const float alpha = top == -INFINITY ? 1.0f : ex2f(m[nt][c] - top);
          m[nt][c] = top;
          l[nt][c] *= alpha;
          pm[nt][c] *= alpha;
          const float both = alpha * beta;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[nt][i][c] *= both;
            acc[nt][i][2 + c] *= both;
          }
        }
    }
    // ---- P^T
    uint32_t pf[NT][2];
    const float vsn[2] = {vs[0] * v_scale, vs[1] * v_scale};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = k >> 1, c = k & 1;
        const float ref = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
        const float e = ex2f(sc[nt][k] - ref);
        l[nt][c] += e;
        if (edge) {  // what lies at a masked key (also NaN parameters) counts for nothing
          w[k] = seen[nt][k] ? e * vsn[r] : 0.f;
          pm[nt][c] += seen[nt][k] ? e * vm[r] : 0.f;
        } else {
          w[k] = e * vsn[r];
          pm[nt][c] = fmaf(e, vm[r], pm[nt][c]);
        }
      }
      const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
      pf[nt][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
      pf[nt][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t v[4];  // (keys 0-7, keys 8-15) of chunk 2 half, then of chunk 2 half + 1
      ldmatrix_x4_trans(st_addr + (lm_off ^ (half * 32)), v);
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const uint32_t x0 = v[2 * cc], x1 = v[2 * cc + 1], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(acc[nt][4 * half + 2 * cc], code_lo(x0), code_hi(x0), code_lo(x1), code_hi(x1), pf[nt][0], pf[nt][1]);
          mma_f16(acc[nt][4 * half + 2 * cc + 1], code_lo(y0), code_hi(y0), code_lo(y1), code_hi(y1), pf[nt][0], pf[nt][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    const int next = n + STAGES;
    if (next < count) {
      if ((next & 31) == 0) look_up(next);
      if (lane == (next & 31)) issue(next);
      __syncwarp();
    }
  }
  if (ok) {
    flush();
  } else {
    // a wait ran out: this warp's copies may still be on their way into shared memory
    const uint64_t t_stop = globaltimer_ns() + 2000000ull;
    while (globaltimer_ns() < t_stop) __nanosleep(1000);
  }
}

// Merges the partial results of requests and heads that were cut between warps, in the order of the warps:
// out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i. One warp a (request, new token, query head).
template <int COLS>
__global__ void attention_paged4_merge_kernel(const AttnParams p, int attn_ctas, int attn_warps) {
  grid_dependency_wait();
  grid_launch_dependents();
  const long long id = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (id >= static_cast<long long>(p.requests) * p.max_new * p.q_heads) return;
  const int b = static_cast<int>(id / (p.max_new * p.q_heads));
  const int rest = static_cast<int>(id - static_cast<long long>(b) * p.max_new * p.q_heads);
  const int j = rest / p.q_heads, head = rest - j * p.q_heads;
  const Weight w = request_weight<COLS>(p, b);
  if (j >= min(w.fresh, p.max_new)) return;
  const int row = (p.row_starts != nullptr ? p.row_starts[b] : b) + j;
  if (row < 0 || row >= p.rows) return;
  const int kvh = head / p.group, c = j * p.group + head - kvh * p.group;
  const int block = c / COLS, local = c - block * COLS;
  const long long total = p.prefix[p.requests];
  const long long workers = worker_count(total, static_cast<long long>(attn_ctas) * attn_warps);
  const long long first = p.prefix[b] + static_cast<long long>(kvh * w.blocks + block) * w.granules;
  const long long w0 = part_of(total, workers, first), w1 = part_of(total, workers, first + w.granules - 1);
  if (w0 == w1) return;  // written by the attention launch
  float best = -INFINITY;
  for (long long i = w0 + lane; i <= w1; i += 32)
    best = fmaxf(best, p.partial[((i * 2 + (i == w0 ? 1 : 0)) * COLS + local) * PARTIAL_FLOATS + HEAD_DIM]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  float o4[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (long long i = w0; i <= w1; ++i) {
    const float* s = p.partial + ((i * 2 + (i == w0 ? 1 : 0)) * COLS + local) * PARTIAL_FLOATS;
    const float f = s[HEAD_DIM] == -INFINITY ? 0.f : ex2f(s[HEAD_DIM] - best);
    const float2 a = *reinterpret_cast<const float2*>(s + lane * 4), c2 = *reinterpret_cast<const float2*>(s + lane * 4 + 2);
    sum += f * s[HEAD_DIM + 1];
    o4[0] += f * a.x;
    o4[1] += f * a.y;
    o4[2] += f * c2.x;
    o4[3] += f * c2.y;
  }
  const float inv = 1.0f / sum;
  const bool any = sum != 0.0f;  // no keys: zeros
  const __nv_bfloat162 lo = __floats2bfloat162_rn(any ? o4[0] * inv : 0.f, any ? o4[1] * inv : 0.f);
  const __nv_bfloat162 hi = __floats2bfloat162_rn(any ? o4[2] * inv : 0.f, any ? o4[3] * inv : 0.f);
  *reinterpret_cast<uint2*>(p.out + row * p.ld_out + head * HEAD_DIM + lane * 4) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

}  // namespace paged
}  // namespace df

namespace df {
namespace paged {

// Columns (new token x head of the group) of a key/value head that a warp carries: 8 with 16 warps an SM, or 16 with
// 8 warps. 16 read the cache once where 8 would read it twice; 8 or fewer columns have no use for the second set.
constexpr int ATTN_MAX_CTAS = 160;
constexpr int attn_columns(long long columns) { return columns <= 8 ? 8 : 16; }
constexpr int attn_warps(int cols) { return cols == 8 ? 16 : 8; }

template <int NT, int WARPS, int STAGES>
int launch_attention(const AttnParams& p, int grid, cudaStream_t s) {
  constexpr int COLS = 8 * NT;
  using Shared = AttnShared<NT, WARPS, STAGES>;
  static_assert(sizeof(Shared) <= 227 * 1024, "shared memory of an SM");
  static_assert(WARPS == attn_warps(COLS), "the merge launch counts the same workers");
  auto kernel = attention_paged4_kernel<NT, WARPS, STAGES>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
  if (e != cudaSuccess) return fail(DF_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(WARPS * 32, 1, 1);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  cfg.numAttrs = dependent_launch_attr(&attr);
  cfg.attrs = &attr;
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e == cudaSuccess) {
    const long long warps = static_cast<long long>(p.requests) * p.max_new * p.q_heads;
    cfg.gridDim = dim3(static_cast<unsigned>((warps * 32 + 255) / 256), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, attention_paged4_merge_kernel<COLS>, p, grid, WARPS);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(DF_ECUDA, "paged attention launch: %s", cudaGetErrorString(e));
  }
  return DF_OK;
}

}  // namespace paged
}  // namespace df

extern "C" size_t df_attention_paged4_workspace_bytes(int requests, int q_heads, int kv_heads, int max_new) {
  using namespace df::paged;
  if (requests <= 0 || q_heads <= 0 || kv_heads <= 0 || max_new <= 0 || q_heads % kv_heads != 0) return 0;
  const int cols = attn_columns(static_cast<long long>(max_new) * (q_heads / kv_heads));
  const size_t partial = static_cast<size_t>(ATTN_MAX_CTAS) * attn_warps(cols) * 2 * cols * PARTIAL_FLOATS * sizeof(float);
  return partial + ((static_cast<size_t>(requests) + 1) * sizeof(long long) + 15) / 16 * 16;
}

extern "C" int df_attention_paged4_bf16(const void* q, long long ld_q, const void* cache, const int* page_table_dev,
                                        const int* seq_lens_dev, const int* row_starts_dev, const int* new_lens_dev, void* out,
                                        long long ld_out, int rows, int requests, int max_pages, int num_pages, int page_size,
                                        int q_heads, int kv_heads, int head_dim, int max_new, float scale, void* workspace,
                                        size_t workspace_bytes, int max_ctas, df_status_t* dev_status, void* stream) {
  using namespace df;
  using namespace df::paged;
  if (q == nullptr || cache == nullptr || page_table_dev == nullptr || seq_lens_dev == nullptr || out == nullptr || workspace == nullptr ||
      dev_status == nullptr)
    return fail(DF_EINVAL, "NULL pointer argument");
  if ((row_starts_dev == nullptr) != (new_lens_dev == nullptr)) return fail(DF_EINVAL, "row_starts and new_lens come together");
  if (new_lens_dev == nullptr && (max_new != 1 || rows < requests))
    return fail(DF_EINVAL, "without new_lens every request has one row: max_new must be 1 and rows at least requests");
  if (head_dim != HEAD_DIM) return fail(DF_EUNSUPPORTED, "head_dim must be %d (got %d)", HEAD_DIM, head_dim);
  if (rows <= 0 || requests <= 0 || max_pages <= 0 || num_pages <= 0 || max_new <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0)
    return fail(DF_EINVAL, "rows, requests, max_pages, num_pages, max_new and the head counts must be positive, q_heads a multiple of kv_heads");
  if (page_size <= 0 || page_size % GRANULE != 0) return fail(DF_EINVAL, "page_size must be a positive multiple of %d (got %d)", GRANULE, page_size);
  const long long columns = static_cast<long long>(max_new) * (q_heads / kv_heads);
  const int cols = attn_columns(columns);
  if (static_cast<long long>(max_pages) * page_size > 0x7fffffffLL)
    return fail(DF_EUNSUPPORTED, "max_pages * page_size must stay below 2^31");
  const long long longest = (static_cast<long long>(max_pages) * (page_size / GRANULE)) * kv_heads;
  if (columns > 0x7fffffffLL || longest > 0x7fffffffLL / ((columns + cols - 1) / cols))
    return fail(DF_EUNSUPPORTED, "max_pages * page_size / 16 * kv_heads * ceil(max_new * group / %d) must stay below 2^31", cols);
  if (static_cast<long long>(requests) * max_new > 0x7fffffffLL / q_heads / 4)
    return fail(DF_EUNSUPPORTED, "requests * max_new * q_heads must stay below 2^29");
  if (ld_q < static_cast<long long>(q_heads) * HEAD_DIM || ld_out < static_cast<long long>(q_heads) * HEAD_DIM || (ld_q % 8) != 0 || (ld_out % 8) != 0)
    return fail(DF_EINVAL, "row strides must cover the heads and be multiples of 8 elements");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u) != 0)
    return fail(DF_EINVAL, "q, the cache, out and the workspace must be 16-byte aligned");
  if (!(scale > 0.0f)) return fail(DF_EINVAL, "scale must be positive");
  const size_t need = df_attention_paged4_workspace_bytes(requests, q_heads, kv_heads, max_new);
  if (workspace_bytes < need) return fail(DF_EINVAL, "workspace of %zu bytes is too small (need %zu)", workspace_bytes, need);
  const int sms = df_sm_count();
  if (sms <= 0) return fail(DF_ECUDA, "no CUDA device");
  int grid = sms < ATTN_MAX_CTAS ? sms : ATTN_MAX_CTAS;
  if (max_ctas > 0 && max_ctas < grid) grid = max_ctas;
  AttnParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.cache = static_cast<const uint8_t*>(cache);
  p.table = page_table_dev;
  p.seq_lens = seq_lens_dev;
  p.row_starts = row_starts_dev;
  p.new_lens = new_lens_dev;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.prefix = static_cast<long long*>(workspace);
  // the partial results start at a multiple of 16 bytes behind the prefix sums
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ((static_cast<size_t>(requests) + 1) * sizeof(long long) + 15) / 16 * 16);
  p.ld_q = ld_q;
  p.ld_out = ld_out;
  p.rows = rows;
  p.requests = requests;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.page_granules = page_size / GRANULE;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.max_new = max_new;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.timeout_ns = timeout_ns();
  p.status = reinterpret_cast<Status*>(dev_status);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cols == 8 ? launch_attention<1, 16, 6>(p, grid, s) : launch_attention<2, 8, 12>(p, grid, s);
}
