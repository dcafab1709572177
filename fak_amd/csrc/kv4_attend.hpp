// kv4_attend.hpp — what the kernels of attention over the 4-bit cache (kv4_attention.hip, kv4_prefill.hip) share:
// the call, the requests as they walk them, the unpack of the codes.
#pragma once

#include "kernels.hpp"
#include "kv4.hpp"

namespace fhip {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int kStep = 64;   // keys of a wave's step: four granules
constexpr double kLog2e = 1.44269504088896340736;
// Weights are e^(..) 2^14: as two f16 terms they then keep 22 bits, and 2^-38 of the largest below, so that hundreds of
// thousands of small ones add up right. Both terms are cut toward zero: where a score of 2^25 and more rounds the 14 to
// 16, the first is f16's largest number and the second the rest, no infinity. (Terms for what two leave of the
// smaller weights: prompts 330 us where they take 204, 32 single tokens 19 and 16.)
constexpr float kBias = 14.f;

struct Attend {
  const uint8_t *cache;
  const float *q;
  float *out;
  const int32_t *start, *lens, *table;
  int requests, tokens, heads, heads_kv, pages, shift, cols, ldq, window;
  float kh, kl;  // scale * 4 * log2 e = 2^ke (kh + kl), kh in [1, 2)
  int ke;
  int per_request;  // Split entries are by item, so many for each request; 0: by their first workgroup
  int64_t least_rows, most_rows;  // of the requests (tokens times heads of a kv head) that a launch takes
  bool zero_rest;                 // it clears the rows past the last request
};

// An item that several workgroups worked on, `first` to `last`; rows 0: none.
struct Split {
  int rows, first, last, token0, kvh, row0;
};

// Entry i (uniform) of what no kernel here writes, by the scalar unit: a vector load would wait in the
// queue of the cache's.
__device__ inline int32_t uniform(const int32_t *p, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t *)(uintptr_t)p)[i];
}

__device__ inline h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ inline uint32_t as_u(h2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight codes to f16: nibbles p and p + 4 of x are the pair p. Each is put into mantissa bits 6..9 of
// 16.0, which makes it 16 + c, and (16 + c) s - 24 s = (c - 8) s is one exact packed fma. (24 s is finite up to
// the largest scale; the nibble in place for one pair, in 64.0, would need 72 s.)
struct Unpack {
  uint32_t mask, magic;
  __device__ Unpack() : mask(in_reg(0x03C003C0u)), magic(in_reg(0x4C004C00u)) {}
  __device__ f16x8 operator()(uint32_t x, const h2 s0, const h2 s1, const h2 s2, const h2 s3, const h2 c0, const h2 c1,
                              const h2 c2, const h2 c3) const {
    u32x4 v;
    v[0] = as_u(__builtin_elementwise_fma(as_h2(((x << 6) & mask) | magic), s0, c0));
    v[1] = as_u(__builtin_elementwise_fma(as_h2(((x << 2) & mask) | magic), s1, c1));
    v[2] = as_u(__builtin_elementwise_fma(as_h2(((x >> 2) & mask) | magic), s2, c2));
    v[3] = as_u(__builtin_elementwise_fma(as_h2(((x >> 6) & mask) | magic), s3, c3));
    return __builtin_bit_cast(f16x8, v);
  }
};

// a / b of positive numbers: by f32 below 2^22 (its quotient is then at most one off), else by f64. The integer
// division that the compiler makes is many times as long.
__device__ inline int divide(int a, int b) {
  int q = (a | b) >> 22 == 0 ? (int)((float)a * __builtin_amdgcn_rcpf((float)b)) : (int)((double)a / (double)b);
  q -= (int64_t)q * b > a;
  return q + ((int64_t)(q + 1) * b <= a);
}

// a / b for lanes, b uniform: by f32 where `small` (all a below 2^22).
__device__ inline int divide_lanes(int a, int b, bool small) {
  if (!small) return a / b;
  int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
  q -= q * b > a;
  return q + ((q + 1) * b <= a);
}

// The first key that position p sees; p may lie below 0 and the window be as large as an int holds.
__device__ inline int first_key(int p, int window) { return window && p >= window ? p - window + 1 : 0; }

// Bits lo to hi of 64, which may lie outside.
__device__ inline uint64_t keys_between(int lo, int hi) {
  lo = max(lo, 0), hi = min(hi, 63);
  return lo <= hi ? (~0ull >> (63 - hi)) & (~0ull << lo) : 0;
}

// A request as a kernel walks it: row tiles of RPT rows, for each kv head an item of nt steps from tile0;
// an item is worth a unit for every PER steps and COST more. A launch's units are below 2^31 (its host side
// sees to that).
struct Req {
  int len, n, token0, nt, tile0, row_tiles, per_item, units;
};

template <int RPT, int PER, int COST>
__device__ inline Req request(const Attend &a, int begin, int end, int len) {
  Req q;
  q.token0 = min(max(begin, 0), a.tokens);
  q.n = min(max(end, q.token0), a.tokens) - q.token0;
  const int64_t rows = (int64_t)q.n * (a.heads / a.heads_kv);
  if (rows < a.least_rows || rows > a.most_rows) q.n = 0;  // another launch's
  const int64_t room = (int64_t)a.cols << a.shift;
  q.len = (int)min((int64_t)max(len, 0), room);
  const int p0 = q.len - q.n;  // the first token's position, below 0 where it sees nothing
  const int lo = first_key(p0, a.window);
  q.tile0 = min(lo, max(q.len - 1, 0)) / kStep;
  q.nt = max(q.len - 1, 0) / kStep - q.tile0 + 1;  // one step, all of it masked, where there is no key
  q.row_tiles = ((int64_t)q.n * (a.heads / a.heads_kv) + RPT - 1) / RPT;
  q.per_item = (q.nt + PER - 1) / PER + COST;
  q.units = q.row_tiles * a.heads_kv * q.per_item;
  return q;
}

// Whether the requests' first tokens fall here. Where none does, all requests have no more tokens than the call, and
// their units stay below 2^31; else a launch takes none of them, since units past that would name items that are not.
__device__ inline bool falling(const Attend &a, int r) { return a.start[r + 1] < a.start[r]; }

// The inclusive sum over the lanes of a wave; the largest of them of numbers not below 0.
#define FHIP_SCAN(f)                                                                                                          \
  f(0x111, 0xF) f(0x112, 0xF) f(0x114, 0xF) f(0x118, 0xF) /* rows of 16: shifts by 1, 2, 4, 8 */                              \
      f(0x142, 0xA) f(0x143, 0xC)                         /* then the rows' last lanes onto the rows behind */
__device__ inline int32_t sum_lanes(int32_t x) {
#define FHIP_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, false);
  FHIP_SCAN(FHIP_STEP)
#undef FHIP_STEP
  return x;
}
__device__ inline int32_t max_lanes(int32_t x) {
#define FHIP_STEP(ctrl, rows) x = max(x, __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, false));
  FHIP_SCAN(FHIP_STEP)
#undef FHIP_STEP
  return __builtin_amdgcn_readlane(x, 63);
}
#undef FHIP_SCAN

// The sum over a workgroup of W waves of `mine`; *before what the threads before this one have.
template <int W>
__device__ inline int sum_before(int mine, int *scan, int *before) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int incl = sum_lanes(mine);
  if (lane == 63) scan[wave] = incl;
  __syncthreads();
  int total = 0, b = incl - mine;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) b += scan[w];
    total += scan[w];
  }
  *before = b;
  return total;
}

// Zeros for tokens past the last request.
__device__ inline void clear_rest(const Attend &a, int D) {
  const int64_t row = (int64_t)a.heads * D, from = min(max(a.start[a.requests], 0), a.tokens) * row;
  for (int64_t i = from + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < a.tokens * row; i += (int64_t)gridDim.x * blockDim.x) a.out[i] = 0.f;
}

// The granule that holds position `key` of a request, by the id of its page (held inside the cache).
__device__ inline const uint8_t *granule_of(const Attend &a, int page, int key, int kvh, int granule_bytes) {
  const uint32_t id = min(max(page, 0), a.pages - 1), in = ((uint32_t)key & ((1u << a.shift) - 1)) >> 4;
  const uint32_t per = (uint32_t)granule_bytes << (a.shift - 4);  // bytes of a page and kv head
  return a.cache + (uint64_t)(id * (uint32_t)a.heads_kv + kvh) * per + in * (uint32_t)granule_bytes;
}

// Many query rows (kv4_prefill.hip).
int kv4_prefill(const char *who, int D, const Attend &a);

}  // namespace fhip
