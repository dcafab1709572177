// logprobs.hip — log probabilities of given tokens, the distribution's entropy and its top alternatives
// (fhip_logprobs_f32), each logit read once.
//
// Over a row x of n logits, with m = max x:
//   S = sum e^(x_i - m), W = sum (x_i - m) e^(x_i - m)
//   log p_i = x_i - m - log S        H = -sum p log p = log S - W / S
// S, W and m run together in f32: a lane keeps its own m and rescales (S, W) when it grows,
//   S <- S f, W <- f (W + (m - m') S), f = e^(m - m'),
// and lanes, waves and parts of a row join by the same rule in f64. A step's eight terms are summed by themselves first,
// and what follows from S and W is formed in f64: within 3e-8 of the exact log probabilities in the 2-norm and 5e-8 of
// the entropies (511 rows of 152,064), f32's own rounding being 2.6e-8 and 2.9e-8. (All in f32, 4.8e-8 and 1.2e-7, took
// the same time; log2 e in two terms costs 1%.) A masked logit (-inf) adds nothing to
// either sum. A row with a NaN or +inf, or with nothing above -inf, has no distribution.
//
// The alternatives: the order is by value, the lower id first among equals, and (value, ~id) in one
// 64-bit key makes that a total order. A wave keeps candidates above a threshold in LDS. The first
// threshold is a value that `top` lanes' largest reach; when a few times `top` have come together, each
// counts those above it, the first `top` stay, and the last of them is the new threshold, which the
// workgroup's other waves then use too. Later values of a wave have higher ids than it holds, so only
// greater ones can enter.
//
// One row is bound by latency: it is cut over many workgroups, and the last of them to be done joins the
// parts in the same launch. Many rows are bound by memory. 511 rows of 152,064: 66 us, 4.7 TB/s; one row 9.3 us, of
// which the launch is 2.5, a part's chain (load, sums, candidates, their order) 3.5 and the joining part's 3.3.
#include <cstdint>

#include "kernels.hpp"

using namespace fhip;

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMaxTop = 64;
constexpr int kCap = 128;            // candidates a wave holds; 64 stay free for one more append
constexpr int kStep = 512;           // values of a wave's step, eight a lane
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLow = -3.402823466e38f;  // a maximum before the first value: the lowest finite one
constexpr int kMaxVocab = 1 << 24;

typedef uint64_t u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // one load wherever a row begins

__device__ inline float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Ascending whole numbers for ascending floats; -0 and +0 are one value.
__device__ inline uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float order_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ inline u64 make_key(float v, uint32_t id) { return (u64)order_bits(v) << 32 | (0xFFFFFFFFu - id); }
__device__ inline float key_value(u64 k) { return order_value((uint32_t)(k >> 32)); }
__device__ inline uint32_t key_id(u64 k) { return 0xFFFFFFFFu - (uint32_t)k; }

// What lanes, waves and parts join: few additions of large numbers, in f64, since in f32 they would be most of the error.
struct Sums {
  float m;
  double s, w;
};

// The same by a maximum m that is no smaller. s = 0 also where nothing was seen: then all is 0 whatever m is.
__device__ inline Sums below(const Sums a, float m) {
  const float d = fmaxf(a.m - m, -1e30f);
  const double f = exp_fast(d);
  return {m, a.s * f, f * (a.w + d * a.s)};
}

// f over all lanes, in each of them: by rotations of 16 lanes, then by swaps of their groups.
template <int N>
__device__ inline uint32_t rotate(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xF, 0xF, true);
}
template <int N>
__device__ inline float rotate(float x) { return __uint_as_float(rotate<N>(__float_as_uint(x))); }
template <int N>
__device__ inline double rotate(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)rotate<N>((uint32_t)(u >> 32)) << 32 | rotate<N>((uint32_t)u));
}
struct Both {
  uint64_t a, b;
};
template <int N>
__device__ inline Both swapped(uint64_t x) {
  auto swap = [](uint32_t v) {
    if constexpr (N == 16) return __builtin_amdgcn_permlane16_swap(v, v, false, false);
    else return __builtin_amdgcn_permlane32_swap(v, v, false, false);
  };
  const auto lo = swap((uint32_t)x), hi = swap((uint32_t)(x >> 32));
  return {(uint64_t)hi[0] << 32 | lo[0], (uint64_t)hi[1] << 32 | lo[1]};
}
template <typename T, typename F>
__device__ inline T over_wave(T x, F f) {
  x = f(x, rotate<1>(x));
  x = f(x, rotate<2>(x));
  x = f(x, rotate<4>(x));
  x = f(x, rotate<8>(x));
  auto of = [](uint64_t u) {
    if constexpr (sizeof(T) == 8) return __builtin_bit_cast(double, u);
    else return __uint_as_float((uint32_t)u);
  };
  auto bits = [](T v) {
    if constexpr (sizeof(T) == 8) return __builtin_bit_cast(uint64_t, v);
    else return (uint64_t)__float_as_uint(v);
  };
  const Both p = swapped<16>(bits(x));
  x = f(of(p.a), of(p.b));
  const Both q = swapped<32>(bits(x));
  return f(of(q.a), of(q.b));
}
__device__ inline Sums join_wave(Sums a) {
  auto add = [](double x, double y) { return x + y; };
  a = below(a, over_wave(a.m, [](float x, float y) { return fmaxf(x, y); }));
  return {a.m, over_wave(a.s, add), over_wave(a.w, add)};
}

// The inclusive sum over the lanes up to this one.
__device__ inline int scan_lanes(int v) {
#define FHIP_SCAN(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false);
  FHIP_SCAN(0x111, 0xF) FHIP_SCAN(0x112, 0xF) FHIP_SCAN(0x114, 0xF) FHIP_SCAN(0x118, 0xF)  // rows of 16: shifts by 1, 2, 4, 8
  FHIP_SCAN(0x142, 0xA) FHIP_SCAN(0x143, 0xC)  // then the rows' last lanes onto the rows behind
#undef FHIP_SCAN
  return v;
}

// A value that at least `top` of the lanes' reach: the least of the ceil(top / 4) largest of each 16
// lanes. Ranks go by rotating the 16 (a rank over all 64 by reading each lane took 3,600 cycles).
__device__ inline uint32_t edge_of(uint32_t mine, int top) {
  int rank = 0;
#define FHIP_ROTATE(n) rank += rotate<n>(mine) > mine;
  FHIP_ROTATE(1) FHIP_ROTATE(2) FHIP_ROTATE(3) FHIP_ROTATE(4) FHIP_ROTATE(5) FHIP_ROTATE(6) FHIP_ROTATE(7) FHIP_ROTATE(8)
  FHIP_ROTATE(9) FHIP_ROTATE(10) FHIP_ROTATE(11) FHIP_ROTATE(12) FHIP_ROTATE(13) FHIP_ROTATE(14) FHIP_ROTATE(15)
#undef FHIP_ROTATE
  uint32_t e = 4 * rank < top ? mine : 0xFFFFFFFFu;
  e = min(e, rotate<1>(e));
  e = min(e, rotate<2>(e));
  e = min(e, rotate<4>(e));
  e = min(e, rotate<8>(e));
  const auto a = __builtin_amdgcn_permlane16_swap(e, e, false, false);
  e = min(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(e, e, false, false);
  return min(b[0], b[1]);
}

// The candidates of one wave. A wave's LDS accesses are in order; the fences keep the compiler's so.
struct Best {
  u64 *buf;  // kCap of them and eight more
  int count, top;
  float thr;
  __device__ void fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }
  // The first min(top, count) by rank, in order; the last of them is the threshold once there are `top`.
  __device__ void keep() {
    const int lane = threadIdx.x & 63;
    if (lane < 8) buf[count + lane] = 0;
    fence();
    const u64 a = lane < count ? buf[lane] : 0, b = lane + 64 < count ? buf[lane + 64] : 0;
    int ra = 0, rb = 0;
#pragma unroll 1
    for (int i = 0; i < count; i += 8) {
      u64 k[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = buf[i + j];
#pragma unroll
      for (int j = 0; j < 8; ++j) ra += k[j] > a;
      if (count > 64) {
#pragma unroll
        for (int j = 0; j < 8; ++j) rb += k[j] > b;
      }
    }
    fence();
    if (a && ra < top) buf[ra] = a;
    if (b && rb < top) buf[rb] = b;
    fence();
    if (count >= top) {
      count = top;
      thr = fmaxf(thr, key_value(buf[top - 1]));
    }
  }
  __device__ void add(bool take, u64 key) {
    if (count > kCap - 64) keep();
    const u64 mask = __ballot(take);
    if (take) buf[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
    count += __popcll(mask);
  }
};

// Output of one row from its sums and its sorted candidates (the first wave of a workgroup).
struct Out {
  const float *x;
  const int32_t *tokens;
  float *logp, *entropy, *top_logp;
  int32_t *top_ids;
  int n, top;
  int64_t ld;
};

__device__ inline void finish(const Out &o, int row, float chosen, const Sums t, const u64 *best, int have) {
  const int lane = threadIdx.x & 63;
  const bool fine = t.s > 0. && t.s < __builtin_inf() && t.m < __builtin_inff();  // NaN fails too
  const float nan = __builtin_nanf("");
  // log S by its power of two and a mantissa of 1 +- 0.3, and all that follows in f64, rounded once: differences of
  // numbers of ten and more would each lose 2^-21 in f32.
  int k;
  double mant = frexp(t.s, &k);
  if (mant < 0.70710678) mant *= 2., --k;
  const float near = (float)mant;
  const double ls = k * 0.69314718055994530942 + ((double)logf(near) + (double)((float)(mant - near) / near)), m = t.m;
  if (lane == 0) {
    if (o.entropy) o.entropy[row] = fine ? (float)(ls - t.w / t.s) : nan;
    if (o.logp) o.logp[row] = fine ? (float)(chosen - m - ls) : nan;
  }
  if (lane < o.top) {
    const bool in = fine && lane < have;
    const u64 key = in ? best[lane] : 0;
    o.top_logp[(size_t)row * o.top + lane] = in ? (float)(key_value(key) - m - ls) : nan;
    o.top_ids[(size_t)row * o.top + lane] = in ? (int32_t)key_id(key) : -1;
  }
}

// One part of a row (grid.x parts, grid.y rows). The waves take steps of 512 values in turn; the part that
// is the last of its row to be done joins them all (with one part, at once).
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Out o, Sums *part_sums, u64 *part_best, uint32_t *done, int per) {
  __shared__ __align__(16) u64 buf[kWaves][kCap + 8];
  __shared__ float shared_thr;
  __shared__ Sums wsum[kWaves];
  __shared__ int wcount[kWaves];
  __shared__ uint32_t lane_max[kThreads];
  __shared__ uint32_t is_last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y, parts = gridDim.x, part = blockIdx.x;
  const int i0 = part * per, i1 = part == parts - 1 ? o.n : i0 + per;
  const float *x = o.x + row * o.ld;
  // The token's logit (NaN for no id of the vocabulary), asked for before all else: at the end it would be
  // two loads in turn.
  float chosen = __builtin_nanf("");
  if (o.logp) {
    const int id = o.tokens[row];
    if (id >= 0 && id < o.n) chosen = x[id];
  }
  float tm = kLow, ts = 0.f, tw = 0.f;
  Best best{buf[wave], 0, o.top, -__builtin_inff()};

  // Two runs of four values a lane; what lies behind the end counts as -inf and is no candidate.
  typedef float f32x8 __attribute__((ext_vector_type(8)));
  const float low = -__builtin_inff();
  auto load = [&](int at) {
    f32x8 v = {low, low, low, low, low, low, low, low};
    if (at + kStep <= i1) {
      const f32x4u p = *reinterpret_cast<const f32x4u *>(x + at + 4 * lane), q = *reinterpret_cast<const f32x4u *>(x + at + 256 + 4 * lane);
      v = f32x8{p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
    } else if (at < i1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = at + 256 * (j >> 2) + 4 * lane + (j & 3);
        if (i < i1) v[j] = x[i];
      }
    }
    return v;
  };
  constexpr int kTurn = kWaves * kStep;
  int at = i0 + wave * kStep;
  f32x8 v = load(at), v1 = load(at + kTurn);  // two steps under way beside the one worked on
  bool first = true;
  do {
    const f32x8 v2 = load(at + 2 * kTurn);
    float mx = fmaxf(v[0], v[1]);
#pragma unroll
    for (int j = 2; j < 8; ++j) mx = fmaxf(mx, v[j]);
    const float m = fmaxf(tm, mx), d0 = fmaxf(tm - m, -1e30f), f = exp_fast(d0);
    tw = f * (tw + d0 * ts);
    ts *= f;
    tm = m;
    float es = 0.f, ws = 0.f;  // a step's own sums first: beside a sum that holds the maximum, 1, each would lose 2^-24
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[j] - m, e = exp_fast(d);
      es += e;
      ws += fmaxf(d, -1e30f) * e;
    }
    ts += es;
    tw += ws;
    if (o.top) {
      float edge;
      if (first) {
        // What follows has higher ids than all of the first steps': only what exceeds the edge can enter.
        // The largest of a lane and the other waves' same: some 30 of 2,048 values reach the
        // edge of 20 then; the greatest of the waves' own edges let 100 in.
        lane_max[threadIdx.x] = order_bits(mx);
        __syncthreads();
        const uint32_t a = max(lane_max[lane], lane_max[lane + 64]), b = max(lane_max[lane + 128], lane_max[lane + 192]);
        edge = order_value(edge_of(max(a, b), o.top));
        best.thr = edge;
        shared_thr = edge;  // by all the same; a later rise of one wave's may be lost to another's, no harm
      } else {
        edge = fmaxf(best.thr, *(volatile float *)&shared_thr);
      }
      // an equal value enters at the first step, and where another wave's threshold is the higher one
      const bool equal = first || edge > best.thr;
      if (first || __any(mx >= edge)) {
        bool in[8];
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          in[j] = at + 256 * (j >> 2) + 4 * lane + (j & 3) < i1 && (v[j] > edge || (equal && v[j] == edge));
          n += in[j];
        }
        const int upto = scan_lanes(n), all = __builtin_amdgcn_readlane(upto, 63);
        if (best.count + all <= kCap) {
          int p = best.count + upto - n;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (in[j]) buf[wave][p++] = make_key(v[j], at + 256 * (j >> 2) + 4 * lane + (j & 3));
          best.count += all;
        } else {
          f32x8 r = v;
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            const int i = at + 256 * (j >> 2) + 4 * lane + (j & 3);
            const float y = r[0];
            best.add(i < i1 && (y > edge || (equal && y == edge)), make_key(y, i));
            r = f32x8{r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[0]};
          }
        }
        if (all && !first && best.count >= 2 * o.top) {
          best.keep();
          if (lane == 0 && best.thr > edge) shared_thr = best.thr;
        }
      }
    }
    first = false;
    at += kTurn;
    v = v1;
    v1 = v2;
  } while (at < i1);
  // ---- the waves' sums and candidates in the first wave; then, in the last part of a row, the parts' the
  // same way (and by the same instructions: fetched once, they are cheap)
  const size_t p0 = (size_t)row * parts;
  Sums t{tm, ts, tw};
#pragma unroll 1
  for (bool joined = parts == 1;; joined = true) {
    t = join_wave(t);
    if (lane == 0) {
      wsum[wave] = t;
      wcount[wave] = best.count;
    }
    __syncthreads();
    if (wave == 0) {
      t.m = wsum[0].m;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) t.m = fmaxf(t.m, wsum[w].m);
      t.s = t.w = 0.;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const Sums x = below(wsum[w], t.m);
        t.s += x.s, t.w += x.w;
      }
      if (o.top) {
        int all = 0;
        for (int w = 0; w < kWaves; ++w) all += wcount[w];
        if (all <= kCap) {
          for (int w = 1; w < kWaves; ++w) {
            for (int i = lane; i < wcount[w]; i += 64) buf[0][best.count + i] = buf[w][i];
            best.count += wcount[w];
          }
        } else {
#pragma unroll 1
          for (int w = 1; w < kWaves; ++w)
#pragma unroll 1
            for (int i = 0; i < wcount[w]; i += 64) best.add(i + lane < wcount[w], i + lane < kCap ? buf[w][i + lane] : (u64)0);
        }
        best.keep();
      }
      if (joined) {
        finish(o, row, chosen, t, best.buf, best.count);
      } else {
        if (lane == 0) {
          put_shared(&part_sums[p0 + part].m, t.m);
          put_shared(&part_sums[p0 + part].s, t.s);
          put_shared(&part_sums[p0 + part].w, t.w);
        }
        if (lane < o.top) put_shared(&part_best[(p0 + part) * o.top + lane], lane < best.count ? best.buf[lane] : (u64)0);
        stores_done();
        if (lane == 0) is_last = atomicAdd(&done[row], 1u) == (uint32_t)parts - 1;
      }
    }
    if (joined) return;
    __syncthreads();
    if (!is_last) return;

    if (threadIdx.x == 0) done[row] = 0;  // as the next launch expects it
    t = Sums{kLow, 0., 0.};
    for (int p = threadIdx.x; p < parts; p += kThreads) {
      const Sums *q = part_sums + p0 + p;
      const Sums y{get_shared(&q->m), get_shared(&q->s), get_shared(&q->w)};
      const float m = fmaxf(t.m, y.m);
      const Sums a = below(t, m), b = below(y, m);
      t = Sums{m, a.s + b.s, a.w + b.w};
    }
    best.count = 0;
    if (o.top) {
      const u64 *keys = part_best + p0 * o.top;
      const int n = parts * o.top;
      u64 k[8];
      auto load_keys = [&](int i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = i + j * kThreads + lane < n ? get_shared(&keys[i + j * kThreads + lane]) : 0;
      };
      load_keys(64 * wave);
      // A key for each lane: the parts' first ones (the largest of several), or the first few of each part
      // where there are fewer than 64; a lane without one would pull the edge down to nothing.
      const int few = min((63 + parts) / parts, o.top);
      u64 head = 0;
#pragma unroll 4
      for (int p = lane; p < parts * few; p += 64) head = max(head, get_shared(&keys[(size_t)(p / few) * o.top + p % few]));
      const uint32_t edge = edge_of((uint32_t)(head >> 32), o.top);
#pragma unroll 1
      for (int i = 64 * wave; i < n;) {
        int in = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if ((uint32_t)(k[j] >> 32) < edge) k[j] = 0;
          in += k[j] != 0;
        }
        const int upto = scan_lanes(in), all = __builtin_amdgcn_readlane(upto, 63);
        if (best.count + all <= kCap) {
          int p = best.count + upto - in;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k[j]) buf[wave][p++] = k[j];
          best.count += all;
        } else {
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            best.add(k[0] != 0, k[0]);
#pragma unroll
            for (int h = 0; h < 7; ++h) k[h] = k[h + 1];
          }
        }
        i += 8 * kThreads;
        if (i < n) load_keys(i);
      }
    }
  }
}

}  // namespace

extern "C" int fhip_logprobs_f32(const float *dLogits, const int32_t *dTokens, float *dLogp, float *dEntropy, float *dTopLogp,
                                 int32_t *dTopIds, int rows, int vocab, int64_t ld, int top) {
  const char *who = "fhip_logprobs_f32";
  clear_error();
  if (rows < 0 || rows > 65535) return fail(FHIP_EINVAL, "%s: rows=%d outside 0..65535", who, rows);
  if (vocab < 1 || vocab > kMaxVocab || ld < vocab)
    return fail(FHIP_EINVAL, "%s: vocab=%d outside 1..%d or ld=%lld below it", who, vocab, kMaxVocab, (long long)ld);
  if (top < 0 || top > kMaxTop || top > vocab) return fail(FHIP_EINVAL, "%s: top=%d outside 0..%d or beyond vocab=%d", who, top, kMaxTop, vocab);
  if (rows == 0) return FHIP_OK;
  if (!dLogits || (dLogp && !dTokens) || (top && (!dTopLogp || !dTopIds))) return fail(FHIP_EINVAL, "%s: null pointer", who);
  if ((uintptr_t)dLogits & 3) return fail(FHIP_EINVAL, "%s: dLogits must be 4-byte aligned", who);
  if (dLogp) untag_range(dLogp, (size_t)rows * 4);
  if (dEntropy) untag_range(dEntropy, (size_t)rows * 4);
  if (top) {
    untag_range(dTopLogp, (size_t)rows * top * 4);
    untag_range(dTopIds, (size_t)rows * top * 4);
  }
  constexpr int kTile = kWaves * kStep;
  // A row's end of less than a step joins the tile before: alone it would have lanes without values, no edge
  // and every value a candidate (28,000 cycles where a tile takes 3,000).
  const int tiles = max(1, (vocab + kTile - kStep) / kTile);
  // As many parts as fill the card, of a tile each where there are few rows (one row of 152,064: 75 parts 13.5 us,
  // parts of two tiles 14.9, of four 18.7).
  int parts = max(1, min(tiles, 4 * cu_count() / rows));
  const int per = ((tiles - 1) / parts + 1) * kTile;
  parts = (tiles * kTile - 1) / per + 1;
  const Out o{dLogits, dTokens, dLogp, dEntropy, dTopLogp, dTopIds, vocab, top, ld};
  Sums *sums = nullptr;
  u64 *best = nullptr;
  uint32_t *done = nullptr;
  if (parts > 1) {
    if (!(done = counters(rows))) return FHIP_ENOMEM;
    const size_t sb = ((size_t)rows * parts * sizeof(Sums) + 255) & ~(size_t)255, bb = (size_t)rows * parts * top * 8;
    uint8_t *ws = (uint8_t *)workspace(sb + bb);
    if (!ws) return FHIP_ENOMEM;
    if (int rc = check_disjoint(who, dLogits, ((size_t)(rows - 1) * ld + vocab) * 4, ws, sb + bb)) return rc;
    sums = (Sums *)ws;
    best = (u64 *)(ws + sb);
  }
  logprobs_kernel<<<dim3(parts, rows), kThreads, 0, stream()>>>(o, sums, best, done, per);
  FHIP_CHECK_LAUNCH(who);
  return FHIP_OK;
}
