// kv4_attention.hip — attention over the paged 4-bit cache (fhip_kv4_attention_f32).
//
// For a request with L keys, of which the last n came with its n tokens of this batch, token i stands at
// p = L - n + i and sees the keys j with max(0, p - window + 1) <= j <= p (window 0: all up to p). For
// each of its heads (heads / heads_kv of them share a kv head)
//   o = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m)
// and zeros where no key is seen.
//
// Both products run on the 16x16x32 f16 matrix instruction. The cache's values are exact in f16 (kv4.hpp);
// what is f32, the queries and the weights e^(..), goes in as two f16 terms, hi = f16(x) and
// lo = f16(x - hi), 22 bits together, summed in f32. A row is a query token and a head; rows are the
// columns of the score tile S^T = K Q^T (16 keys x 16 rows), so that the softmax statistics of a row
// belong to a lane, and the weights leave S^T in the lane layout that the second product
// O^T = V^T P^T reads them in: no shuffle between the two. For that, row 4 g + i of score tile t is key
// 16 g + 4 t + i of a step of 64 keys: lane group g then holds the scores of granule g's 16 tokens, in
// the order that the transposing LDS read hands V's nibbles to it.
//
// An item is a request, a kv head and a tile of 8 or 16 rows; its keys go in rounds of a step (64 keys) for each of
// a workgroup's waves, which keep their own maximum, sum and output and join them in LDS at the end. All items'
// rounds, whatever the lengths are, are cut into one equal run per workgroup. The parts of an item that a cut
// crosses are joined by the last of its workgroups to be done or, where there can be many, by a second launch.
//
// What bounds it (128 dimensions, 28 heads over 4): a wave's step is some 530 vector instructions, most of them
// the unpack and the softmax, and takes 3,800 to 4,500 cycles with two waves on a SIMD, since each part of it
// waits for the one before (scores, maximum, weights, product). One token against 131,071 keys, 75 MB: 24 us and
// 4.5 for the join, 3.1 TB/s of the first; the same loads with no arithmetic take 16. 32 requests of up to 8,192
// keys, 20 MB: 16.2 us, of which the workgroups' start (lengths, table, queries, first loads: four dependent
// reads) is 4.5, the waves' steps 6.5, the joins 3. 128 requests of 8,000 keys: 4.8 TB/s. Two steps loaded ahead
// instead of one: 23.3 where one took 22.4, and 32.2 for the long one where one took 31.4. A tile walks all steps of
// its request, also those that its mask hides: a fresh prompt of 2,048 tokens, 16 heads over 8 of 256, 306 us.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kv4_attend.hpp"

using namespace fhip;

namespace {

// Waves of a workgroup: eight, which fill a CU two to a SIMD and leave half the parts that two workgroups of
// four would (32 requests: 22.4 us with four, 20.5 with eight; many items: run_waves); heads of 256 need four
// waves' registers and LDS.
constexpr int split_waves(int D) { return D == 256 ? 4 : 8; }
// Work is counted in rounds, one step of each wave. An item's queries, first loads and result cost as much as
// item_cost rounds more, and a workgroup gets `least` units at least. Cost and least for
// tiles of 8, 32 requests: 17.4 us with 1 and 2, 19.5 with 1 and 1, 20.3 with 2 and 3; for tiles of 16, 16
// requests of up to 35 rows: 22.9 with 2 and 3, 25.0 with 1 and 2.
constexpr int item_cost(bool pack) { return pack ? 1 : 2; }
constexpr int least(bool pack) { return pack ? 2 : 3; }
// Items of at most so many parts are joined in the launch: their last workgroup reads them in one round of
// loads. With more, a second launch with a workgroup for each row is the faster. One launch and two: 9.1 and
// 12.5 us for one request of 517 keys, 17.4 and 19.2 for 32 requests, 22.9 and 27.3 for 16 of up to 35 rows.
constexpr int kFewParts = 16;
constexpr int kMostParts = 1024;  // of an item: the workgroups of a launch

// Parts of an item, left by one workgroup for another of the launch.
__device__ inline void put_shared2(float *p, float x, float y) {
  put_shared(reinterpret_cast<uint64_t *>(p), (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x));
}
__device__ inline void put_shared4(float *p, f32x4 v) {
  put_shared2(p, v[0], v[1]);
  put_shared2(p + 2, v[2], v[3]);
}
__device__ inline void get_shared2(const float *p, float &x, float &y) {
  const uint64_t v = get_shared(reinterpret_cast<const uint64_t *>(p));
  x = __uint_as_float((uint32_t)v), y = __uint_as_float((uint32_t)(v >> 32));
}
__device__ inline f32x4 get_shared4(const float *p) {
  float a, b, c, d;
  get_shared2(p, a, b);
  get_shared2(p + 2, c, d);
  return f32x4{a, b, c, d};
}

// x + the same of the lane 8 away in its group of 16.
__device__ inline float add_ror8(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF, true));
}
// f over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
template <typename F>
__device__ inline float over_groups(float x, F f) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// PACK: tiles of 8 rows, their hi terms in columns 0..7 and lo terms in 8..15 of one operand; else of 16 rows,
// hi and lo terms in operands of their own. (Tiles of 32 rows, four waves to a CU for their registers: 30.3 us
// for 16 requests of up to 35 rows, where tiles of 16 take 24.9.)
template <int D, bool PACK, int kWaves>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void kv4_split_kernel(
    Attend a, Split *__restrict__ split, float *__restrict__ part_o, float *__restrict__ part_ml, uint32_t *__restrict__ done) {
  constexpr int NB = D / 32, DT = D / 16, RPT = PACK ? 8 : 16;
  constexpr int kThreads = 64 * kWaves, kItemCost = item_cost(PACK), kLeast = least(PACK);
  // A wave's stage in LDS, in words: the K codes of four granules, V codes, scales. The granules' strides
  // spread the reads of a lane group over the banks.
  constexpr int KS = 2 * D + 4, VS = 2 * D + (D == 64 ? 16 : 32), SS = D / 2;  // (D 64: two workgroups fit)
  constexpr int V0 = 4 * KS, S0 = V0 + 4 * VS, STAGE = S0 + 4 * SS;
  constexpr int LI = (D + 127) / 128;  // loads of a granule's codes, and of the step's scales
  constexpr int CH = D / 2;            // 16-byte chunks of them
  constexpr int OS = D + 4;            // a row of a wave's results, padded
  static_assert(RPT * (OS + 2) <= STAGE, "a wave's results have to fit its stage");
  __shared__ u32x4 buf0[kWaves * STAGE / 4], buf1[kWaves * STAGE / 4];
  __shared__ int scan[kWaves], found_before, found_r;
  __shared__ bool fallen[kWaves];
  __shared__ uint32_t is_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15, row = PACK ? col & 7 : col;
  const int group = a.heads / a.heads_kv;

  // ---- this workgroup's run of units. Up to 64 requests: a lane each, in every wave alike, with no LDS and no
  // second look at the lengths.
  auto load_request = [&](int i) { return request<RPT, kWaves, kItemCost>(a, a.start[i], a.start[i + 1], a.lens[i]); };
  const bool few = a.requests <= 64;
  const int per = few ? 1 : (a.requests + kThreads - 1) / kThreads, r0 = min((few ? lane : tid) * per, a.requests), r1 = min(r0 + per, a.requests);
  int mine = 0, before, total;
  bool falls = false;
  Req held;
  if (few) {
    held = load_request(min(r0, a.requests - 1));
    mine = r0 < a.requests ? held.units : 0;
    falls = __any(r0 < a.requests && falling(a, r0));
    const int upto = sum_lanes(mine);
    before = upto - mine;
    total = __builtin_amdgcn_readlane(upto, 63);
  } else {
    for (int r = r0; r < r1; ++r) mine += load_request(r).units, falls |= falling(a, r);
    falls = __any(falls);
    if (lane == 0) fallen[wave] = falls;
    total = sum_before<kWaves>(mine, scan, &before);
    falls = false;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) falls |= fallen[v];
  }
  if (falls) total = 0, a.least_rows = INT64_MAX;
  const int G = total < (int)gridDim.x * kLeast ? max(total / kLeast, 1) : gridDim.x;
  // Neighbouring runs go to one XCD (blockIdx mod 8) and the row tiles of a kv head follow each other, so that
  // the tiles of many rows share their keys' lines in one L2: worth 2 to 3% (window of 1,024: 24.0 us, else 24.8 before the queries were shared).
  int w = blockIdx.x;
  if (w < G) {
    const int x = w & 7;
    w = x * (G >> 3) + min(x, G & 7) + (w >> 3);
  }
  // entries that no workgroup below writes
  if (!done && !a.per_request && tid == 0) split[w].rows = 0;
  if (!done && a.per_request && w == 0 && (!few || wave == 0))
    for (int r = r0; r < r1; ++r)
      for (int i = load_request(r).row_tiles * a.heads_kv; i < a.per_request; ++i) split[(size_t)r * a.per_request + i].rows = 0;
  if (a.zero_rest) clear_rest(a, D);
  if (w >= G) return;
  const int share = divide(total, G), more = total - share * G;  // the first so many workgroups take one unit more
  const int u0 = share * w + min(w, more), u1 = u0 + share + (w < more);
  if (u0 == u1) return;
  const bool found = before <= u0 && u0 < before + mine;
  int r, pre;
  if (few) {
    r = __builtin_ctzll(__ballot(found));
    pre = __builtin_amdgcn_readlane(before, r);
  } else {
    if (found) found_r = r0, found_before = before;
    __syncthreads();
    r = __builtin_amdgcn_readfirstlane(found_r);
    pre = __builtin_amdgcn_readfirstlane(found_before);
  }
  auto at = [&](int i) {
    if (!few) return request<RPT, kWaves, kItemCost>(a, uniform(a.start, i), uniform(a.start, i + 1), uniform(a.lens, i));
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
    return Req{of(held.len), of(held.n), of(held.token0), of(held.nt), of(held.tile0), of(held.row_tiles), of(held.per_item), of(held.units)};
  };
  Req rq = at(r);

  const Unpack unpack;
  const h2 k24 = {(_Float16)-24.f, (_Float16)-24.f};
  const float lo_half = PACK && col >= 8 ? 1.f : 0.f;
  // this lane's places in a stage, in words
  const uint32_t base = in_reg(wave * STAGE);
  const uint32_t k_at = base + (col >> 2) * KS + (col & 3) * (D / 8) + g * NB;
  const uint32_t ks_at = base + S0 + (col >> 2) * SS;
  const uint32_t v_at = base + V0 + g * VS + 2 * col;
  const uint32_t vs_at = base + S0 + g * SS + D / 4;
  const uint32_t san_at = 2 * (base + S0 + g * SS) + D / 2;  // in f16: V's scales of this lane's granule
  auto words = [](u32x4 *b) { return reinterpret_cast<uint32_t *>(b); };

  // O and its weights' sum to the output; the values' factor of 4 goes in, and no key gives 0.
  auto write_row = [&](int token0, int kvh, int rr, int d4, f32x4 O, float L) {
    const int tok = divide_lanes(rr, group, rr < 1 << 22), h = kvh * group + rr - tok * group;
    f32x4 y = O * (4.f / L);
    if (L == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
    reinterpret_cast<f32x4 *>(a.out + ((size_t)(token0 + tok) * a.heads + h) * D)[d4] = y;
  };
  for (int u = u0; u < u1;) {
    while (u >= pre + rq.units) {
      pre += rq.units;
      rq = at(++r);
    }
    const int per_item = rq.per_item, rounds = per_item - kItemCost;
    const int item = divide(u - pre, per_item), x0 = u - pre - item * per_item, x1 = min(x0 + u1 - u, per_item);
    const int first_round = max(x0 - kItemCost, 0), end_round = max(x1 - kItemCost, 0);
    const int item_end = u - x0 + per_item;
    u += x1 - x0;
    if (first_round == end_round) continue;  // the item begins with the next workgroup
    const int t0 = first_round * kWaves, t1 = min(end_round * kWaves, rq.nt);
    const int kvh = rq.row_tiles == 1 ? item : divide(item, rq.row_tiles), rt = item - kvh * rq.row_tiles;
    const int rows_all = rq.n * group, row0 = rt * RPT, rows = min(RPT, rows_all - row0);
    auto token_of = [&](int rr) { return rq.n == 1 ? 0 : divide(rr, group); };
    const int p_last = rq.len - rq.n + token_of(row0 + rows - 1);   // of the tile's rows
    const int p_first = rq.len - rq.n + token_of(row0);
    const int first_last = first_key(p_last, a.window);
    const int32_t *table = a.table + (size_t)r * a.cols;

    // ---- page ids of this wave's next 16 steps, a lane for each granule
    const int lim = max(p_last, 0);
    auto page_ids = [&](int t) {
      const int64_t k = min((int64_t)(rq.tile0 + t + kWaves * (lane >> 2)) * kStep + 16 * (lane & 3), (int64_t)lim);
      return min(max(table[k >> a.shift], 0), a.pages - 1);  // past the last key: its own granule again
    };
    int t = t0 + wave, ids_from = min(t, t1 - 1), ids = page_ids(ids_from);

    // ---- queries: a wave's rows are converted for all waves, and the first step's loads issued behind them. (Every
    // wave all rows for itself: 24.2 us for the window of 1,024, where this takes 21.0, 17.4 for 32 requests, where
    // this takes 17.0; the loads first: 22 and 17.5.) A lane has dimensions j and j + 4 of a run of eight, the two
    // halves of an operand's word.
    constexpr int RW = RPT / kWaves, PL = (D + 127) / 128;  // rows of a wave, pairs of a lane
    auto pair_of = [&](int i) { return min(64 * i + lane, D / 2 - 1); };
    const int my_row = row0 + min(row, rows - 1), my_token = divide_lanes(my_row, group, rows_all < 1 << 22);
    const int pos = row < rows ? rq.len - rq.n + my_token : INT32_MAX;
    const int first = row < rows ? first_key(pos, a.window) : 0;
    const int64_t my_q = (int64_t)(rq.token0 + my_token) * a.ldq + (kvh * group + my_row - my_token * group) * D;
    float x[RW][PL][2];
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      auto of = [&](int64_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, wave * RW + k); };  // lane i has row i
      const float *src = a.q + ((int64_t)of(my_q >> 32) << 32 | of(my_q));
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const int q = pair_of(i), at = 8 * (q >> 2) + (q & 3);
        x[k][i][0] = src[at], x[k][i][1] = src[at + 4];
      }
    }
    __builtin_amdgcn_sched_barrier(0);

    auto load = [&](int t, u32x4 *buf) {
      const int at = 4 * ((t - ids_from) / kWaves);
      const uint8_t *gr[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        gr[c] = granule_of(a, __builtin_amdgcn_readlane(ids, at + c), min((rq.tile0 + t) * kStep + 16 * c, lim), kvh, kv4_granule_bytes(D));
      uint32_t *dst = words(buf) + wave * STAGE;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < LI; ++i)
          if (CH % 64 == 0 || lane < CH) {
            lds_load16(gr[c], dst + c * KS + 256 * i, 16 * lane, 1024 * i);
            lds_load16(gr[c], dst + V0 + c * VS + 256 * i, 16 * lane, kv4_v_codes(D) + 1024 * i);
          }
#pragma unroll
      for (int i = 0; i < LI; ++i) {
        const int ch = 64 * i + lane, c = ch / (D / 8), off = ch - c * (D / 8);
        const uint8_t *p = c == 0 ? gr[0] : c == 1 ? gr[1] : c == 2 ? gr[2] : gr[3];
        if (CH % 64 == 0 || lane < CH)
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(p + kv4_k_scales(D) + 16 * off),
                                           (__attribute__((address_space(3))) void *)(dst + S0 + 256 * i), 16, 0, 0);
      }
    };
    // Times the scale, by the row's power of two into [2^12, 2^14): with the factor's own rounding (kl) in,
    // since it would shift a score of several hundred by more than all else. Their place is where the second
    // step will go.
    constexpr int QS = NB * 4 + 1;  // a row of operands and a pad, 16 bytes each
    static_assert(8 * RPT * QS + RPT <= STAGE, "the operands have to fit a wave's stage");
    float *units = reinterpret_cast<float *>(buf1) + 8 * RPT * QS;
#pragma unroll
    for (int k = 0; k < RW; ++k) {
      const int rho = wave * RW + k;
      int big = 0;
#pragma unroll
      for (int i = 0; i < PL; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) big = max(big, __float_as_int(x[k][i][j]) & 0x7FFFFFFF);
      big = max_lanes(big);
      int e = 0;
      if (big < 0x7F800000) (void)frexpf(__int_as_float(big), &e);
      if (lane == 0) units[rho] = ldexpf(1.f, max(e - 13 + a.ke, -120));  // a raw score's worth in powers of two, itself one
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        h2 hi, lo;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float v = ldexpf(x[k][i][j], 13 - e), y = __builtin_fmaf(v, a.kh, v * a.kl);
          hi[j] = (_Float16)y;
          lo[j] = (_Float16)(y - (float)hi[j]);
        }
        words(buf1)[4 * rho * QS + pair_of(i)] = as_u(hi);
        words(buf1)[4 * (RPT + rho) * QS + pair_of(i)] = as_u(lo);
      }
    }
    auto all_waves = [&] {  // __syncthreads would wait for the first step's loads too
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    __builtin_amdgcn_sched_barrier(0);
    load(ids_from, buf0);  // a wave without a step too
    __builtin_amdgcn_sched_barrier(0);
    all_waves();
    f16x8 qh[NB], ql[PACK ? 1 : NB];
    const float unit = units[row];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      qh[b] = __builtin_bit_cast(f16x8, buf1[(PACK ? col : row) * QS + 4 * b + g]);
      if (!PACK) ql[b] = __builtin_bit_cast(f16x8, buf1[(RPT + row) * QS + 4 * b + g]);
    }
    all_waves();

    f32x4 o[DT];
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int t, u32x4 *buf) {
      const uint32_t *b32 = words(buf);
      const int k0 = (rq.tile0 + t) * kStep;
      const bool whole = k0 >= first_last && k0 + kStep - 1 <= p_first;
      // The step's K codes and scales are all asked for at once, and V's before the softmax: read where they are
      // used, each would be waited for (32 requests 16.6 us, else 17.3; the long token 28.3, else 29.9).
      uint32_t kc[4][NB];
      _Float16 ksc[4][NB];
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4) {
        if constexpr (NB % 4 == 0) {
#pragma unroll
          for (int b = 0; b < NB; b += 4) {
            const u32x4 v = buf[k_at / 4 + t4 * (D / 8) + b / 4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kc[t4][b + j] = v[j];
          }
        } else {
#pragma unroll
          for (int b = 0; b < NB; ++b) kc[t4][b] = b32[k_at + t4 * 4 * (D / 8) + b];
        }
        const _Float16 *sc = reinterpret_cast<const _Float16 *>(b32 + ks_at) + (4 * t4 + (col & 3)) * NB;
#pragma unroll
        for (int b = 0; b < NB; ++b) ksc[t4][b] = sc[b];
      }
      __builtin_amdgcn_sched_barrier(0);
      if (!whole) {
        // Keys that some row does not see. What they hold must not reach it: a V scale that no written block has
        // (NaN, or bytes left by someone else) counts as 0, and a row that does see the key gets the NaN in the
        // block's sums, where the product would have put it.
        _Float16 *s = reinterpret_cast<_Float16 *>(buf);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const bool odd = !(fabsf((float)s[san_at + 16 * b + kv4_v_place(col)]) <= kMaxScale);
          if (const uint64_t bad = __ballot(odd)) {  // bit j: key k0 + j
            if (odd) s[san_at + 16 * b + kv4_v_place(col)] = (_Float16)0.f;
            const float taint = bad & keys_between(first - k0, pos - k0) ? __builtin_nanf("") : 0.f;
            o[2 * b] += taint, o[2 * b + 1] += taint;
          }
        }
        asm volatile("" ::: "memory");  // the words just written are read below as another type
      }
      f32x4 s[4];
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4) {
        s[t4] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const h2 sk = {ksc[t4][b], ksc[t4][b]}, ck = sk * k24;
          const f16x8 k = unpack(kc[t4][b], sk, sk, sk, sk, ck, ck, ck, ck);
          s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[b], s[t4], 0, 0, 0);
          if (!PACK) s[t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[b], s[t4], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      u32x4 vs[NB][2];
      i32x2 vc[DT];
      auto ask_v = [&](int b) {
        vs[b][0] = buf[(vs_at + 8 * b) / 4], vs[b][1] = buf[(vs_at + 8 * b) / 4 + 1];
#pragma unroll
        for (int d = 2 * b; d < 2 * b + 2; ++d)
          vc[d] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2 *)(b32 + v_at + 32 * d));
      };
      constexpr int VP = PACK ? NB : NB / 2;  // as many blocks as the registers allow
#pragma unroll
      for (int b = 0; b < VP; ++b) ask_v(b);
      __builtin_amdgcn_sched_barrier(0);
      f16x8 ph[2], pl[2];
      float x[4][4], mx = -__builtin_inff();
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t4][i] = PACK ? add_ror8(s[t4][i]) : s[t4][i];
      if (!whole) {
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + 16 * g + 4 * t4 + i;
            if (key < first || key > pos) x[t4][i] = -__builtin_inff();
          }
      }
#pragma unroll
      for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[t4][i]);
      mx = over_groups(mx, [](float p, float q) { return fmaxf(p, q); });
      if (__any(mx > m)) {
        const float f = mx > m ? exp2_fast((m - mx) * unit) : 1.f;
        m = fmaxf(m, mx);
        l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
      }
      const float bias = m == -__builtin_inff() ? kBias : __builtin_fmaf(-m, unit, kBias);
      u32x4 hi[2], lo[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e0 = exp2_fast(__builtin_fmaf(x[2 * h][i], unit, bias));
          const float e1 = exp2_fast(__builtin_fmaf(x[2 * h + 1][i], unit, bias));
          l += e0;
          l += e1;
          const h2 p = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e0, e1));
          if (PACK) {
            const float d0 = __builtin_fmaf((float)p.x, -lo_half, e0), d1 = __builtin_fmaf((float)p.y, -lo_half, e1);
            hi[h][i] = as_u(__builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(d0, d1)));
          } else {
            hi[h][i] = as_u(p);
            lo[h][i] = as_u(__builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e0 - (float)p.x, e1 - (float)p.y)));
          }
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ph[h] = __builtin_bit_cast(f16x8, hi[h]);
        if (!PACK) pl[h] = __builtin_bit_cast(f16x8, lo[h]);
      }
#pragma unroll
      for (int b = VP; b < NB; ++b) ask_v(b);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        h2 sv[8], cv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sv[i] = as_h2(vs[b][i >> 2][i & 3]);
          cv[i] = sv[i] * k24;
        }
#pragma unroll
        for (int d = 2 * b; d < 2 * b + 2; ++d) {
          const f16x8 v0 = unpack((uint32_t)vc[d].x, sv[0], sv[1], sv[2], sv[3], cv[0], cv[1], cv[2], cv[3]);
          const f16x8 v1 = unpack((uint32_t)vc[d].y, sv[4], sv[5], sv[6], sv[7], cv[4], cv[5], cv[6], cv[7]);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], o[d], 0, 0, 0);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], o[d], 0, 0, 0);
          if (!PACK) {
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], o[d], 0, 0, 0);
          }
        }
      }
    };

    // ---- the segment's steps, the waves in turn; each wave on its own, one step loaded ahead
    constexpr int NL = 9 * LI;
    auto landed = [&](bool more) {
      // vmcnt: the next step's loads may be under way, this one's not
      if (more) __builtin_amdgcn_s_waitcnt(0x0F70 | (NL & 15) | (NL >> 4) << 14);
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      asm volatile("" ::: "memory");
    };
    auto ahead = [&](int t, u32x4 *buf) {
      if (t >= t1) return false;
      if (t - ids_from == 16 * kWaves) ids = page_ids(t), ids_from = t;
      // this wave's reads of the place are done
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      asm volatile("" ::: "memory");
      load(t, buf);
      return true;
    };
    while (t < t1) {
      const bool more0 = ahead(t + kWaves, buf1);
      landed(more0);
      compute(t, buf0);
      t += kWaves;
      if (!more0) break;
      const bool more1 = ahead(t + kWaves, buf0);
      landed(more1);
      compute(t, buf1);
      t += kWaves;
    }

    landed(false);  // nothing may still arrive where the results go
    // ---- the waves' results to LDS, each in its own stage: m, l, then the rows of O, and joined. With
    // 4 * 2^-14 in O and 2^-14 in l the bias falls out and the scales' factor goes in.
    float *res = reinterpret_cast<float *>(buf0);
    f32x4 *res4 = reinterpret_cast<f32x4 *>(buf0);
    l = over_groups(l, [](float p, float q) { return p + q; });
    if (PACK) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] = add_ror8(o[d][i]);
    }
    if (g == 0 && (!PACK || col < 8)) {
      res[wave * STAGE + row] = m * unit;
      res[wave * STAGE + RPT + row] = l;
    }
    if (!PACK || col < 8)
#pragma unroll
      for (int d = 0; d < DT; ++d) res4[(wave * STAGE + 2 * RPT + row * OS + 16 * d + 4 * g) / 4] = o[d];
    __syncthreads();
    const bool is_whole = first_round == 0 && end_round == rounds;
    const size_t slot = 2 * (size_t)w + (first_round == 0);
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int rho = i / (D / 4), d4 = i - rho * (D / 4);
      float mw[kWaves], mm = -__builtin_inff();
#pragma unroll
      for (int v = 0; v < kWaves; ++v) mm = fmaxf(mm, mw[v] = res[v * STAGE + rho]);
      const float z = mm == -__builtin_inff() ? 0.f : mm;
      float L = 0.f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const float f = exp2_fast(mw[v] - z);
        L += f * res[v * STAGE + RPT + rho];
        O += f * res4[(v * STAGE + 2 * RPT + rho * OS) / 4 + d4];
      }
      if (is_whole) {
        write_row(rq.token0, kvh, row0 + rho, d4, O, L);
      } else {
        put_shared4(part_o + (slot * RPT + rho) * D + 4 * d4, O);
        if (d4 == 0) put_shared2(part_ml + (slot * RPT + rho) * 2, mm, L);
      }
    }
    if (is_whole) {
      if (!done && a.per_request && tid == 0) split[(size_t)r * a.per_request + item].rows = 0;
    } else {
      // the workgroups with the item's first and last units
      auto owner = [&](int v) {
        const int big_end = (share + 1) * more;
        return v < big_end ? divide(v, share + 1) : more + divide(v - big_end, share);
      };
      const int w1 = owner(item_end - 1);
      if (!done) {
        if (first_round == 0 && tid == 0)
          split[a.per_request ? (size_t)r * a.per_request + item : w] = Split{rows, w, w1, rq.token0, kvh, row0};
      } else {
        // The first part is of the first workgroup that does any of the item's rounds: one of its units
        // past the item's cost.
        const int w0 = owner(item_end - rounds), parts = w1 - w0 + 1;
        stores_done();
        __syncthreads();
        if (tid == 0) is_last = atomicAdd(&done[w0], 1u) == (uint32_t)parts - 1;
        __syncthreads();
        if (is_last) {
          if (tid == 0) done[w0] = 0;  // as the next launch expects it
          auto slot_of = [&](int i) { return 2 * (size_t)(w0 + i) + (i == 0); };
          for (int i = tid; i < rows * (D / 4); i += kThreads) {  // all parts requested at once
            const int rho = i / (D / 4), d4 = i - rho * (D / 4);
            float mw[kFewParts], lw[kFewParts], mm = -__builtin_inff(), L = 0.f;
            f32x4 y[kFewParts], O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < kFewParts; ++p) {
              const size_t at = slot_of(min(p, parts - 1)) * RPT + rho;
              get_shared2(part_ml + 2 * at, mw[p], lw[p]);
              y[p] = get_shared4(part_o + at * D + 4 * d4);
            }
#pragma unroll
            for (int p = 0; p < kFewParts; ++p) mm = fmaxf(mm, mw[p]);
            const float z = mm == -__builtin_inff() ? 0.f : mm;
#pragma unroll
            for (int p = 0; p < kFewParts; ++p)
              if (p < parts) {
                const float f = exp2_fast(mw[p] - z);
                L += f * lw[p];
                O += f * y[p];
              }
            write_row(rq.token0, kvh, row0 + rho, d4, O, L);
          }
        }
      }
    }
    __syncthreads();
  }
}

// One row of an item that several workgroups worked on: their parts in order, weighted by 2^(m - max). The
// first parts' values are requested before the weights are known. Bound by two dependent reads: 4.7 us for 28 rows
// of 64 parts each.
template <int D>
__global__ __launch_bounds__(256) void kv4_join_kernel(Attend a, const Split *__restrict__ split, const float *__restrict__ part_o,
                                                       const float *__restrict__ part_ml, int rpt) {
  constexpr int L4 = D / 4, PG = 256 / L4, AHEAD = 16;  // lanes of a row, parts at a time, of them requested first
  __shared__ float wt[kMostParts], red[8];
  __shared__ float4 sum[PG][L4];
  const Split s = split[blockIdx.x];
  const int tid = threadIdx.x;
  const int rho = blockIdx.y;
  if (rho >= s.rows) return;
  const int parts = s.last - s.first + 1;
  auto slot = [&](int i) { return 2 * (size_t)(s.first + i) + (i == 0); };
  const int x = tid % L4, pg = tid / L4;
  auto value = [&](int i) { return reinterpret_cast<const float4 *>(part_o + (slot(i) * rpt + rho) * D)[x]; };
  float4 v[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (pg + j * PG < parts) v[j] = value(pg + j * PG);
  float mm = -__builtin_inff();
  for (int i = tid; i < parts; i += 256) mm = fmaxf(mm, part_ml[(slot(i) * rpt + rho) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mm = fmaxf(mm, __shfl_xor(mm, d));
  if ((tid & 63) == 0) red[tid >> 6] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float z = mm == -__builtin_inff() ? 0.f : mm;
  float l = 0.f;
  for (int i = tid; i < parts; i += 256) {
    const float *ml = part_ml + (slot(i) * rpt + rho) * 2;
    const float f = exp2_fast(ml[0] - z);
    wt[i] = f;
    l += f * ml[1];
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);
  float4 acc{0.f, 0.f, 0.f, 0.f};
  auto add = [&](float f, const float4 y) { acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w; };
  if (pg < PG) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (pg + j * PG < parts) add(wt[pg + j * PG], v[j]);
#pragma unroll 8
    for (int i = pg + AHEAD * PG; i < parts; i += PG) add(wt[i], value(i));
    sum[pg][x] = acc;
  }
  __syncthreads();
  if (tid < L4) {
#pragma unroll
    for (int i = 1; i < PG; ++i) {
      const float4 y = sum[i][x];
      acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
    }
    const float f = l == 0.f ? 0.f : 4.f / l;
    const int group = a.heads / a.heads_kv, rr = s.row0 + rho, tok = rr / group, h = s.kvh * group + rr - tok * group;
    const float4 y = l == 0.f ? float4{0.f, 0.f, 0.f, 0.f} : float4{acc.x * f, acc.y * f, acc.z * f, acc.w * f};
    reinterpret_cast<float4 *>(a.out + ((size_t)(s.token0 + tok) * a.heads + h) * D)[x] = y;
  }
}

// An item's steps are bounded by its table row and its window.
int64_t steps_bound(const Attend &a) {
  const int64_t keys = (int64_t)a.cols << a.shift, seen = a.window ? std::min(keys, (int64_t)a.window + a.tokens + 2 * kStep) : keys;
  return (seen + kStep - 1) / kStep;
}

template <int D, bool PACK, int kWaves>
int run_split(const char *who, Attend a) {
  constexpr int RPT = PACK ? 8 : 16, kItemCost = item_cost(PACK), kLeast = least(PACK);
  // As many workgroups as stay resident (by the stages' LDS).
  constexpr int kPerCu = (D == 256 ? 4 : D == 64 ? 16 : 8) / kWaves;
  const int group = a.heads / a.heads_kv;
  const int64_t steps = (((int64_t)a.cols << a.shift) - 1) / kStep + 1;
  const int64_t row_tiles = ((int64_t)a.tokens * group) / RPT + a.requests;
  const int64_t most = std::min(row_tiles * a.heads_kv, (int64_t)1 << 31) * ((steps + kWaves - 1) / kWaves + kItemCost) / kLeast + 1;
  const int grid = (int)std::min(std::min((int64_t)kPerCu * cu_count(), (int64_t)kMostParts), most);
  // A request's items are bounded by the tokens that all requests have; where that bounds them all below the
  // grid, the joining launch is as large as that (28 rows of one long request: 32 workgroups, not 4,096).
  const int64_t per_request = ((int64_t)a.tokens * group + RPT - 1) / RPT * a.heads_kv;
  a.per_request = per_request * a.requests <= grid ? (int)per_request : 0;
  const int entries = a.per_request ? a.per_request * a.requests : grid;
  const size_t sb = ((size_t)grid * sizeof(Split) + 255) & ~(size_t)255, mb = ((size_t)grid * 2 * RPT * 8 + 255) & ~(size_t)255;
  const size_t need = sb + mb + (size_t)grid * 2 * RPT * D * 4;
  uint8_t *ws = (uint8_t *)workspace(need);
  if (!ws) return FHIP_ENOMEM;
  Split *split = (Split *)ws;
  float *ml = (float *)(ws + sb), *po = (float *)(ws + sb + mb);
  // An item's parts are bounded by its rounds and the least share of a workgroup.
  const int64_t rounds = (steps_bound(a) + kWaves - 1) / kWaves + 1;
  uint32_t *done = nullptr;
  if ((rounds + kLeast - 1) / kLeast + 1 <= kFewParts && !(done = counters(grid))) return FHIP_ENOMEM;
  kv4_split_kernel<D, PACK, kWaves><<<grid, 64 * kWaves, 0, stream()>>>(a, split, po, ml, done);
  FHIP_CHECK_LAUNCH(who);
  if (done) return FHIP_OK;
  kv4_join_kernel<D><<<dim3(entries, RPT), 256, 0, stream()>>>(a, split, po, ml, RPT);
  FHIP_CHECK_LAUNCH(who);
  return FHIP_OK;
}

// Workgroups of four waves for single tokens of more items than CUs: an item's start and joins then keep half as
// many waves from work. Eight and four waves, us, 8 key heads, all requests of one length:
//   heads of 128  256 items of 128 keys 7.6 and 6.9, 500: 9.3 and 12.4, 2,000: 21 and 27
//                 320                   11.2 and 8.4     14.7 and 12.7      31 and 30
//                 1,024                 20.2 and 14.0    29.4 and 24.1      72 and 62
//   heads of 64   256                   7.9 and 6.4      9.0 and 10.4       27 and 24
//                 320                   11.5 and 7.4     14.0 and 10.4      30 and 25
//                 512                   11.6 and 7.7     14.2 and 16.4      26 and 34
//                 1,024                 19.3 and 13.7    24.0 and 18.3      47 and 41
// and heads of 96 as of 128. What 512 items of heads of 64 lose, one for each place of an eight-wave workgroup, holds
// for equal lengths alone: spread evenly over their logarithm up to 2,000 they take 25 and 17, up to 700 19 and 12.5.
// (Tiles of 16 rows have no registers for four.)
template <int D, bool PACK>
int run_waves(const char *who, const Attend &a, int64_t rows) {
  constexpr int W = split_waves(D);
  if constexpr (PACK && W == 8)
    if ((rows + 7) / 8 * a.requests * a.heads_kv > cu_count()) return run_split<D, PACK, 4>(who, a);
  return run_split<D, PACK, W>(who, a);
}

// Requests of more than kFewRows rows take the prefill kernel (which has no heads of 256), others the split
// kernel; a batch of both takes both launches, and where every request has max_new tokens, or none can have
// many rows, one does for all. With 28 heads over 4, microseconds of split and prefill kernel: 16 requests of
// 8,000 keys, 63 rows 62 and 80, 84 rows 99 and 83, 252 rows 238 and 153.
// But the split kernel cuts finer: where all rows in tiles of 16 are at most kSmall steps for each CU, it is the
// faster for any number of rows: 252 rows of one request of 1,000 keys (4 a CU) 15 and 25, of 8,000 (31) 30 and
// 43, of 32,000 (125) 69 and 66; of 16 requests of 1,000 keys (64) 54 and 42, 189 rows of them (48) 42 and 42.
constexpr int kFewRows = 64, kSmall = 64;

template <int D>
int run(const char *who, Attend a, int max_new) {
  const int64_t group = a.heads / a.heads_kv, rows = std::max(max_new, 1) * group;
  const int64_t steps = steps_bound(a), small_tiles = a.tokens * group / 16 + a.requests;
  if (D != 256 && rows > kFewRows && small_tiles * a.heads_kv * steps > kSmall * (int64_t)cu_count()) {
    const bool both = (int64_t)a.requests * max_new != a.tokens;
    a.least_rows = both ? kFewRows + 1 : 0;
    if (int rc = kv4_prefill(who, D, a)) return rc;
    if (!both) return FHIP_OK;
    a.least_rows = 0, a.most_rows = kFewRows, a.zero_rest = false;
  }
  // Tiles of 8 rows where there are no more, or where all of them in tiles of 8 are two steps at most for each of
  // a full grid's waves: then a step's latency counts, not the unpack done twice (14 rows of 8,000 keys: 17 us
  // in tiles of 8, 23 of 16; the same for 16 requests: 45 and 31).
  const int64_t tiles = a.tokens * group / 8 + a.requests;
  return rows <= 8 || tiles * a.heads_kv * steps <= 16 * (int64_t)cu_count() ? run_waves<D, true>(who, a, rows) : run_waves<D, false>(who, a, rows);
}

}  // namespace

extern "C" int fhip_kv4_attention_f32(const void *dCache, const float *dQ, float *dOut, const int32_t *dStart, const int32_t *dLens,
                                      const int32_t *dTable, int requests, int tokens, int max_new, int heads, int heads_kv,
                                      int head_dim, int pages, int page, int table_cols, int ldq, int window, float scale) {
  const char *who = "fhip_kv4_attention_f32";
  clear_error();
  if (int rc = kv4_check_shape(who, heads_kv, head_dim, pages, page)) return rc;
  if (heads <= 0 || heads % heads_kv) return fail(FHIP_EINVAL, "%s: heads=%d is no positive multiple of heads_kv=%d", who, heads, heads_kv);
  if ((int64_t)heads * head_dim > (1 << 20)) return fail(FHIP_EINVAL, "%s: heads * head_dim = %lld passes 2^20", who, (long long)heads * head_dim);
  if (requests < 1 || requests > 65535) return fail(FHIP_EINVAL, "%s: requests=%d outside 1..65535", who, requests);
  if (tokens < 0 || max_new < 0 || window < 0) return fail(FHIP_EINVAL, "%s: tokens=%d, max_new=%d or window=%d below 0", who, tokens, max_new, window);
  if (table_cols < 1 || (int64_t)table_cols * page > INT32_MAX)
    return fail(FHIP_EINVAL, "%s: table_cols=%d of %d tokens: need 1 or more and positions below 2^31", who, table_cols, page);
  if (ldq < heads * head_dim || ldq % 4) return fail(FHIP_EINVAL, "%s: ldq=%d must be a multiple of 4, at least heads * head_dim", who, ldq);
  if (!(scale > 0.f) || scale > 1e37f) return fail(FHIP_EINVAL, "%s: scale=%g outside (0, 1e37]", who, scale);
  if (tokens == 0) return FHIP_OK;
  if (!dCache || !dQ || !dOut || !dStart || !dLens || !dTable) return fail(FHIP_EINVAL, "%s: null pointer", who);
  if (((uintptr_t)dCache | (uintptr_t)dQ | (uintptr_t)dOut) & 15) return fail(FHIP_EINVAL, "%s: dCache, dQ and dOut must be 16-byte aligned", who);
  untag_range(dOut, (size_t)tokens * heads * head_dim * 4);
  int shift = 0, ke = 0;
  while ((1 << shift) < page) ++shift;
  const double km = std::frexp((double)scale * (4. * kLog2e), &ke) * 2.;
  const float kh = (float)km;
  Attend a{(const uint8_t *)dCache, dQ, dOut, dStart, dLens, dTable, requests, tokens, heads, heads_kv, pages, shift, table_cols, ldq, window, kh, (float)(km - kh), ke - 1, 0, 0, INT64_MAX, true};
  // A launch counts its units in 31 bits: for each row tile and kv head, a unit for 64 keys at most and two more.
  // Requests whose tables allow more go by turns.
  const int64_t group = heads / heads_kv, rows = std::max(max_new, 1) * group;
  const bool wide = head_dim != 256 && rows > kFewRows;
  const int rpt = wide ? 128 : rows <= 8 ? 8 : 16;  // (smaller tiles are taken where units are few)
  const int64_t steps = ((int64_t)table_cols * page - 1) / kStep + 3, tiles = INT32_MAX / heads_kv / steps;
  const int64_t spare = std::min(tiles - (tokens * group / rpt + 1), tiles / 4);  // a wide batch's few-row requests: 4 tiles each
  if (spare < 1)
    return fail(FHIP_EINVAL, "%s: %d tokens of %d heads over %lld positions are too many for one call", who, tokens, heads, (long long)table_cols * page);
  for (int r = 0; r < requests; r += a.requests) {
    a.requests = (int)std::min((int64_t)requests - r, spare);
    a.start = dStart + r, a.lens = dLens + r, a.table = dTable + (size_t)r * table_cols;
    a.zero_rest = r + a.requests == requests;
    const int rc = head_dim == 64 ? run<64>(who, a, max_new) : head_dim == 96 ? run<96>(who, a, max_new)
                 : head_dim == 128 ? run<128>(who, a, max_new) : run<256>(who, a, max_new);
    if (rc) return rc;
  }
  return FHIP_OK;
}
