// kv4_prefill.hip — attention over the 4-bit cache for many query rows (prompts' chunks).
//
// The products are those of kv4_attention.hip, on the 32x32x16 instruction. An item is 128 rows (query
// tokens times the heads of a kv head) of one request and kv head; a workgroup's four waves have 32 rows
// each. For every 64 keys each wave unpacks one granule to f16 in LDS, K as rows and V transposed, then
// all read both: the unpack costs a quarter of what it would if every wave did it for itself.
//
// Bound by the matrix instructions: two terms of each f32 operand make 2 * 2 * 32 * 64 * 128 products of
// a step, 2,048 of a SIMD's cycles, beside some 1,600 of vector instructions, which the CU's second
// workgroup overlaps. A chunk of 2,048 tokens behind 2,048 keys (beside one of ten tokens), 28 heads over 4 of 128: 190
// to 225 us with the card's clock, 182 GFLOP of products in two terms or 0.8 to 0.95 PFLOP/s, where a large f16 product
// reaches 1.13; matrix and vector units are each busy a little over half of the time. In turn, not side by side, the same
// took 226. A fresh prompt of 4,096 tokens: 286 us, of 1,536 in cut items 93, since a cut counts the masked steps too.
//
// Items are whole where there are enough of them for the card; the steps of few long items are cut into
// equal runs and joined by a second launch. Heads of 256 stay with the split kernel: 32 rows of them, two
// terms of the queries and the outputs, pass the registers.
#include <algorithm>
#include <cstdint>

#include "kv4_attend.hpp"

using namespace fhip;

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;

// f over the two halves of a wave.
template <typename F>
__device__ inline float over_halves(float x, F f) {
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Runs of four units at least, of which an item's cost is two (2,100 rows of 1,000 keys: 33 us, with eight 37; 252
// rows: 25 and 34).
constexpr int kRows = 128, kCost = 2, kLeast = 4;

template <int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void kv4_prefill_kernel(
    Attend a, Split *__restrict__ split, float *__restrict__ part_o, float *__restrict__ part_ml, int split_wgs) {
  constexpr int NB = D / 32, NS = D / 16;              // scale blocks; 16-dimension steps of Q K^T
  constexpr int GW = kv4_granule_bytes(D) / 4, GL = (kv4_granule_bytes(D) + 1023) / 1024;  // a granule: words, loads
  constexpr int KU = D / 8 + 1, VU = 9;                // 16-byte units of a K row, a V column (a pad each)
  __shared__ u32x4 P0[kWaves * GW / 4], P1[kWaves * GW / 4];  // packed granules, a wave's own
  __shared__ u32x4 KF[64 * KU], VF[D * VU];
  __shared__ uint8_t bad_blocks[2][kStep];  // of each key of odd and even steps: a bit for each block
  __shared__ int scan_i[kWaves], scan_u[kWaves], found_before, found_r;
  __shared__ bool fallen[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31, l16 = lane & 15, q4 = lane >> 4;
  const int group = a.heads / a.heads_kv, w = blockIdx.x;
  auto words = [](u32x4 *b) { return reinterpret_cast<uint32_t *>(b); };

  // ---- this workgroup's items, or its run of units
  const int per = (a.requests + kThreads - 1) / kThreads, r0 = min(tid * per, a.requests), r1 = min(r0 + per, a.requests);
  int my_items = 0, my_units = 0;
  bool falls = false;
  for (int r = r0; r < r1; ++r) {
    const Req q = request<kRows, 1, kCost>(a, a.start[r], a.start[r + 1], a.lens[r]);
    my_items += q.row_tiles * a.heads_kv;
    my_units += q.units;
    falls |= falling(a, r);
  }
  falls = __any(falls);
  if (lane == 0) fallen[wave] = falls;
  int before_i, before_u;
  int items = sum_before<kWaves>(my_items, scan_i, &before_i), units = sum_before<kWaves>(my_units, scan_u, &before_u);
  if (fallen[0] || fallen[1] || fallen[2] || fallen[3]) items = units = 0;
  if (a.zero_rest) clear_rest(a, D);
  if (w < split_wgs && tid == 0) split[w].rows = 0;
  // 16 requests of 8,000 keys, 128 items: cut 150 us, whole 247; from 3/4 of the resident workgroups on, the joins
  // cost more than the last round's idle ones.
  const bool by_items = items >= 3 * (int)gridDim.x / 4;
  const int G = by_items ? gridDim.x : max(1, min(split_wgs, units / kLeast));
  if (w >= G) return;
  const int share = by_items ? 1 : divide(units, G), more = by_items ? 0 : units - share * G;
  // Whole items in an order that puts the longest (a request's last row tiles) first, and lets a CU's second
  // workgroup have a short one where its first has a long one.
  int u = by_items ? w : share * w + min(w, more);
  const int u_end = by_items ? items : u + share + (w < more), stride = by_items ? gridDim.x : 0;
  if (by_items && items <= (int)gridDim.x && w >= (int)gridDim.x / 2) u = items - 1 - (w - (int)gridDim.x / 2);
  if (by_items && w >= items) return;
  if (u >= u_end) return;
  const int mine = by_items ? my_items : my_units, before = by_items ? before_i : before_u;
  if (before <= u && u < before + mine) found_r = r0, found_before = before;
  __syncthreads();
  int r = __builtin_amdgcn_readfirstlane(found_r);
  int pre = __builtin_amdgcn_readfirstlane(found_before);
  auto at = [&](int i) { return request<kRows, 1, kCost>(a, uniform(a.start, i), uniform(a.start, i + 1), uniform(a.lens, i)); };
  Req rq = at(r);

  const Unpack unpack;
  const h2 k24 = {(_Float16)-24.f, (_Float16)-24.f};
  // Places, opaque and in units of what is read or written there. Packed: this lane's part of a token's K
  // codes, that token's scales, its column's V codes (lane groups: four 16-dimension tiles at a time) and
  // scales; f16: the rows it writes, and those it reads as operands.
  constexpr int WU = NB % 4 == 0 ? 4 : NB % 2 == 0 ? 2 : 1;  // words of a K read
  const int tok = lane >> 2, part = lane & 3;
  const uint32_t pk = in_reg((wave * GW + lane * NB) / WU);
  const uint32_t pks = in_reg(2 * (wave * GW + 4 * D) + tok * NB);                       // f16
  const uint32_t pv = in_reg((wave * GW + 2 * D) / 2 + 16 * q4 + l16);                   // i32x2
  const uint32_t pvs = in_reg((wave * GW + 17 * D / 4) / 4 + 2 * (q4 >> 1));             // u32x4
  const uint32_t kw = in_reg((16 * wave + tok) * KU + part), vw = in_reg((16 * q4 + l16) * VU + 2 * wave);
  const uint32_t kr = in_reg((16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3)) * KU + h), vr = in_reg(col * VU + 2 * h);

  for (; u < u_end;) {
    while (u >= pre + (by_items ? rq.row_tiles * a.heads_kv : rq.units)) {
      pre += by_items ? rq.row_tiles * a.heads_kv : rq.units;
      rq = at(++r);
    }
    int item, t0 = 0, t1 = rq.nt;
    int item_end = 0;
    if (by_items) {
      item = u - pre;
      u += stride;
    } else {
      item = divide(u - pre, rq.per_item);
      const int x0 = u - pre - item * rq.per_item, x1 = min(x0 + u_end - u, rq.per_item);
      t0 = max(x0 - kCost, 0), t1 = max(x1 - kCost, 0);
      item_end = u - x0 + rq.per_item;
      u += x1 - x0;
      if (t0 == t1) continue;
    }
    const bool is_whole = t0 == 0 && t1 == rq.nt, is_first = t0 == 0;
    const int tile = item / a.heads_kv, rt = rq.row_tiles - 1 - tile, kvh = item - tile * a.heads_kv;
    const int row0 = rt * kRows, rows = min(kRows, rq.n * group - row0);
    const int p_first = rq.len - rq.n + row0 / group, p_last = rq.len - rq.n + (row0 + rows - 1) / group;
    const int first_last = first_key(p_last, a.window), lowest = first_key(p_first, a.window);
    // the steps of this part that some row of the tile sees
    t0 = max(t0, lowest / kStep - rq.tile0);
    t1 = p_last < 0 ? t0 : min(t1, p_last / kStep - rq.tile0 + 1);
    const int32_t *table = a.table + (size_t)r * a.cols;
    const int lim = max(p_last, 0);
    auto key_of = [&](int t) { return min((rq.tile0 + t) * kStep + 16 * wave, lim); };  // past the last: its own granule
    auto page_of = [&](int t) { return uniform(table, key_of(t) >> a.shift); };
    auto load = [&](int t, int page, u32x4 *P) {
      const uint8_t *gr = granule_of(a, page, key_of(t), kvh, kv4_granule_bytes(D));
#pragma unroll
      for (int i = 0; i < GL; ++i) {  // the last one drawn back to the granule's end
        const int off = i < GL - 1 ? 1024 * i : kv4_granule_bytes(D) - 1024;
        lds_load16(gr, words(P) + wave * GW + off / 4, 16 * lane, off);
      }
    };

    // ---- queries, as in kv4_attention.hip
    // This lane's row, worked out where it is needed: held, it would not fit the registers of the steps.
    struct Row {
      int rho, token, head;
    };
    auto my_row = [&] {
      const int rho = 32 * wave + (int)(in_reg(threadIdx.x) & 31u), rr = row0 + min(rho, rows - 1), token = rr / group;
      return Row{rho, token, kvh * group + rr - token * group};
    };
    f16x8 qh[NS], ql[NS];
    float unit;
    {
      const Row q = my_row();
      const float *src = a.q + (size_t)(rq.token0 + q.token) * a.ldq + (size_t)q.head * D + 8 * h;
      uint32_t big = 0;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const float4 v0 = *reinterpret_cast<const float4 *>(src + 16 * s), v1 = *reinterpret_cast<const float4 *>(src + 16 * s + 4);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) big = max(big, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
      big = max(big, (uint32_t)__shfl_xor((int)big, 32));
      int e = 0;
      if (big < 0x7F800000u) (void)frexpf(__uint_as_float(big), &e);
      unit = ldexpf(1.f, max(e - 13 + a.ke, -120));
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const float4 v0 = *reinterpret_cast<const float4 *>(src + 16 * s), v1 = *reinterpret_cast<const float4 *>(src + 16 * s + 4);
        const float x[8] = {v0.x, v1.x, v0.y, v1.y, v0.z, v1.z, v0.w, v1.w};  // pairs of dimensions p, p + 4
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = ldexpf(x[j], 13 - e), y = __builtin_fmaf(v, a.kh, v * a.kl);
          qh[s][j] = (_Float16)y;
          ql[s][j] = (_Float16)(y - (float)qh[s][j]);
        }
      }
    }
    f32x16 o[NB];
    float m = -__builtin_inff(), l = 0.f;
    uint32_t taint = 0;  // blocks of 32 dimensions that are NaN
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

    // The unpack of this wave's granule of a step: K codes and scales, then rows; V's a turn of 64 dimensions.
    struct KRaw {
      uint32_t c[NB];
      _Float16 sc[NB];
    };
    auto read_k = [&](u32x4 *P) {
      KRaw k;
      if constexpr (WU == 4) {
#pragma unroll
        for (int b = 0; b < NB; b += 4) {
          const u32x4 v = P[pk + b / 4];
          k.c[b] = v[0], k.c[b + 1] = v[1], k.c[b + 2] = v[2], k.c[b + 3] = v[3];
        }
      } else if constexpr (WU == 2) {
        const uint64_t v = reinterpret_cast<const uint64_t *>(P)[pk];
        k.c[0] = (uint32_t)v, k.c[1] = (uint32_t)(v >> 32);
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) k.c[b] = words(P)[pk + b];
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) k.sc[b] = reinterpret_cast<const _Float16 *>(P)[pks + b];
      return k;
    };
    auto row = [&](const KRaw &k, int b) {
      const h2 s2 = {k.sc[b], k.sc[b]}, c8 = s2 * k24;
      return unpack(k.c[b], s2, s2, s2, s2, c8, c8, c8, c8);
    };
    struct VRaw {
      i32x2 c;
      u32x4 sa, sb;
    };
    constexpr int JV = (NB + 1) / 2;
    auto v_here = [&](int j) { return NB % 2 == 0 || j < NB / 2 || q4 < 2; };  // 96 dimensions: half a second turn
    auto read_v = [&](u32x4 *P, int j) {
      const bool real = v_here(j);
      const uint32_t a_v = pv + (real ? 64 * j : 0), a_s = pvs + (real ? 4 * j : 0);
      VRaw v;
      v.c = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2 *)(reinterpret_cast<i32x2 *>(P) + a_v));
      v.sa = P[a_s], v.sb = P[a_s + 1];
      return v;
    };
    auto column = [&](const VRaw &v, int j) {
      h2 sv[8], cv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sv[i] = as_h2(i < 4 ? v.sa[i] : v.sb[i - 4]);
        cv[i] = sv[i] * k24;
      }
      const f16x8 x = unpack((uint32_t)v.c.x, sv[0], sv[1], sv[2], sv[3], cv[0], cv[1], cv[2], cv[3]);
      const f16x8 y = unpack((uint32_t)v.c.y, sv[4], sv[5], sv[6], sv[7], cv[4], cv[5], cv[6], cv[7]);
      if (v_here(j)) {
        VF[vw + 64 * VU * j] = __builtin_bit_cast(u32x4, x);
        VF[vw + 64 * VU * j + 1] = __builtin_bit_cast(u32x4, y);
      }
    };
    // What one wave wrote to LDS another reads past this.
    auto meet = [] {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    auto landed = [] {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      asm volatile("" ::: "memory");
    };

    // One step, in two halves with a meeting after each: Q K^T, beside it the unpack of this step's V and the
    // next one's K; then the softmax and P V, with the next K's write. So every unpack runs beside matrix
    // instructions, one buffer of each operand is enough, and P is free for the step after the next.
    auto step = [&](int t, u32x4 *P, u32x4 *next) {
      const int k0 = (rq.tile0 + t) * kStep;
      const bool whole = k0 >= first_last && k0 + kStep - 1 <= p_first;
      landed();
      const int page = page_of(min(t + 2, t1 - 1));
      if (!whole) {  // as in kv4_attention.hip: what some row does not see counts as 0, or NaN by the sums
        _Float16 *s = reinterpret_cast<_Float16 *>(P);
        const uint32_t psan = in_reg(2 * (wave * GW + 17 * D / 4) + kv4_v_place(threadIdx.x & 15));
        uint32_t bad = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {  // (four lanes to a token, with the same; masks of lanes would need scalar registers)
          const _Float16 v = s[psan + 16 * b];
          const bool odd = !(fabsf((float)v) <= kMaxScale);
          s[psan + 16 * b] = odd ? (_Float16)0.f : v;
          bad |= odd ? 1u << b : 0;
        }
        bad_blocks[t & 1][16 * wave + (threadIdx.x & 15)] = (uint8_t)bad;
        asm volatile("" ::: "memory");
      }
      f32x16 s[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
      // operands are read one step ahead of their instructions; the barriers keep the order written here
      f16x8 ka = __builtin_bit_cast(f16x8, KF[kr]), kb = __builtin_bit_cast(f16x8, KF[kr + 32 * KU]);
      VRaw vraw;
      KRaw kraw;
      f16x8 knext[NB];
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        const int f = min(e + 1, NS - 1);
        const u32x4 n0 = KF[kr + 2 * f], n1 = KF[kr + 32 * KU + 2 * f];
        if (e < 2 * JV && e % 2 == 0) vraw = read_v(P, e / 2);
        if (e == 2 * JV - 1) kraw = read_k(next);
        __builtin_amdgcn_sched_barrier(0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qh[e], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kb, qh[e], s[1], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, ql[e], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kb, ql[e], s[1], 0, 0, 0);
        if (e < 2 * JV && e % 2 == 1) column(vraw, e / 2);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          if (e == 2 * JV + b / 2) knext[b] = row(kraw, b);
        ka = __builtin_bit_cast(f16x8, n0);
        kb = __builtin_bit_cast(f16x8, n1);
        __builtin_amdgcn_sched_barrier(0);
      }
      meet();
#pragma unroll
      for (int b = 0; b < NB; ++b) KF[kw + 4 * b] = __builtin_bit_cast(u32x4, knext[b]);
      if (t + 2 < t1) load(t + 2, page, P);
      if (!whole) {
        const Row q = my_row();
        const int pos = q.rho < rows ? rq.len - rq.n + q.token : INT32_MAX, first = q.rho < rows ? first_key(pos, a.window) : 0;
        const uint64_t seen = keys_between(first - k0, pos - k0);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const int mine = (int)(seen >> (32 * kt)) >> (16 * h);
#pragma unroll
          for (int i = 0; i < 16; ++i) {  // by bits: masks of lanes would take the scalar registers from the whole loop
            const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe(mine, i, 1);
            s[kt][i] = __uint_as_float((__float_as_uint(s[kt][i]) & keep) | (0xFF800000u & ~keep));
          }
        }
        const uint32_t bad = bad_blocks[t & 1][lane];
        if (__any(bad != 0)) {
#pragma unroll 1
          for (int d = 0; d < NB; ++d)
            if (__ballot((bad >> d) & 1) & seen) taint |= 1u << d;
        }
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
      mx = over_halves(mx, [](float p, float q) { return fmaxf(p, q); });
      if (__any(mx > m)) {
        const float f = mx > m ? exp2_fast((m - mx) * unit) : 1.f;
        m = fmaxf(m, mx);
        l *= f;
#pragma unroll
        for (int d = 0; d < NB; ++d) o[d] *= f;
      }
      const float bias = m == -__builtin_inff() ? kBias : __builtin_fmaf(-m, unit, kBias);
      // Sixteen keys' weights at a time, in four parts, made while the matrix instructions of the sixteen
      // before run.
      u32x4 hi[4], lo[4];
      auto weights = [&](int n, int i) {
        const int kt = n >> 1, v = n & 1;
        const float e0 = exp2_fast(__builtin_fmaf(s[kt][8 * v + i], unit, bias)), e1 = exp2_fast(__builtin_fmaf(s[kt][8 * v + 4 + i], unit, bias));
        l += e0;
        l += e1;
        const h2 p = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e0, e1));
        hi[n][i] = as_u(p);
        lo[n][i] = as_u(__builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e0 - (float)p.x, e1 - (float)p.y)));
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) weights(0, i);
      auto values = [&](int j) { return __builtin_bit_cast(f16x8, VF[vr + 32 * VU * (j % NB) + 4 * ((j / NB) >> 1) + ((j / NB) & 1)]); };
      f16x8 x = values(0), before;
#pragma unroll
      for (int j = 0; j <= 4 * NB; ++j) {  // the hi terms of a value tile and the lo terms of the one before
        const int n = j / NB, d = j % NB;
        const f16x8 y = j + 1 < 4 * NB ? values(j + 1) : x;
        __builtin_amdgcn_sched_barrier(0);
        if (j < 4 * NB) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, __builtin_bit_cast(f16x8, hi[n]), o[d], 0, 0, 0);
        if (j > 0) {
          const int u = (j - 1) / NB, c = (j - 1) % NB;
          o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(before, __builtin_bit_cast(f16x8, lo[u]), o[c], 0, 0, 0);
        }
        if (n < 3) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i * NB / 4 == d) weights(n + 1, i);
        }
        before = x;
        x = y;
        __builtin_amdgcn_sched_barrier(0);
      }
      meet();
    };
    if (t0 < t1) {
      load(t0, page_of(t0), P0);
      landed();
      if (t0 + 1 < t1) load(t0 + 1, page_of(t0 + 1), P1);
      const KRaw k = read_k(P0);
#pragma unroll
      for (int b = 0; b < NB; ++b) KF[kw + 4 * b] = __builtin_bit_cast(u32x4, row(k, b));
      meet();
    }
    for (int t = t0; t < t1; t += 2) {
      step(t, P0, P1);
      if (t + 1 < t1) step(t + 1, P1, P0);
    }

    // ---- this lane's part of its row: dimensions 32 d + 8 i + 4 h and the next three
    const Row q = my_row();
    l = over_halves(l, [](float p, float q) { return p + q; });
    if (__any(taint != 0)) {
#pragma unroll
      for (int d = 0; d < NB; ++d) o[d] += (taint >> d) & 1 ? __builtin_nanf("") : 0.f;
    }
    if (q.rho < rows) {
      if (is_whole) {
        const float f = l == 0.f ? 0.f : 4.f / l;
        f32x4 *out = reinterpret_cast<f32x4 *>(a.out + ((size_t)(rq.token0 + q.token) * a.heads + q.head) * D);
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4 y = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * f;
            if (l == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
            out[8 * d + 2 * i + h] = y;
          }
      } else {
        const size_t slot = 2 * (size_t)w + is_first, at = slot * kRows + q.rho;
        f32x4 *out = reinterpret_cast<f32x4 *>(part_o + at * D);
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) out[8 * d + 2 * i + h] = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (h == 0) {
          part_ml[2 * at] = m == -__builtin_inff() ? m : m * unit;
          part_ml[2 * at + 1] = l;
        }
      }
    }
    if (!is_whole && is_first && tid == 0) {
      const int v = item_end - 1, big_end = (share + 1) * more;  // whose unit the item's last is
      const int last = v < big_end ? divide(v, share + 1) : more + divide(v - big_end, share);
      split[w] = Split{rows, w, last, rq.token0, kvh, row0};
    }
  }
}

// An item that several workgroups worked on: their parts in order, weighted by 2^(m - max). D / 4 lanes have a
// row and read its parts eight at a time; blockIdx.y takes so many rows of the item. 128 items of 128 rows in 256
// parts: 12 us, 33 MB.
template <int D>
__global__ __launch_bounds__(kThreads) void kv4_join_rows_kernel(Attend a, const Split *__restrict__ split, const float *__restrict__ part_o,
                                                                 const float *__restrict__ part_ml) {
  constexpr int L4 = D / 4, kAtOnce = kThreads / L4, AHEAD = 8;
  const Split s = split[blockIdx.x];
  const int x = threadIdx.x % L4, mine = threadIdx.x / L4, rho = blockIdx.y * kAtOnce + mine;
  if (mine >= kAtOnce || rho >= s.rows) return;
  const int parts = s.last - s.first + 1;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; p += AHEAD) {
    float pm[AHEAD], pl[AHEAD];
    f32x4 y[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      // past the last: the last again, at no weight (a branch here would wait for each load)
      const size_t at = (2 * (size_t)min(s.first + p + j, s.last) + (p + j == 0)) * kRows + rho;
      pm[j] = part_ml[2 * at], pl[j] = part_ml[2 * at + 1];
      y[j] = reinterpret_cast<const f32x4 *>(part_o + at * D)[x];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (p + j >= parts) pm[j] = -__builtin_inff(), pl[j] = 0.f, y[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = m;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) top = fmaxf(top, pm[j]);
    const float z = top == -__builtin_inff() ? 0.f : top, f = exp2_fast(m - z);
    m = top, l *= f, o *= f;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const float e = exp2_fast(pm[j] - z);
      l += e * pl[j];
      o += e * y[j];
    }
  }
  const int group = a.heads / a.heads_kv, rr = s.row0 + rho, tok = rr / group, h = s.kvh * group + rr - tok * group;
  f32x4 y = o * (4.f / l);
  if (l == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
  reinterpret_cast<f32x4 *>(a.out + ((size_t)(s.token0 + tok) * a.heads + h) * D)[x] = y;
}

template <int D>
int run(const char *who, const Attend &a) {
  // The workgroups that stay resident; runs of units go to half as many (their parts are 64 KB each).
  const int grid = 2 * cu_count(), split_wgs = cu_count();
  const size_t sb = ((size_t)split_wgs * sizeof(Split) + 255) & ~(size_t)255, mb = (size_t)split_wgs * 2 * kRows * 8;
  uint8_t *ws = (uint8_t *)workspace(sb + mb + (size_t)split_wgs * 2 * kRows * D * 4);
  if (!ws) return FHIP_ENOMEM;
  Split *split = (Split *)ws;
  float *ml = (float *)(ws + sb), *po = (float *)(ws + sb + mb);
  kv4_prefill_kernel<D><<<grid, kThreads, 0, stream()>>>(a, split, po, ml, split_wgs);
  FHIP_CHECK_LAUNCH(who);
  // Whether an item was cut is known on the device only.
  constexpr int kAtOnce = kThreads / (D / 4);
  kv4_join_rows_kernel<D><<<dim3(split_wgs, (kRows - 1) / kAtOnce + 1), kThreads, 0, stream()>>>(a, split, po, ml);
  FHIP_CHECK_LAUNCH(who);
  return FHIP_OK;
}

}  // namespace

namespace fhip {
int kv4_prefill(const char *who, int D, const Attend &a) {
  if (D == 64) return run<64>(who, a);
  if (D == 96) return run<96>(who, a);
  return run<128>(who, a);
}
}  // namespace fhip
