// Paged key/value cache held in 4 bits: page tables and slots from request lengths, norm + rotation + quantised store,
// attention over the pages, rows back as values.  Layout and rules: include/seedless_hip.h.
//
// Everything here only enqueues on the caller's stream.  What is read on the device (lengths, tables, slots) is checked
// on the device: an index that leaves its array is never followed.
#include "sl_device.cuh"
#include "../../include/seedless_hip.h"
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

using namespace sl;

namespace {

// ---- layout -----------------------------------------------------------------------------------------------------------
struct Pool {
  unsigned char* pages;
  int n_pages, page_shift, n_kv;      // page_size = 1 << page_shift
};
template <int D>
SL_DEV size_t head_bytes(const Pool& p) { return (size_t)(9 * D / 8) << p.page_shift; }
// First byte of a head's part of a page: key codes, key scales, value codes, value scales.
template <int D>
SL_DEV unsigned char* head_at(const Pool& p, int page, int h) {
  return p.pages + ((size_t)page * p.n_kv + h) * head_bytes<D>(p);
}
template <int D>
SL_DEV int key_codes_at(int off, int d) { return off * (D / 2) + ((d % 64) / 16) * (D / 8) + (d / 64) * 8 + (d % 16) / 2; }
template <int D>
SL_DEV int value_codes_at(int off, int d) { return (((off >> 3) * 16 + d / (D / 16)) * 8 + (off & 7)) * (D / 32) + (d % (D / 16)) / 2; }

// ---- element types ------------------------------------------------------------------------------------------------------
SL_DEV float bf2f(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
SL_DEV uint16_t f2bf(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }      // to nearest, ties to even: one instruction here
template <bool BF>
SL_DEV float elem_f(uint16_t u) { return BF ? bf2f(u) : h2f(u); }
template <bool BF>
SL_DEV uint16_t f_elem(float x) { return BF ? f2bf(x) : f2h(x); }
template <bool BF>
SL_DEV void elems4(uint2 r, float* x) {
  x[0] = elem_f<BF>((uint16_t)r.x); x[1] = elem_f<BF>((uint16_t)(r.x >> 16));
  x[2] = elem_f<BF>((uint16_t)r.y); x[3] = elem_f<BF>((uint16_t)(r.y >> 16));
}
template <bool BF>
SL_DEV void load4(const uint16_t* p, float* x) { elems4<BF>(*reinterpret_cast<const uint2*>(p), x); }

// ---- page tables, slots and row offsets -----------------------------------------------------------------------------------
constexpr int PLAN_MAX_REQ = 4096;
constexpr int PLAN_THREADS = 512;

// Sums in front of the caller's value over the workgroup, with sums capped at `cap` (the cap of a sum of capped sums is
// the cap of the sum).  Returns the sum before this thread; `total` the sum of all.
SL_DEV unsigned scan_before(unsigned v, unsigned cap, unsigned* s_wave, unsigned& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned y = (unsigned)__shfl_up((int)x, d);
    if (lane >= d) x = min(cap, x + y);
  }
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  unsigned before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 64; ++w) {
    const unsigned s = s_wave[w];
    if (w < wave) before = min(cap, before + s);
    all = min(cap, all + s);
  }
  __syncthreads();
  total = all;
  const unsigned y = (unsigned)__shfl_up((int)x, 1);
  return lane ? min(cap, before + y) : before;
}
// Largest r with first[r] <= x, for first[0] = 0 <= x (of equal entries the last: requests without a share are stepped over).
SL_DEV int owner_of(const int* first, int n, int x) {
  int lo = 0, hi = n;                     // first[lo] <= x < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Every workgroup forms the running sums over the requests (rows; pages missing and pages given back) for itself, in LDS, and then
// fills its share of the outputs: one launch, no exchange between workgroups.  The requests' numbers are 12 bytes each and
// come from L2; up to 64 requests are one wave's work, without a barrier.  A few KB: bound by the launch and three dependent trips to
// memory (32 requests 4.5 us), with many requests by the sums that every workgroup repeats (1024 requests of up to 32K
// tokens 13 us, of which the table's rows take 4).
__global__ __launch_bounds__(PLAN_THREADS) void k_kv4_plan(sl_kv4_plan_args a, int page_shift) {
  __shared__ int s_row[PLAN_MAX_REQ + 1], s_need[PLAN_MAX_REQ + 1], s_give[PLAN_MAX_REQ + 1];
  __shared__ unsigned s_wave[PLAN_THREADS / 64];
  __shared__ unsigned s_fit[PLAN_MAX_REQ / 32];     // the request is served
  __shared__ unsigned s_taken, s_unserved;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n_req, page = 1 << page_shift;
  const int W = a.table_width;
  const unsigned cap = (unsigned)a.max_tokens;
  const unsigned count = (unsigned)min(max(a.free_count_in[0], 0), a.n_free);
  for (int i = tid; i < (n + 31) / 32; i += PLAN_THREADS) s_fit[i] = 0;
  if (tid == 0) s_taken = s_unserved = 0;

  // pages that a request misses and gives back, as far as its numbers make sense
  auto pages_of = [&](int ctx, int nw, int held, unsigned row, unsigned& need, unsigned& give) {
    const long total = (long)ctx + nw;
    const bool fits = (unsigned)max(nw, 0) <= cap - row;
    need = give = 0;
    if (!(ctx >= 0 && nw >= 0 && fits && held >= 0 && held <= W && total <= ((long)W << page_shift) && ctx <= ((long)held << page_shift))) return false;
    const int want = (int)((total + page - 1) >> page_shift);
    need = (unsigned)max(want - held, 0); give = (unsigned)max(held - want, 0);
    return true;
  };
  unsigned all_rows, all_need, all_give;
  if (n <= 64) {
    __syncthreads();
    if (wave == 0) {
      const bool there = lane < n;
      const int ctx = there ? a.ctx_len[lane] : 0, nw = there ? a.new_len[lane] : 0, held = there ? a.held_in[lane] : 0;
      unsigned x = min(cap, (unsigned)max(nw, 0));
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { const unsigned y = (unsigned)__shfl_up((int)x, d); if (lane >= d) x = min(cap, x + y); }
      unsigned row = (unsigned)__shfl_up((int)x, 1);
      if (lane == 0) row = 0;
      unsigned need, give;
      const bool sane = pages_of(ctx, nw, held, row, need, give) && there;
      unsigned nb = need, gb = give;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const unsigned y = (unsigned)__shfl_up((int)nb, d), z = (unsigned)__shfl_up((int)gb, d);
        if (lane >= d) { nb += y; gb += z; }
      }
      const unsigned give_all = (unsigned)__shfl((int)gb, 63), have = count + give_all;
      const bool fit = sane && (need == 0 || nb <= have);
      if (there) { s_row[lane] = (int)row; s_need[lane] = (int)(nb - need); s_give[lane] = (int)(gb - give); }
      unsigned taken = fit ? need : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) taken += (unsigned)__shfl_xor((int)taken, d);
      const unsigned long long fits = __ballot(fit);
      if (lane == 63) {
        s_row[n] = (int)x; s_need[n] = (int)nb; s_give[n] = (int)gb;
        s_taken = taken; s_unserved = (unsigned)(n - __popcll(fits));
        if (n > 0) s_fit[0] = (unsigned)fits;
        if (n > 32) s_fit[1] = (unsigned)(fits >> 32);
      }
    }
    __syncthreads();
    all_rows = (unsigned)s_row[n]; all_give = (unsigned)s_give[n];
  } else {
    const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS;
    unsigned rows = 0;
    for (int j = 0; j < per; ++j) {
      const int r = tid * per + j;
      if (r < n) rows = min(cap, rows + min(cap, (unsigned)max(a.new_len[r], 0)));
    }
    unsigned row = scan_before(rows, cap, s_wave, all_rows);
    unsigned need_sum = 0, give_sum = 0, need, give;
    unsigned at_row = row;
    for (int j = 0; j < per; ++j) {
      const int r = tid * per + j;
      if (r >= n) continue;
      const int nw = a.new_len[r];
      pages_of(a.ctx_len[r], nw, a.held_in[r], at_row, need, give);
      at_row = min(cap, at_row + min(cap, (unsigned)max(nw, 0)));
      need_sum += need; give_sum += give;
    }
    unsigned nb = scan_before(need_sum, 0x7fffffffu, s_wave, all_need);
    unsigned gb = scan_before(give_sum, 0x7fffffffu, s_wave, all_give);
    const unsigned have = count + all_give;
    unsigned taken = 0, unserved = 0;
    for (int j = 0; j < per; ++j) {
      const int r = tid * per + j;
      if (r >= n) continue;
      const int nw = a.new_len[r];
      const bool sane = pages_of(a.ctx_len[r], nw, a.held_in[r], row, need, give);
      s_row[r] = (int)row; s_need[r] = (int)nb; s_give[r] = (int)gb;
      if (sane && (need == 0 || nb + need <= have)) { atomicOr(&s_fit[r >> 5], 1u << (r & 31)); taken += need; }
      else ++unserved;
      row = min(cap, row + min(cap, (unsigned)max(nw, 0)));
      nb += need; gb += give;
    }
    if (taken) atomicAdd(&s_taken, taken);               // (whole numbers: in any order)
    if (unserved) atomicAdd(&s_unserved, unserved);
    if (tid == 0) { s_row[n] = (int)all_rows; s_need[n] = (int)all_need; s_give[n] = (int)all_give; }
    __syncthreads();
  }

  const int have = (int)(count + all_give), left = have - (int)s_taken;
  auto fit = [&](int r) { return (s_fit[r >> 5] >> (r & 31)) & 1u; };
  // entry x of the free list with the pages given back behind it
  auto free_at = [&](int x) {
    if (x < (int)count) return a.free_in[x];
    const int k = x - (int)count, r = owner_of(s_give, n, k);
    return a.table_in[(size_t)r * W + (a.held_in[r] - (s_give[r + 1] - s_give[r])) + (k - s_give[r])];
  };
  // page c of request r in the new table
  auto page_at = [&](int r, int c, int held) {
    const int need_r = s_need[r + 1] - s_need[r];
    if (c < held - (s_give[r + 1] - s_give[r])) return a.table_in[(size_t)r * W + c];
    if (c >= held && c < held + need_r && fit(r)) return free_at(have - 1 - s_need[r] - (c - held));
    return -1;
  };
  const int step = gridDim.x * PLAN_THREADS, at = blockIdx.x * PLAN_THREADS + tid;
  for (int r = blockIdx.x; r < n; r += gridDim.x) {      // a workgroup per row of the table
    const int held = min(max(a.held_in[r], 0), W), need_r = fit(r) ? s_need[r + 1] - s_need[r] : 0, kept = held - (s_give[r + 1] - s_give[r]);
    const int32_t* from = a.table_in + (size_t)r * W;
    int32_t* to = a.table_out + (size_t)r * W;
    const int top = have - 1 - s_need[r] + held;
#pragma unroll 4
    for (int c = tid; c < W; c += PLAN_THREADS) {
      int id = -1;
      if (c < kept) id = from[c];
      else if (c >= held && c < held + need_r) id = free_at(top - c);
      to[c] = id;
    }
    if (tid == 0) {
      a.held_out[r] = kept + need_r;
      a.kv_len[r] = fit(r) ? a.ctx_len[r] + a.new_len[r] : 0;
      a.q_start[r] = s_row[r];
    }
  }
  for (int i = at; i < a.n_free; i += step) a.free_out[i] = i < left ? free_at(i) : -1;
  for (int t = at; t < a.max_tokens; t += step) {
    int slot = -1, pos = 0;
    if (t < (int)all_rows) {
      const int r = owner_of(s_row, n, t);
      pos = (int)((unsigned)a.ctx_len[r] + (unsigned)(t - s_row[r]));
      if (fit(r)) {
        const int id = page_at(r, pos >> page_shift, a.held_in[r]);      // (a table may hold anything: no id turns into another's slot)
        if (id >= 0 && id <= (0x7fffffff >> page_shift)) slot = (id << page_shift) + (pos & (page - 1));
      }
    }
    a.slot[t] = slot; a.pos[t] = pos;
  }
  if (at == 0) { a.q_start[n] = (int)all_rows; a.free_count_out[0] = min(left, a.n_free); a.unserved[0] = (int)s_unserved; }
}

// ---- norm, rotation, quantised store ----------------------------------------------------------------------------------------
// Double-precision counterparts of the lane reductions: DPP moves the two halves of a value.
template <int CTRL>
SL_DEV double dpp_d(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned long long lo = dpp_u<CTRL>((uint32_t)u), hi = dpp_u<CTRL>((uint32_t)(u >> 32));
  return __builtin_bit_cast(double, lo | (hi << 32));
}
template <class F>
SL_DEV double row16(double v, F f) {                  // over the 16 lanes of a row
  v = f(v, dpp_d<DPP_XOR1>(v)); v = f(v, dpp_d<DPP_XOR2>(v));
  v = f(v, dpp_d<DPP_HALF_MIRROR>(v)); return f(v, dpp_d<DPP_MIRROR>(v));
}
template <int LANES>
SL_DEV double sum_lanes(double v) {
  v = row16(v, [](double a, double b) { return a + b; });
  if (LANES >= 32) v = v + __shfl_xor(v, 16);
  if (LANES >= 64) v = v + __shfl_xor(v, 32);
  return v;
}
template <int LANES>
SL_DEV float sum_lanes(float v) { return tree_sum<LANES>(v); }
SL_DEV float inv_sqrt(float x) { return __builtin_amdgcn_rsqf(x); }
// (Not a shorter form: where a group's largest is the opposite of its smallest, the last bit decides between 7 and 8 steps.  An estimate with two
// Newton steps, within 2^-51, gave 1-2 % of such rows another scale than x * rsqrt(mean + eps) * weight in doubles has, at the same speed.)
SL_DEV double inv_sqrt(double x) { return rsqrt(x); }

// What a lane needs of a token beside its row: four weights, four cosines and sines, and from which lane the other half comes.
struct Turn {
  float w[4], c[4], s[4];
  int from;
  bool norm, low, turns;
};
template <int D, bool BF>
SL_DEV Turn turn_of(const uint16_t* weight, const float* cos_t, const float* sin_t, int half, int pos, int l) {
  Turn u;
  const int lane = threadIdx.x & 63, hl = half / 4;     // a half of the rotated dims, in lanes
  u.norm = weight != nullptr; u.low = l < hl; u.turns = l < 2 * hl;
  u.from = u.turns ? (u.low ? lane + hl : lane - hl) : lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) { u.w[i] = 1.0f; u.c[i] = 1.0f; u.s[i] = 0.0f; }
  if (weight) load4<BF>(weight + 4 * l, u.w);
  if (u.turns) {
    const size_t row = (size_t)pos * half + 4 * (u.low ? l : l - hl);
    const float4 c = *reinterpret_cast<const float4*>(cos_t + row), s = *reinterpret_cast<const float4*>(sin_t + row);
    u.c[0] = c.x; u.c[1] = c.y; u.c[2] = c.z; u.c[3] = c.w;
    u.s[0] = s.x; u.s[1] = s.y; u.s[2] = s.z; u.s[3] = s.w;
  }
  return u;
}
// A head row over D/4 lanes, four consecutive dims each: norm and rotation in precision F.
template <class F, int D>
SL_DEV void turn_row(F* x, const Turn& u, int half, double eps) {
  if (u.norm) {
    const F inv = inv_sqrt(sum_lanes<D / 4>((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) * (F)(1.0 / D) + (F)eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * (F)u.w[i];
  }
  if (half) {
    F y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __shfl(x[i], u.from);
    if (u.turns) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = u.low ? x[i] * (F)u.c[i] - y[i] * (F)u.s[i] : x[i] * (F)u.c[i] + y[i] * (F)u.s[i];
    }
  }
}

// The four codes of this lane (16 lanes = one group of 64 dims), low nibble first, and the group's scale and bias.
// Double precision decides: a value next to the border of two codes takes the side that exact arithmetic takes.  Codes are
// formed in fp32 with one reciprocal and only those formed again by a double division that lie so near a border that fp32 could
// be wrong: with t = (x - b) / s its error stays below (|x| + |b|) / |s| * 2^-21 + 2^-18 (three roundings of x, b and the
// difference, each within 2^-24 of their size, the reciprocal's and the product's on |t| < 16).
SL_DEV float row16_f(float v, bool least) {
  auto f = [&](float a, float b) { return least ? fminf(a, b) : fmaxf(a, b); };
  v = f(v, dpp_f<DPP_XOR1>(v)); v = f(v, dpp_f<DPP_XOR2>(v));
  v = f(v, dpp_f<DPP_HALF_MIRROR>(v)); return f(v, dpp_f<DPP_MIRROR>(v));
}
// Least and largest of a group: fp32 values (what comes in as halves is exact there) or doubles.
SL_DEV void group_range(const float* x, double& mn, double& mx) {
  mn = (double)row16_f(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), true);
  mx = (double)row16_f(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), false);
}
SL_DEV void group_range(const double* x, double& mn, double& mx) {
  mn = row16(fmin(fmin(x[0], x[1]), fmin(x[2], x[3])), [](double a, double b) { return fmin(a, b); });
  mx = row16(fmax(fmax(x[0], x[1]), fmax(x[2], x[3])), [](double a, double b) { return fmax(a, b); });
}
template <class F>
SL_DEV uint32_t quantise4(const F* v, uint32_t& sb) {
  const F lim = (F)65504.0;
  F x[4];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bad = bad || !(fabs(v[i]) <= (F)1e300 && fabs(v[i]) < (F)__builtin_inf());
    x[i] = v[i] < -lim ? -lim : (v[i] > lim ? lim : v[i]);
  }
  double mn, mx;
  group_range(x, mn, mx);
  const unsigned long long bads = __ballot(bad);
  if ((bads >> (threadIdx.x & 48)) & 0xffffull) { sb = 0x7e007e00u; return 0; }
  const bool low = fabs(mn) > fabs(mx);
  double scale = fmax((mx - mn) * (1.0 / 15.0), 1e-7);
  scale = low ? scale : -scale;
  const double edge = low ? mn : mx, steps = rint(edge / scale);
  double bias = 0.0;
  if (steps != 0.0) { scale = edge / steps; bias = edge; }
  const uint16_t hs = f2h((float)scale), hb = f2h((float)bias);
  sb = (uint32_t)hs | ((uint32_t)hb << 16);
  const float s = h2f(hs), b = h2f(hb), inv = 1.0f / s;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = (float)x[i], t = (f - b) * inv, near = fmaf((fabsf(f) + fabsf(b)) * fabsf(inv), 4.76837158203125e-7f, 3.814697265625e-6f);
    float c = rintf(t);
    if (!(fabsf(fabsf(t - c) - 0.5f) > near)) c = (float)rint(((double)x[i] - (double)b) / (double)s);
    codes |= (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f) << (4 * i);
  }
  return codes;
}

// A wave per token and `per` times 256/D heads: D/4 lanes carry a head row.  blockIdx.y: runs of query heads, then of key heads, then
// of value heads; the token's weights and angles are loaded once for a run, the rows of four units ahead of their use.  Bound by the
// issue of vector instructions: 7.6K tokens of 32 + 8 heads of 128 dims 51 us (3400 instructions a token, half of them for the
// 16 rows that are quantised; 187 MB in and out at 3.6 TB/s), 2048 tokens of 16 + 2 heads of 256 dims 13 us, one token 3.6.
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_kv4_append(Pool pool, sl_kv4_append_args a, int q_units, int kv_units, int per) {
  constexpr int LANES = D / 4, HEADS = 64 / LANES, AHEAD = 4;
  const int lane = threadIdx.x & 63, l = lane % LANES, sub = lane / LANES;
  // neighbouring tokens on one XCD (workgroups go round the eight): their value codes lie in one line, in turns of D / 32 bytes
  const int block = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), t = block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= a.n_tokens) return;
  const int q_runs = (q_units + per - 1) / per, kv_runs = (kv_units + per - 1) / per;
  const int pos = a.rot_dim ? a.pos[t] : 0, half = a.rot_dim / 2;
  const bool placed = !a.rot_dim || (pos >= 0 && pos < a.max_pos);
  int run = blockIdx.y;
  if (run < q_runs) {
    const int u1 = min(q_units, (run + 1) * per);
    const uint16_t* src = (const uint16_t*)a.q + t * a.q_token + 4 * l;
    uint16_t* dst = (uint16_t*)a.q_out + t * a.out_token + 4 * l;
    const Turn turn = turn_of<D, BF>((const uint16_t*)a.q_weight, a.cos, a.sin, placed ? half : 0, pos, l);
    for (int u0 = run * per; u0 < u1; u0 += AHEAD) {
      uint2 raw[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int h = (u0 + j) * HEADS + sub;
        raw[j] = make_uint2(0, 0);
        if (u0 + j < u1 && h < a.n_heads && placed) raw[j] = *reinterpret_cast<const uint2*>(src + h * a.q_head);
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (u0 + j >= u1) break;
        const int h = (u0 + j) * HEADS + sub;           // (lanes without a head still take part in the exchanges)
        float x[4];
        elems4<BF>(raw[j], x);
        if (placed) turn_row<float, D>(x, turn, half, a.eps);
        if (h < a.n_heads)
          *reinterpret_cast<uint2*>(dst + h * a.out_head) =
              make_uint2((uint32_t)f_elem<BF>(x[0]) | ((uint32_t)f_elem<BF>(x[1]) << 16), (uint32_t)f_elem<BF>(x[2]) | ((uint32_t)f_elem<BF>(x[3]) << 16));
      }
    }
    return;
  }
  run -= q_runs;
  const int slot = a.slot[t];
  if (!placed || slot < 0 || (slot >> pool.page_shift) >= pool.n_pages) return;
  const bool key = run < kv_runs;
  if (!key) run -= kv_runs;
  const int u1 = min(kv_units, (run + 1) * per);
  const int off = slot & ((1 << pool.page_shift) - 1), part = (D / 2) << pool.page_shift, sbs = (D / 16) << pool.page_shift;
  unsigned char* page = head_at<D>(pool, slot >> pool.page_shift, 0) + (key ? 0 : part + sbs);
  const int codes_at = key ? key_codes_at<D>(off, 4 * l) : value_codes_at<D>(off, 4 * l);
  const uint16_t* src = key ? (const uint16_t*)a.k + t * a.k_token + 4 * l : (const uint16_t*)a.v + t * a.v_token + 4 * l;
  const int64_t stride = key ? a.k_head : a.v_head;
  Turn turn;
  if (key) turn = turn_of<D, BF>((const uint16_t*)a.k_weight, a.cos, a.sin, half, pos, l);
  for (int u0 = run * per; u0 < u1; u0 += AHEAD) {
    uint2 raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int h = (u0 + j) * HEADS + sub;
      raw[j] = make_uint2(0, 0);
      if (u0 + j < u1 && h < pool.n_kv) raw[j] = *reinterpret_cast<const uint2*>(src + h * stride);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (u0 + j >= u1) break;
      const int h = (u0 + j) * HEADS + sub;
      float x[4];
      elems4<BF>(raw[j], x);
      uint32_t sb, codes;
      if (key) {
        double y[4] = {x[0], x[1], x[2], x[3]};
        turn_row<double, D>(y, turn, half, a.eps);
        codes = quantise4(y, sb);
      } else codes = quantise4(x, sb);
      if (h >= pool.n_kv) continue;
      unsigned char* at = page + h * head_bytes<D>(pool);
      *reinterpret_cast<uint16_t*>(at + codes_at) = (uint16_t)codes;
      if (l % 16 == 0) reinterpret_cast<uint32_t*>(at + part)[off * (D / 64) + l / 16] = sb;
    }
  }
}

// ---- rows as values -----------------------------------------------------------------------------------------------------
// A lane takes four dims of a key row and of a value row; a workgroup 4096 / D rows of one head, four loads of each kind in flight.
// Bound by memory: 39K rows of 8 heads of 128 dims to fp32 78 us, 4.75 TB/s (one load in flight: 110); 500 rows of 2 heads 3.5 us.
template <int D, bool F16>
__global__ __launch_bounds__(256) void k_kv4_read(Pool pool, const int32_t* slots, int n, void* k_out, void* v_out) {
  constexpr int LANES = D / 4, ROWS = 256 / LANES, TURNS = 4;
  const int l = threadIdx.x % LANES, h = blockIdx.y;
  const int part = (D / 2) << pool.page_shift, sbs = (D / 16) << pool.page_shift, mask = (1 << pool.page_shift) - 1;
  const int row0 = blockIdx.x * (ROWS * TURNS) + threadIdx.x / LANES;
  int slot[TURNS];
  uint32_t codes[TURNS][2], sb[TURNS][2];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) slot[i] = row0 + i * ROWS < n ? slots[row0 + i * ROWS] : -1;
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const bool in = slot[i] >= 0 && (slot[i] >> pool.page_shift) < pool.n_pages;
    if (!in) slot[i] = -1;
    const int off = in ? slot[i] & mask : 0;
    const unsigned char* at = head_at<D>(pool, in ? slot[i] >> pool.page_shift : 0, h);
    codes[i][0] = *reinterpret_cast<const uint16_t*>(at + key_codes_at<D>(off, 4 * l));
    codes[i][1] = *reinterpret_cast<const uint16_t*>(at + part + sbs + value_codes_at<D>(off, 4 * l));
    sb[i][0] = reinterpret_cast<const uint32_t*>(at + part)[off * (D / 64) + l / 16];
    sb[i][1] = reinterpret_cast<const uint32_t*>(at + 2 * part + sbs)[off * (D / 64) + l / 16];
  }
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int row = row0 + i * ROWS;
    if (row >= n) return;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      void* out = kv ? v_out : k_out;
      if (!out) continue;
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (slot[i] >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(lo_h(sb[i][kv]), (float)((codes[i][kv] >> (4 * j)) & 15u), hi_h(sb[i][kv]));
      }
      const size_t to = ((size_t)row * pool.n_kv + h) * D + 4 * l;
      if (F16) *reinterpret_cast<uint2*>((uint16_t*)out + to) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
      else *reinterpret_cast<float4*>((float*)out + to) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
}

// ---- attention ------------------------------------------------------------------------------------------------------------
// Flash attention on the matrix cores (v_mfma_f32_16x16x32_f16), straight from the codes.  A wave takes 32 keys a step and
// 16 * NT query rows (row = token * group + head within the group):
//   S[key, row] = sum over groups of 64 dims of  s_g * (sum q c) + b_g * (sum q)      c = code
//   O[dim, row] += sum over keys of  (p s_g) * (c - 8)  +  p * (b_g + 8 s_g)
// Codes become fp16 operands without rounding: a masked nibble IS the fp16 number c * 2^-24 (or c * 2^-20 four bits up; the
// query's operand makes that good for the keys, the last step for the values).  So the scales meet fp32 scores.  Rounded to fp16 on the
// way, by half a step of 2^-11 each, are the operands p s_g, p and b_g + 8 s_g of the second line, and the softmax's sum is that of
// the rounded p, so that weights stay in proportion; the first meets c - 8 (the sums take the 8 off), which keeps its rounding at the size of a
// value's own spread.  Everything else, scores, maxima and sums, is fp32.  Queries become fp16 after a power of two per row that
// puts the largest near 2^10: exact for both element types but for dims 2^-20 below the row's largest.
// Layouts: S comes out with a lane holding 8 consecutive keys of one row, which is how the second product wants p, because
// row m of the two key operands is key 8 (m / 4) + m % 4 (+ 4).  Values are stored as a lane loads them (8 keys x D/16
// dims) and change lanes through LDS on their way, so that the 16 rows of an operand lie in one group and share p s_g.
// Each of the four waves of a workgroup takes every fourth step; their sums are joined in LDS at the end.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int AT_WAVES = 4, AT_STEP = 32, AT_UNIT = AT_WAVES * AT_STEP;   // keys of a workgroup's round
constexpr int AT_MAX_REQ = 4096;

// How the work of a call is cut.  An item is a row tile of a request and a key/value head; its rounds of 128 keys are shared
// out to as many workgroups as its cost (rounds, weighted by the row tile's width) holds shares, a share being the cost of the
// whole call over `want` workgroups.  So every workgroup has one part of one item: runs of equal length across items would need
// fewer workgroups, but one that ends an item and begins another pays the start and the end twice, and the call
// waits for it (32 lanes: 47 us where the others end at 35).  The host launches enough workgroups whatever the lengths are; those
// behind the last part leave at once, as do those whose rows see fewer keys than the request has.
struct AttnCut {
  int want;           // workgroups to share the cost out to
  int turns;          // how often the share may grow until there are no more than that
  int rows;           // rows of a partial sum
  int32_t* first;     // [n_req + 1] parts before each request, then share (written by the first workgroup, for the merge)
  float* part;        // partial sums by workgroup: [grid][rows][D], then maxima [grid][rows], sums [grid][rows]
  long slots;         // = grid
};
SL_DEV long seen_keys(const sl_kv4_attn_args& a, const Pool& pool, int r) {
  const long cap = (long)a.table_width << pool.page_shift;
  return max(0l, min((long)a.kv_len[r], cap));
}
// rows of request r that this call computes
SL_DEV int rows_of(const sl_kv4_attn_args& a, int r, int& start, int& n) {
  start = a.q_start[r];
  n = a.q_start[r + 1] - start;
  if (start < 0 || n <= 0 || start >= a.n_tokens) return 0;
  return min(min(n, a.max_rows), a.n_tokens - start);
}
SL_DEV int rounds_for(long keys) { return max(1, (int)((keys + AT_UNIT - 1) / AT_UNIT)); }
// Cost of a round: a workgroup of 32 rows takes 4/3 of the time where more than 16 of them are there (measured 72 against 55 us).
SL_DEV int round_cost(int tile_rows, int rows) { return tile_rows == 32 ? (rows > 16 ? 4 : 3) : 1; }
SL_DEV int parts_of(int rounds, int cost, int share) { return (int)(((unsigned)rounds * (unsigned)cost + (unsigned)share - 1u) / (unsigned)share); }
// cost of a part: total / want, rounded up (a quotient of doubles is exact where it is whole)
SL_DEV int share_of(long total, int want) { return max(1, (int)fmin(ceil((double)total / (double)want), 2147483647.0)); }
struct AttnPart { int r, tile, h, part, share; };
// What a request asks for: its items, its most and least rounds, their cost, and the sum of its items' costs (row tiles further up see
// fewer keys: their rounds lie evenly between the first tile's and the last's).
template <int TILE>
SL_DEV void request_work(const sl_kv4_attn_args& a, const Pool& pool, int r, int& items, int& rounds, int& least, int& cost, long& all) {
  int start, n;
  const int rows = rows_of(a, r, start, n), group = a.n_heads / pool.n_kv;
  items = rounds = least = 0; cost = 1; all = 0;
  if (rows <= 0) return;
  const int tiles = (rows * group + TILE - 1) / TILE;
  const long keys = seen_keys(a, pool, r);
  items = tiles * pool.n_kv; rounds = rounds_for(min(keys, keys - n + rows)); cost = round_cost(TILE, rows * group);
  least = tiles > 1 ? rounds_for(keys - n + min(rows, TILE / group + 1)) : rounds;
  all = (long)items * (rounds + least) * cost / 2;
}
// Rounds of a row tile and how they are cut: `parts` of `per` rounds (at most parts_of() of the request's most rounds).
template <int TILE>
SL_DEV void tile_cut(long keys, int n, int rows_total, int tile, int group, int share, long& last, int& parts, int& per) {
  const int end = min((tile + 1) * TILE, rows_total);             // rows in front of the tile's end
  last = max(0l, min(keys, keys - n + (end - 1) / group + 1));    // keys that its last row sees
  const int rounds = rounds_for(last);
  parts = parts_of(rounds, round_cost(TILE, rows_total), share);
  per = (rounds + parts - 1) / parts;
}
// The part that workgroup `idx` has; false if there is none.  Up to 64 requests: every wave finds it by itself, a request
// per lane; more: the workgroup with running sums in LDS (s_first: n_req + 1 words, s_tmp: 12 words).
template <int TILE>
SL_DEV bool find_part(const sl_kv4_attn_args& a, const Pool& pool, const AttnCut& cut, int idx, int* s_first, int* s_tmp, AttnPart& out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n_req;
  int before, items, rounds, least, cost, share;
  long all;
  // Rounding up makes more parts than were asked for, and a few more than the chip has places cost another turn: while the items
  // alone are fewer, the share grows until their parts are too (row tiles further up have parts for fewer keys).
  auto used = [&] { return items * (parts_of(rounds, cost, share) + parts_of(least, cost, share)); };       // twice the parts
  auto too_many = [&](int twice, int items_now) { return twice / 2 > cut.want && items_now < cut.want; };
  auto grown = [&](int twice) { return (int)fmin(ceil((double)share * (double)twice / (2.0 * (double)cut.want)), 2147483647.0); };
  if (n <= 64) {
    items = rounds = least = 0; cost = 1; all = 0;
    if (lane < n) request_work<TILE>(a, pool, lane, items, rounds, least, cost, all);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
    share = share_of(all, cut.want);
    for (int it = 0; it < cut.turns; ++it) {
      int twice = used(), all_items = items;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { twice += __shfl_xor(twice, d); all_items += __shfl_xor(all_items, d); }
      if (!too_many(twice, all_items)) break;
      share = grown(twice);
    }
    const int parts = parts_of(rounds, cost, share), own = items * parts;
    int upto = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int y = __shfl_up(upto, d); if (lane >= d) upto += y; }
    if (idx == 0 && wave == 0) {
      if (lane < n) cut.first[lane] = upto - own;
      if (lane == 63) { cut.first[n] = upto; cut.first[n + 1] = share; }
    }
    const int r = __popcll(__ballot(upto <= idx));
    if (r >= n) return false;                      // (lanes behind n hold the total as well)
    out.r = r;
    before = __builtin_amdgcn_readlane(upto - own, r); rounds = __builtin_amdgcn_readlane(parts, r); items = __builtin_amdgcn_readlane(items, r);
    share = __builtin_amdgcn_readfirstlane(share);
  } else {
    const int per = (n + 255) / 256;
    long total = 0;
    int all_items = 0;
    for (int j = 0; j < per; ++j) {
      const int r = tid * per + j;
      if (r < n) { request_work<TILE>(a, pool, r, items, rounds, least, cost, all); total += all; all_items += items; }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { total += __shfl_xor(total, d); all_items += __shfl_xor(all_items, d); }
    long* s_total = reinterpret_cast<long*>(s_tmp);
    if (lane == 0) { s_total[wave] = total; s_tmp[8 + wave] = all_items; }
    __syncthreads();
    total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    all_items = (s_tmp[8] + s_tmp[9]) + (s_tmp[10] + s_tmp[11]);
    share = share_of(total, cut.want);
    int at, sum;
    for (int it = 0;; ++it) {
      int own = 0, twice = 0;
      for (int j = 0; j < per; ++j) {
        const int r = tid * per + j;
        if (r < n) { request_work<TILE>(a, pool, r, items, rounds, least, cost, all); own += items * parts_of(rounds, cost, share); twice += used(); }
      }
      int upto = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) { const int y = __shfl_up(upto, d); if (lane >= d) upto += y; twice += __shfl_xor(twice, d); }
      __syncthreads();
      if (lane == 63) { s_tmp[wave] = twice; s_tmp[8 + wave] = upto; }
      __syncthreads();
      at = upto - own; sum = 0; twice = 0;
#pragma unroll
      for (int w = 0; w < AT_WAVES; ++w) { if (w < wave) at += s_tmp[8 + w]; sum += s_tmp[8 + w]; twice += s_tmp[w]; }
      if (it >= cut.turns || !too_many(twice, all_items)) break;
      share = grown(twice);
    }
    for (int j = 0; j < per; ++j) {
      const int r = tid * per + j;
      if (r < n) { request_work<TILE>(a, pool, r, items, rounds, least, cost, all); s_first[r] = at; at += items * parts_of(rounds, cost, share); }
    }
    if (tid == 0) s_first[n] = sum;
    __syncthreads();
    if (idx == 0) for (int i = tid; i <= n + 1; i += 256) cut.first[i] = i <= n ? s_first[i] : share;
    if (idx >= sum) return false;
    out.r = __builtin_amdgcn_readfirstlane(owner_of(s_first, n, idx));
    before = s_first[out.r];
    request_work<TILE>(a, pool, out.r, items, rounds, least, cost, all);
    rounds = parts_of(rounds, cost, share);
  }
  // (rounds: from here on the most parts of an item.)  Workgroups go round the eight XCDs in turn: eight items side by side, part
  // after part, so that every XCD gets items of all lengths and their later parts, which the shorter items lack, alike.
  const int in = idx - before, full = items & ~7, side = in < full * rounds ? 8 : items - full;
  const int from = in < full * rounds ? in / (8 * rounds) * 8 : full, rest = in - from * rounds, item = from + rest % side;
  out.share = share;
  out.part = rest / side;
  out.tile = item / pool.n_kv; out.h = item - out.tile * pool.n_kv;
  return true;
}

SL_DEV float swap16_max(float v) {
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
SL_DEV float swap32_max(float v) {
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
SL_DEV float rows4_max(float v) { return swap32_max(swap16_max(v)); }     // over the four rows of 16 lanes
SL_DEV float nth_half(const uint32_t* w, int i) { return i & 1 ? hi_h(w[i / 2]) : lo_h(w[i / 2]); }
SL_DEV uint32_t half_pair(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }
SL_DEV uint32_t pair_of(float a, float b) { return __builtin_bit_cast(uint32_t, h2_t{(_Float16)a, (_Float16)b}); }   // (a product and its rounding may become one instruction)
// Sends what the wave has written to LDS ahead of what it reads there next (its LDS operations stay in order by themselves).
SL_DEV void wave_lds_order() { asm volatile("" ::: "memory"); __builtin_amdgcn_wave_barrier(); }

// Raw bytes of a step as the lanes load them.
template <int D>
struct KvStep {
  uint32_t k[2][D / 32];      // two key operands' quarter rows: words [group][2]
  uint32_t v[D / 16];         // 8 keys x D/32 bytes
  uint32_t sb[D / 64];        // lanes 0..31: key s|b of key `lane`, lanes 32..63: value s|b of key lane - 32
  bool there;                 // this lane's s|b key exists
};
template <int N>
SL_DEV void load_words(uint32_t* to, const unsigned char* p) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) { const uint4 x = ld16(p + 4 * i); to[i] = x.x; to[i + 1] = x.y; to[i + 2] = x.z; to[i + 3] = x.w; }
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p); to[0] = x.x; to[1] = x.y;
  } else to[0] = *reinterpret_cast<const uint32_t*>(p);
}
// Page ids for a step's three uses by this lane.
struct KvPages { int k, v, sb; };

// ---- one step of 32 keys: the parts that the kernels share ----
constexpr uint32_t mask_lo = 0x000F000Fu, mask_hi = 0x00F000F0u;       // nibbles 0 | 4 and 1 | 5 of a word: as halves, code * 2^-24 and code * 2^-20
constexpr int V_STRIDE = 64 * 16 + 16;        // bytes of a group's value pieces: [quarter of the keys][16 lanes][8 keys x 4 dims], padded against bank conflicts
// LDS of a step as the lanes read it.
struct StepLds {
  uint16_t *ks, *vs, *kb, *vb;                // key s, value s, key b [32][G], value b + 8 s [G][32]; vs follows ks
  unsigned char* v;                           // value pieces [G][V_STRIDE]
  template <int D>
  static SL_DEV StepLds at(unsigned char* p) {
    constexpr int G = D / 64;
    uint16_t* h = reinterpret_cast<uint16_t*>(p + G * V_STRIDE);
    return StepLds{h, h + AT_STEP * G, h + 2 * AT_STEP * G, h + 3 * AT_STEP * G, p};
  }
  template <int D>
  static constexpr int bytes() { return (D / 64) * (V_STRIDE + 4 * AT_STEP * 2); }
};
// The keys of a step whose values in a group are not finite.  They stay away from the matrix instructions, where a NaN would reach all
// dims of a row (it meets the zeros of the operands beside its own) and rows that do not see the key.
template <int D>
struct BadValues {
  unsigned any = 0;
  uint32_t keys[D / 64];                      // by group, where there are any
};
// Weights meet the values as fp16 operands, p s and p, which have 11 bits from 2^-14 to 2^16 and lose them below.  So both are taken in units:
// p is formed 2^6 times too large (a row's output is a quotient, from which that falls out), and the value scales of a group are taken times a power of
// two, 2^15 at most, that brings the largest near 2^6.  It only falls while a wave goes along its keys, and its sums with it; below 1 it
// stands where scales beyond 128 (values beyond some 1000) are met, and only then can a scale 2^21 below the largest lose bits.
// p keeps its 11 bits down to 2^-20 and p s down to 2^-25 of the largest s; they are there down to 2^-31 and 2^-36.  One key 13 above 4095
// others, values of 0.02: rows in bf16 are off by 1.6e-3 of their size, which is that type's own rounding (without units 6e-3 with
// 64 dims, 2.3e-2 in tiles of 64 rows); values of 1e-5: 1.5e-3 (4.7e-2).  Some ten instructions a step and the first step's maximum: with
// what else keeps numbers that are not finite and large scores right, one token at 4K 0.6 us of 18, 32 lanes of 256 dims 1.2 of 43, a prompt 3.5 of 143.
constexpr float P_UNIT_LOG2 = 6.0f;
constexpr uint32_t UNIT_TOP = 0x58005800u;          // 128 as halves: p reaches 2^8.875, p s then 2^15.875
template <int D>
struct ValueUnit {
  uint32_t f[(D / 64 + 1) / 2];                // by group, as halves; the same in all lanes
  SL_DEV bool operator!=(const ValueUnit& o) const {
    bool other = false;
#pragma unroll
    for (int w = 0; w < (D / 64 + 1) / 2; ++w) other = other || f[w] != o.f[w];
    return other;
  }
  SL_DEV int log2_of(int g) const { return (int)((f[g / 2] >> (16 * (g & 1) + 10)) & 31u) - 15; }
};
template <int D>
SL_DEV ValueUnit<D> first_unit() {
  ValueUnit<D> u;
#pragma unroll
  for (int w = 0; w < (D / 64 + 1) / 2; ++w) u.f[w] = 0x78007800u;            // 2^15
  return u;
}
SL_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
SL_DEV uint32_t max_halves(uint32_t a, uint32_t b) {                           // of two pairs of 16-bit numbers
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// The unit for value scales (lanes 32..63, two groups a word) of which one is too large for the present one.
template <int D>
SL_DEV void lower_unit(const uint32_t (&sc)[(D / 64 + 1) / 2], ValueUnit<D>& unit) {
#pragma unroll
  for (int w = 0; w < (D / 64 + 1) / 2; ++w) {
    uint32_t x = sc[w] & 0x7fff7fffu;
    x = max_halves(x, dpp_u<DPP_XOR1>(x)); x = max_halves(x, dpp_u<DPP_XOR2>(x));
    x = max_halves(x, dpp_u<DPP_HALF_MIRROR>(x)); x = max_halves(x, dpp_u<DPP_MIRROR>(x));
    x = max_halves((uint32_t)__builtin_amdgcn_readlane((int)x, 32), (uint32_t)__builtin_amdgcn_readlane((int)x, 48));
    uint32_t f = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int top = (int)((x >> (16 * u)) & 0x7fffu), old = (int)((unit.f[w] >> (16 * u)) & 0xffffu);
      const int e = top >= 0x400 ? (top >> 10) - 15 : 31 - __builtin_clz(top | 1) - 24;          // 2^e <= the largest < 2^(e+1)
      f |= (uint32_t)min(old, top ? (min(15, 5 - e) + 15) << 10 : old) << (16 * u);
    }
    unit.f[w] = __builtin_amdgcn_readfirstlane(f);
  }
}
// Scales and biases (lanes 0..31: key `lane`, lanes 32..63: value of key lane - 32) into LDS; a key that is not there gets
// zeros.  Value lanes turn b into b + 8 s; a group in which that is not finite gets zeros and is named in what comes back.
template <int D>
SL_DEV BadValues<D> put_scales(const uint32_t (&sb)[D / 64], bool there, const StepLds& st, ValueUnit<D>& unit) {
  constexpr int G = D / 64, W = (G + 1) / 2;
  const int lane = threadIdx.x & 63;
  uint32_t sc[W], bi[W];
#pragma unroll
  for (int g = 0; g < W; ++g) {
    const uint32_t w0 = there ? sb[G == 1 ? 0 : 2 * g] : 0u, w1 = G == 1 ? 0u : (there ? sb[G == 1 ? 0 : 2 * g + 1] : 0u);
    sc[g] = __builtin_amdgcn_perm(w1, w0, 0x05040100u); bi[g] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
  }
  h2_t odd = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
  for (int g = 0; g < W; ++g) {
    const h2_t eight = {(_Float16)8.0f, (_Float16)8.0f}, zero = {(_Float16)0.0f, (_Float16)0.0f};
    const h2_t b = __builtin_elementwise_fma(as_h2(sc[g]), eight, as_h2(bi[g]));
    odd = __builtin_elementwise_fma(b, zero, odd);
    bi[g] = lane < 32 ? bi[g] : __builtin_bit_cast(uint32_t, b);
  }
  const _Float16 none = odd.x + odd.y;
  BadValues<D> out;
  out.any = __any(none != none && lane >= 32);
  if (out.any) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t half = 0xffffu << (16 * (g & 1)), top = 0x7c00u << (16 * (g & 1));
      const bool bad = lane >= 32 && (bi[g / 2] & top) == top;
      out.keys[g] = (uint32_t)(__ballot(bad) >> 32);
      if (bad) { bi[g / 2] &= ~half; sc[g / 2] &= ~half; }
    }
  }
  auto in_unit = [&](int w) { return __builtin_bit_cast(uint32_t, as_h2(sc[w]) * as_h2(unit.f[w])); };
  uint32_t over = 0, x[W];
#pragma unroll
  for (int w = 0; w < W; ++w) { x[w] = in_unit(w); over |= (x[w] & 0x7fff7fffu) + (0x7fff7fffu - UNIT_TOP); }
  if (__any((over & 0x80008000u) != 0 && lane >= 32)) {
    lower_unit<D>(sc, unit);
#pragma unroll
    for (int w = 0; w < W; ++w) x[w] = in_unit(w);
  }
#pragma unroll
  for (int w = 0; w < W; ++w) sc[w] = lane < 32 ? sc[w] : x[w];
  if constexpr (G == 4) {
    *reinterpret_cast<uint2*>(st.ks + lane * G) = make_uint2(sc[0], sc[1]);
    if (lane < 32) *reinterpret_cast<uint2*>(st.kb + lane * G) = make_uint2(bi[0], bi[1]);
  } else if constexpr (G == 2) {
    *reinterpret_cast<uint32_t*>(st.ks + lane * G) = sc[0];
    if (lane < 32) *reinterpret_cast<uint32_t*>(st.kb + lane * G) = bi[0];
  } else {
    st.ks[lane] = (uint16_t)sc[0];
    if (lane < 32) st.kb[lane] = (uint16_t)bi[0];
  }
  if (lane >= 32) {
#pragma unroll
    for (int g = 0; g < G; ++g) st.vb[g * AT_STEP + (lane & 31)] = (uint16_t)(bi[g / 2] >> (16 * (g & 1)));
  }
  return out;
}
// s[row tile][8]: this lane's keys 8 kg .. 8 kg + 7 against row n16.  All products of the step first, so that no scale waits for
// the product before it.  `query(nt, i)`: the operand of dims word i; k: the two key operands' words.
template <int D, int LIVE, class Q, int NT>
SL_DEV void step_scores(const uint32_t (&k)[2][D / 32], Q query, const h8 (&qs)[NT], const StepLds& st, float (&s)[LIVE][8]) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  f4 acc[LIVE][2][G], accb[LIVE][2];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      h8 qf[LIVE];
#pragma unroll
      for (int nt = 0; nt < LIVE; ++nt) qf[nt] = query(nt, 2 * g + c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = k[i][2 * g + c], w8 = w >> 8;
        const h8 kf = __builtin_bit_cast(h8, make_uint4(w & mask_lo, w & mask_hi, w8 & mask_lo, w8 & mask_hi));
#pragma unroll
        for (int nt = 0; nt < LIVE; ++nt) acc[nt][i][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[nt], c ? acc[nt][i][g] : f4{0, 0, 0, 0}, 0, 0, 0);
      }
    }
  // sum over groups of b_g * (sum q), the sum in two halves
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = 8 * (n16 >> 2) + 4 * i + (n16 & 3);
    uint4 b;
    if constexpr (G == 4) { const uint2 x = *reinterpret_cast<const uint2*>(st.kb + key * G); b = make_uint4(x.x, x.y, x.x, x.y); }
    else if constexpr (G == 2) { const uint32_t x = *reinterpret_cast<const uint32_t*>(st.kb + key * G); b = make_uint4(x, x, 0, 0); }
    else { const uint32_t x = st.kb[key]; b = make_uint4(x | (x << 16), 0, 0, 0); }
#pragma unroll
    for (int nt = 0; nt < LIVE; ++nt) accb[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, b), qs[nt], f4{0, 0, 0, 0}, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t ks[2 * G];
    load_words<2 * G>(ks, (const unsigned char*)(st.ks + (8 * kg + 4 * i) * G));
#pragma unroll
    for (int nt = 0; nt < LIVE; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = accb[nt][i][j] * 2.384185791015625e-7f;
#pragma unroll
        for (int g = 0; g < G; ++g) x = fmaf(nth_half(ks, j * G + g), acc[nt][i][g][j], x);
        s[nt][4 * i + j] = x;
      }
  }
}
// The running maximum per row, p relative to it; pw: the operands p s_g of each group, then p itself.
template <int D, int LIVE, int NT>
SL_DEV void step_weights(float (&s)[LIVE][8], unsigned there, int k0, const int (&limit)[NT], const float (&mul)[NT], const StepLds& st, float (&m)[NT],
                         f4 (&o)[NT][D / 64][4], f4 (&ob)[NT], uint32_t (&pw)[LIVE][D / 64 + 1][4]) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 63, kg = lane >> 4;
  uint32_t vs[4 * G];
  load_words<4 * G>(vs, (const unsigned char*)(st.vs + 8 * kg * G));
#pragma unroll
  for (int nt = 0; nt < LIVE; ++nt) {
    // only the step at the end of a row's keys, and one with a page that is not there, has keys to hide
    const bool hides = there != 0xffffffffu || __any(limit[nt] < k0 + AT_STEP);
    if (hides) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (!((there >> (8 * kg + t)) & 1u) || k0 + 8 * kg + t >= limit[nt]) s[nt][t] = -__builtin_inff();
    }
    float top = s[nt][0];
#pragma unroll
    for (int t = 1; t < 8; ++t) top = fmaxf(top, s[nt][t]);
    top = rows4_max(top);
    // The reference moves only where a row's maximum has grown past it by a factor of 2^2.875 = 7.3: until then p lies above 1.
    if (__any((top - m[nt]) * mul[nt] > 2.875f)) {
      const float next = fmaxf(m[nt], top), back = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m[nt] - next) * mul[nt]);
      ob[nt] = ob[nt] * back;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][g][i] = o[nt][g][i] * back;
      m[nt] = next;
    }
    float from = m[nt] == -__builtin_inff() ? 0.0f : fmaf(-m[nt], mul[nt], P_UNIT_LOG2);
    // The fused difference is off by the rounding of m * mul: 2^-12 here at most.  Beyond that the scores are subtracted first, which is
    // exact where it counts, next to the reference.
    if (__any(fabsf(from) > 4096.0f)) {
      const float ref = m[nt] == -__builtin_inff() ? 0.0f : m[nt];
#pragma unroll
      for (int t = 0; t < 8; ++t) s[nt][t] = s[nt][t] - ref;
      from = P_UNIT_LOG2;
    }
    float p[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) p[t] = __builtin_amdgcn_exp2f(fmaf(s[nt][t], mul[nt], from));
#pragma unroll
    for (int t = 0; t < 4; ++t) pw[nt][G][t] = pair_of(p[2 * t], p[2 * t + 1]);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int t = 0; t < 4; ++t) pw[nt][g][t] = pair_of(fmaf(p[2 * t], nth_half(vs, 2 * t * G + g), 0.0f), fmaf(p[2 * t + 1], nth_half(vs, (2 * t + 1) * G + g), 0.0f));   // (fma: takes the half as it is)
  }
}
// The sums of (p s) c and of p s brought to another unit.
template <int D, int NT>
SL_DEV void change_unit(const ValueUnit<D>& was, const ValueUnit<D>& unit, f4 (&o)[NT][D / 64][4], f4 (&ob)[NT]) {
  const int kg = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    const float by = pow2(unit.log2_of(g) - was.log2_of(g));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ob[nt][g] = kg == 2 ? ob[nt][g] * by : ob[nt][g];                // (lanes of the third 16 hold rows 8..11 of ob)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][g][i] = o[nt][g][i] * by;
    }
  }
}
// Rows that see a key whose values in a group are not finite: their sum over b + 8 s of that group becomes NaN, and all its dims with it.
template <int D, int LIVE, int NT>
SL_DEV void mark_bad(const BadValues<D>& bad, int k0, const int (&limit)[NT], f4 (&ob)[NT]) {
  const int kg = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int nt = 0; nt < LIVE; ++nt) {
    const int seen = min(max(limit[nt] - k0, 0), AT_STEP);
    const uint32_t sees = seen == AT_STEP ? ~0u : (1u << seen) - 1u;
#pragma unroll
    for (int g = 0; g < D / 64; ++g)
      if (kg == 0 && (bad.keys[g] & sees)) ob[nt][g] = __builtin_nanf("");       // (lanes of the first 16 hold rows 0..3 of ob)
  }
}
// Values: o[group][i] gathers (p s_g) c of the dims 4 m' + i, in units of 2^-24 (odd i: 2^-20, the nibble standing four bits up).
// Codes run from 0, so the rounding of p s_g is as large as c makes it; ob takes what brings it back to c - 8: row g of ob
// is sum p (b_g + 8 s_g), row 8 + g the sum of the rounded p s_g (times 8 to be taken off), row G the sum of p, the softmax's own.
template <int D>
struct OnesRows { h8 at[D / 64]; };              // per group: an operand whose row 8 + g is ones
template <int D>
SL_DEV OnesRows<D> ones_rows() {
  constexpr int G = D / 64;
  const int n16 = threadIdx.x & 15;
  OnesRows<D> r;
#pragma unroll
  for (int g = 0; g < G; ++g) { const uint32_t x = n16 == 8 + g ? 0x3c003c00u : 0u; r.at[g] = __builtin_bit_cast(h8, make_uint4(x, x, x, x)); }
  return r;
}
template <int D, int LIVE, int NT>
SL_DEV void step_values(const uint32_t (&pw)[LIVE][D / 64 + 1][4], const StepLds& st, const OnesRows<D>& ones, f4 (&o)[NT][D / 64][4], f4 (&ob)[NT]) {
  constexpr int G = D / 64;
  const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  const uint32_t one = n16 == G ? 0x3c003c00u : 0u;
  uint4 vb = make_uint4(one, one, one, one);
  if (n16 < G) vb = *reinterpret_cast<const uint4*>(st.vb + n16 * AT_STEP + 8 * kg);
#pragma unroll
  for (int nt = 0; nt < LIVE; ++nt)
    ob[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, vb), __builtin_bit_cast(h8, make_uint4(pw[nt][G][0], pw[nt][G][1], pw[nt][G][2], pw[nt][G][3])), ob[nt], 0, 0, 0);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint4 raw = ld16(st.v + g * V_STRIDE + lane * 16);
    const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
    h8 weight[LIVE];
#pragma unroll
    for (int nt = 0; nt < LIVE; ++nt) weight[nt] = __builtin_bit_cast(h8, make_uint4(pw[nt][g][0], pw[nt][g][1], pw[nt][g][2], pw[nt][g][3]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) w[t] = (i & 2 ? x[t] >> 8 : x[t]) & (i & 1 ? mask_hi : mask_lo);
      const h8 vf = __builtin_bit_cast(h8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int nt = 0; nt < LIVE; ++nt) o[nt][g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, weight[nt], o[nt][g][i], 0, 0, 0);
    }
#pragma unroll
    for (int nt = 0; nt < LIVE; ++nt) ob[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones.at[g], weight[nt], ob[nt], 0, 0, 0);
  }
}
// The softmax's sum of row n16.
template <int D>
SL_DEV float sum_of(const f4& ob) { return __shfl(ob[D / 64 % 4], (int)(threadIdx.x & 15) + 16 * (D / 256)); }

template <int D, int NT>
struct AttnLds {
  static constexpr int G = D / 64;                                    // groups of a row
  static constexpr int WAVE = StepLds::bytes<D>();
  static constexpr int Q = NT * (D / 32) * 64 * 16;                   // query operands in the order of the lanes
  static constexpr int JOIN = AT_WAVES * 16 * (D + 4) * 4;            // one row tile of every wave
  static constexpr int MAIN = AT_WAVES * WAVE + Q > JOIN ? AT_WAVES * WAVE + Q : JOIN;
  static constexpr int STAT = (2 * AT_WAVES + 2 + 4) * 16 * NT * 4;   // maximum and sum per wave and row; per row factor, keys seen, sums of q
  static constexpr int BYTES = MAIN + STAT;
};

constexpr int NO_LIMIT = 0x7fffffff;          // of the columns behind the last row, which are never written
struct QueryLds {
  uint4 *word, *sum;                          // operands [row tile][D/32][64 lanes], the groups' sums of a row as halves
  float* mul;                                 // factor from a row's scores to units of log2
  int* limit;                                 // keys that a row sees
};
// Row `in` of the workgroup, 16 lanes a row, D/16 dims a lane (bits in `raw`).
template <int D, bool BF>
SL_DEV void put_query(const uint2 (&raw)[D / 64], int in, bool valid, int limit, float scale, const QueryLds& q) {
  constexpr int G = D / 64, PER = D / 16;
  const int l16 = threadIdx.x & 15;
  float x[PER], top = 0.0f;
#pragma unroll
  for (int c = 0; c < PER / 4; ++c) {
    const uint16_t e4[4] = {(uint16_t)raw[c].x, (uint16_t)(raw[c].x >> 16), (uint16_t)raw[c].y, (uint16_t)(raw[c].y >> 16)};
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[4 * c + j] = valid ? elem_f<BF>(e4[j]) : 0.0f; top = fmaxf(top, fabsf(x[4 * c + j])); }
  }
  top = fmaxf(top, dpp_f<DPP_XOR1>(top)); top = fmaxf(top, dpp_f<DPP_XOR2>(top));
  top = fmaxf(top, dpp_f<DPP_HALF_MIRROR>(top)); top = fmaxf(top, dpp_f<DPP_MIRROR>(top));
  const int e = min(max((int)((__float_as_uint(top) >> 23) & 255u) - 127, -100), 127);
  const float f = __uint_as_float((uint32_t)(127 + 10 - e) << 23) * (scale < 0.0f ? -1.0f : 1.0f);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) { x[i] = x[i] * f; sum = sum + x[i]; }
  sum = tree_sum<16 / G>(sum) * 0.25f;               // at most 64 * 2^11 / 4
  if (l16 % (16 / G) == 0) {                         // as two halves, behind each other for G > 1: operand [hi of the groups | lo of the groups]
    uint16_t* w = reinterpret_cast<uint16_t*>(q.sum + in) + l16 / (16 / G);
    const uint16_t hi = f2h(sum);
    w[0] = hi; w[G] = f2h(sum - h2f(hi));
    if (G < 4) {
#pragma unroll
      for (int i = 2; i < 8 / G; ++i) w[i * G] = 0;
    }
  }
  if (l16 == 0) {
    // (a factor of zero would leave hidden keys without their minus infinity, one of infinity the largest score without its zero)
    q.mul[in] = fminf(fmaxf(fabsf(scale) * (1.44269504088896f * 16777216.0f) * pow2(e - 10), 1e-30f), 3e38f);
    q.limit[in] = limit;
  }
  // operand word w of quarter kg in group g: dims 64 g + 16 kg + 8 w + (0 4 | 1 5 | 2 6 | 3 7), the odd ones / 16
  if constexpr (PER >= 8) {
#pragma unroll
    for (int c = 0; c < PER / 8; ++c) {
      const int d = PER * l16 + 8 * c, to = (in / 16 * (D / 32) + 2 * (d / 64) + (d / 8) % 2) * 64 + (d % 64) / 16 * 16 + (in & 15);
      const float* y = x + 8 * c;
      q.word[to] = make_uint4(half_pair(y[0], y[4]), half_pair(y[1] * 0.0625f, y[5] * 0.0625f), half_pair(y[2], y[6]), half_pair(y[3] * 0.0625f, y[7] * 0.0625f));
    }
  } else {
    const int d = 4 * l16, to = (in / 16 * (D / 32) + (d / 8) % 2) * 64 + d / 16 * 16 + (in & 15);
    uint16_t* w = reinterpret_cast<uint16_t*>(q.word + to) + (l16 & 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[2 * j] = f2h(j & 1 ? x[j] * 0.0625f : x[j]);
  }
}

// Normalised, gated, rounded: the last step of a row (sum 0: the row saw no key).
template <bool BF>
SL_DEV float finish_value(const sl_kv4_attn_args& a, float y, float sum, uint16_t gate) {
  y = sum != 0.0f ? y / sum : 0.0f;
  return a.gate ? y * (1.0f / (1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * elem_f<BF>(gate)))) : y;
}
template <bool BF>
SL_DEV void finish_row(const sl_kv4_attn_args& a, int t, int head, int d, float4 y, float sum) {
  uint2 g = make_uint2(0, 0);
  if (a.gate) g = *reinterpret_cast<const uint2*>((const uint16_t*)a.gate + t * a.gate_token + head * a.gate_head + d);
  const float x0 = finish_value<BF>(a, y.x, sum, (uint16_t)g.x), x1 = finish_value<BF>(a, y.y, sum, (uint16_t)(g.x >> 16));
  const float x2 = finish_value<BF>(a, y.z, sum, (uint16_t)g.y), x3 = finish_value<BF>(a, y.w, sum, (uint16_t)(g.y >> 16));
  *reinterpret_cast<uint2*>((uint16_t*)a.out + t * a.out_token + head * a.out_head + d) =
      make_uint2((uint32_t)f_elem<BF>(x0) | ((uint32_t)f_elem<BF>(x1) << 16), (uint32_t)f_elem<BF>(x2) | ((uint32_t)f_elem<BF>(x3) << 16));
}
// A wave's sums of one row tile to LDS [16 rows][D + 4], times f: lane (n16, kg) holds dims 64 g + 16 kg + 4 r + i of row n16.
template <int D>
SL_DEV void put_sums(const f4 (&o)[D / 64][4], const f4& ob, const ValueUnit<D>& unit, float f, float* to) {
  const int lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  float bias[D / 64], even[D / 64], odd[D / 64];
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    const float back = pow2(-unit.log2_of(g));
    even[g] = 16777216.0f * back; odd[g] = 1048576.0f * back;
    bias[g] = fmaf(-8.0f * back, __shfl(ob[g], n16 + 32), __shfl(ob[g], n16));
  }
#pragma unroll
  for (int g = 0; g < D / 64; ++g)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float4 y;
      y.x = fmaf(o[g][0][r], even[g], bias[g]) * f; y.y = fmaf(o[g][1][r], odd[g], bias[g]) * f;
      y.z = fmaf(o[g][2][r], even[g], bias[g]) * f; y.w = fmaf(o[g][3][r], odd[g], bias[g]) * f;
      *reinterpret_cast<float4*>(to + n16 * (D + 4) + 64 * g + 16 * kg + 4 * r) = y;
    }
}
// Four dims of a row: to the output, or as a partial sum (slot >= 0) with its maximum and sum.
template <int D, bool BF>
SL_DEV void put_row(const sl_kv4_attn_args& a, const AttnCut& cut, long slot, int in, int t, int head, int d, float4 y, float best, float sum) {
  if (slot < 0) { finish_row<BF>(a, t, head, d, y, sum); return; }
  *reinterpret_cast<float4*>(cut.part + (slot * cut.rows + in) * D + d) = y;
  if (d == 0) {
    float* stat = cut.part + cut.slots * cut.rows * D;
    stat[slot * cut.rows + in] = best; stat[(cut.slots + slot) * cut.rows + in] = sum;
  }
}

// Up to 16 (NT = 1) or 32 rows a workgroup.  What bounds it: one token at 4K 10.9 us, start and end (lengths, table, page, queries, the
// join in LDS) with one round of keys between; 32 lanes at 1K-16K 34 us, the same 10 us and 107 MB at 4.5 TB/s; six requests
// of 3-5 rows at 20-32K, 128 dims, 51 us, 187 MB, vector instructions in 68 % of the slots; 2333 rows behind 4-16K, 64 dims,
// 185 us, 90 % of the slots (unpacking 1/2, softmax and weights 1/2; the matrix cores are busy 22 %).
// Workgroups on a compute unit: by the registers, of which the running sums alone take NT * D / 4.
constexpr int attn_places(int dim, int nt) { return dim == 64 ? (nt == 1 ? 4 : 3) : (dim == 128 && nt == 1 ? 3 : 2); }
template <int D, bool BF, int NT>
__global__ __launch_bounds__(256, attn_places(D, NT)) void k_kv4_attn(Pool pool, sl_kv4_attn_args a, AttnCut cut) {
  using L = AttnLds<D, NT>;
  constexpr int G = L::G;
  extern __shared__ __align__(16) unsigned char lds[];
  float* s_m = reinterpret_cast<float*>(lds + L::MAIN);
  float *s_l = s_m + AT_WAVES * 16 * NT, *s_mul = s_l + AT_WAVES * 16 * NT;
  int* s_lim = reinterpret_cast<int*>(s_mul + 16 * NT);
  uint4* s_qsum = reinterpret_cast<uint4*>(s_lim + 16 * NT);
  int* s_first = reinterpret_cast<int*>(lds + L::BYTES);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, kg = lane >> 4;
  const StepLds st = StepLds::at<D>(lds + wave * L::WAVE);
  uint4* s_q = reinterpret_cast<uint4*>(lds + AT_WAVES * L::WAVE);
  const QueryLds sq{s_q, s_qsum, s_mul, s_lim};
  const int group = a.n_heads / pool.n_kv, shift = pool.page_shift, page_mask = (1 << shift) - 1;
  const uint32_t page_stride = (uint32_t)(pool.n_kv * (int)head_bytes<D>(pool));
  const int part_c = (D / 2) << shift, part_sb = (D / 16) << shift;

  AttnPart at;
  if (!find_part<16 * NT>(a, pool, cut, blockIdx.x, s_first, reinterpret_cast<int*>(s_m), at)) return;
  {
    const int r = at.r, h = at.h;
    int start, n;
    const int rows = rows_of(a, r, start, n), tile = NT > 1 ? (rows * group + 16 * NT - 1) / (16 * NT) - 1 - at.tile : at.tile, row0 = tile * 16 * NT, rows_here = min(16 * NT, rows * group - row0);      // (the tiles that see most keys first)
    const long keys = seen_keys(a, pool, r);
    long last;
    int parts, per;
    tile_cut<16 * NT>(keys, n, rows * group, tile, group, at.share, last, parts, per);
    if (at.part >= parts) return;
    const long slot = parts > 1 ? (long)blockIdx.x : -1;
    const int key0 = at.part * per * AT_UNIT, key1 = (int)min((long)(at.part + 1) * per * AT_UNIT, last);
    const int32_t* table = a.table + (size_t)r * a.table_width;
    const int end_page = key1 > 0 ? (key1 - 1) >> shift : 0;
    auto pages = [&](int k0) {
      KvPages p;
      if (shift >= 5) p.k = p.v = p.sb = table[min(k0 >> shift, end_page)];
      else {
        p.k = table[min((k0 + 8 * (n16 >> 2)) >> shift, end_page)];
        p.v = table[min((k0 + 8 * kg) >> shift, end_page)];
        p.sb = table[min((k0 + (lane & 31)) >> shift, end_page)];
      }
      return p;
    };
    const unsigned char* head_base = pool.pages + (size_t)h * head_bytes<D>(pool);
    auto base = [&](int page) { return head_base + (uint64_t)((unsigned)page < (unsigned)pool.n_pages ? (uint32_t)page : 0u) * page_stride; };
    auto load_keys = [&](int k0, const KvPages& p, KvStep<D>& s) {
      const int ok = (k0 + 8 * (n16 >> 2) + (n16 & 3)) & page_mask;
      const unsigned char* bk = base(p.k) + ok * (D / 2) + kg * (D / 8);
      load_words<D / 32>(s.k[0], bk);
      load_words<D / 32>(s.k[1], bk + 4 * (D / 2));
    };
    auto load_rest = [&](int k0, const KvPages& p, KvStep<D>& s) {
      const int ov = (k0 + 8 * kg) & page_mask, os = (k0 + (lane & 31)) & page_mask;
      load_words<G>(s.sb, base(p.sb) + (lane < 32 ? part_c : 2 * part_c + part_sb) + os * (D / 16));
      load_words<D / 16>(s.v, base(p.v) + part_c + part_sb + ((ov >> 3) * 16 + n16) * (D / 4));
      s.there = (unsigned)p.sb < (unsigned)pool.n_pages && k0 + (lane & 31) < key1;
    };
    // A step's registers are loaded again as soon as they have been used: the next values while this step's keys are
    // multiplied, the next keys while its softmax and its values are.
    int k0 = key0 + wave * AT_STEP;
    KvStep<D> cur;
    KvPages ahead{};
    // Queries are asked for first, then the first step's bytes, which are on their way while the queries are laid out.
    constexpr int QPER = D / 16;                         // 16 lanes a row
    uint2 raw[NT][QPER / 4];
#pragma unroll
    for (int pass = 0; pass < NT; ++pass) {
      const int in = pass * 16 + (tid >> 4), row = row0 + (in < rows_here ? in : 0), tok = row / group, head = h * group + (row - tok * group);
      const uint16_t* src = (const uint16_t*)a.q + (long)(start + tok) * a.q_token + (long)head * a.q_head + QPER * (tid & 15);
#pragma unroll
      for (int c = 0; c < QPER / 4; ++c) raw[pass][c] = *reinterpret_cast<const uint2*>(src + 4 * c);
    }
    if (k0 < key1) { const KvPages p = pages(k0); ahead = pages(k0 + AT_UNIT); load_rest(k0, p, cur); load_keys(k0, p, cur); }

    // ---- queries: operands in fp16, their sums per group, the factor back to scores in units of log2 ----
#pragma unroll
    for (int pass = 0; pass < NT; ++pass) {
      if (pass * 16 >= rows_here) break;                 // (operands of an empty tile are not used)
      const int in = pass * 16 + (tid >> 4);
      put_query<D, BF>(raw[pass], in, in < rows_here, in < rows_here ? (int)max(0l, keys - n + (row0 + in) / group + 1) : NO_LIMIT, a.scale, sq);
    }
    lds_barrier();
    // (dims of 256 and several row tiles leave no room for the operands in registers)
    constexpr bool Q_REGS = NT == 1 && D < 256;
    h8 q[Q_REGS ? D / 32 : 1], qs[NT];
    float mul[NT];
    int limit[NT];                                       // keys that row n16 of tile nt sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (Q_REGS) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q[i] = __builtin_bit_cast(h8, s_q[i * 64 + lane]);
      }
      mul[nt] = s_mul[nt * 16 + n16]; limit[nt] = s_lim[nt * 16 + n16];
      qs[nt] = __builtin_bit_cast(h8, kg == 0 ? s_qsum[nt * 16 + n16] : make_uint4(0, 0, 0, 0));
    }

    const OnesRows<D> ones = ones_rows<D>();
    f4 o[NT][G][4], ob[NT];
    float m[NT];                                         // the reference of p, in scores before the factor
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -__builtin_inff(); ob[nt] = f4{0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][g][i] = f4{0, 0, 0, 0};
    }

    ValueUnit<D> unit = first_unit<D>();

    // ---- keys: a step of 32 for the first LIVE row tiles ----
    auto keys_loop = [&](auto live_tiles) {
      constexpr int LIVE = decltype(live_tiles)::value;
      for (; k0 < key1; k0 += AT_UNIT) {
        const bool more = k0 + AT_UNIT < key1;
        const unsigned there = (unsigned)__ballot(cur.there);
        wave_lds_order();
        const ValueUnit<D> was = unit;
        const BadValues<D> bad = put_scales<D>(cur.sb, cur.there, st, unit);
        if (unit != was && k0 != key0 + wave * AT_STEP) change_unit<D, NT>(was, unit, o, ob);      // (no sums yet in the first step)
        // values: the piece of 4 dims that belongs to lane m' of group g, 8 keys together
#pragma unroll
        for (int c = 0; c < G; ++c) {
          uint32_t x[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if constexpr (G == 4) x[t] = __builtin_amdgcn_perm(cur.v[4 * t + 2 + c / 2], cur.v[4 * t + c / 2], c & 1 ? 0x07060302u : 0x05040100u);
            else if constexpr (G == 2) x[t] = __builtin_amdgcn_perm(cur.v[2 * t + 1], cur.v[2 * t], c & 1 ? 0x07060302u : 0x05040100u);
            else x[t] = cur.v[t];
          }
          st16(st.v + (n16 / (16 / G)) * V_STRIDE + (kg * 16 + G * (n16 % (16 / G)) + c) * 16, make_uint4(x[0], x[1], x[2], x[3]));
        }
        wave_lds_order();
        if (more) load_rest(k0 + AT_UNIT, ahead, cur);
        float s[LIVE][8];
        step_scores<D, LIVE>(cur.k, [&](int nt, int i) {
          if constexpr (Q_REGS) return q[i];
          else return __builtin_bit_cast(h8, s_q[(nt * (D / 32) + i) * 64 + lane]);
        }, qs, st, s);
        if (more) { load_keys(k0 + AT_UNIT, ahead, cur); ahead = pages(k0 + 2 * AT_UNIT); }
        uint32_t pw[LIVE][G + 1][4];
        step_weights<D, LIVE, NT>(s, there, k0, limit, mul, st, m, o, ob, pw);
        step_values<D, LIVE, NT>(pw, st, ones, o, ob);
        if (bad.any) mark_bad<D, LIVE, NT>(bad, k0, limit, ob);
      }
    };
    if (NT == 1 || rows_here <= 16) keys_loop(std::integral_constant<int, 1>{});
    else keys_loop(std::integral_constant<int, NT>{});
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt] = m[nt] * mul[nt];        // in units of log2 from here on

    // ---- the four waves' sums together; lane (n16, kg) holds dims 64 g + 16 kg + 4 r + i of row n16 ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float sum = sum_of<D>(ob[nt]);
      if (kg == 0) { s_m[wave * 16 * NT + nt * 16 + n16] = m[nt]; s_l[wave * 16 * NT + nt * 16 + n16] = sum; }
    }
    float* s_o = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      lds_barrier();
      if (nt * 16 >= rows_here) continue;                // (the same for the whole workgroup)
      float top = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < AT_WAVES; ++w) top = fmaxf(top, s_m[w * 16 * NT + nt * 16 + n16]);
      const float f = m[nt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[nt] - top);
      put_sums<D>(o[nt], ob[nt], unit, f, s_o + wave * 16 * (D + 4));
      lds_barrier();
      // a thread per four dims of a row
      for (int i = tid; i < 16 * (D / 4); i += 256) {
        const int row = i / (D / 4), d = 4 * (i % (D / 4)), in = nt * 16 + row;
        if (in >= rows_here) break;
        float4 y = make_float4(0, 0, 0, 0);
        float best = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < AT_WAVES; ++w) best = fmaxf(best, s_m[w * 16 * NT + in]);
#pragma unroll
        for (int w = 0; w < AT_WAVES; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(s_o + (w * 16 + row) * (D + 4) + d);
          y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
          const float mw = s_m[w * 16 * NT + in];
          sum += s_l[w * 16 * NT + in] * (mw == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mw - best));
        }
        const int row_of = row0 + in, tok = row_of / group;
        put_row<D, BF>(a, cut, slot, in, start + tok, h * group + (row_of - tok * group), d, y, best, sum);
      }
    }
  }
}

// Many rows of 256 dims: a workgroup takes 64 rows, each wave 16 of them and all keys (the sums of 32 rows would not leave room for two
// waves a SIMD).  The waves lay a step's bytes out in LDS together, a step ahead of its use, so the registers hold no bytes but
// those on their way.  (With fewer dims a wave has room for 32 rows, and waves that unpack their own keys are faster than
// ones that meet at a barrier every step: 64 rows of 128 dims against 32K keys 121 us, with this kernel's scheme 190.)
// A prompt of 2048 rows and 16 heads 144 us, 239 TFLOP/s: 512 workgroups, two to a unit, and the last row tile's 64 steps of 2.2 us
// are its length; 512 rows behind 8K 180 us, 395 TFLOP/s.
template <int D>
struct TileLds {
  static constexpr int KEYS = 16 * D;                                  // key words in the order of the lanes
  static constexpr int STEP = KEYS + StepLds::bytes<D>();
  static constexpr int Q = 4 * (D / 32) * 64 * 16;
  static constexpr int JOIN = 4 * 16 * (D + 4) * 4;
  static constexpr int MAIN = 2 * STEP + Q > JOIN ? 2 * STEP + Q : JOIN;
  static constexpr int STAT = (2 + 2 + 4) * 64 * 4;
  static constexpr int BYTES = MAIN + STAT;
};
template <int D, bool BF>
__global__ __launch_bounds__(256, 2) void k_kv4_attn_tile(Pool pool, sl_kv4_attn_args a, AttnCut cut) {
  using L = TileLds<D>;
  static_assert(D == 256, "a thread brings 16 bytes of keys and of values, half a lane's quarter row");
  constexpr int G = D / 64, NT = 1, KW = 4, HALVES = 2;
  extern __shared__ __align__(16) unsigned char lds[];
  float* s_m = reinterpret_cast<float*>(lds + L::MAIN);
  float *s_l = s_m + 64, *s_mul = s_l + 64;
  int* s_lim = reinterpret_cast<int*>(s_mul + 64);
  uint4* s_qsum = reinterpret_cast<uint4*>(s_lim + 64);
  int* s_first = reinterpret_cast<int*>(lds + L::BYTES);
  uint4* s_q = reinterpret_cast<uint4*>(lds + 2 * L::STEP);
  const QueryLds sq{s_q, s_qsum, s_mul, s_lim};
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, kg = lane >> 4;
  const int group = a.n_heads / pool.n_kv, shift = pool.page_shift, page_mask = (1 << shift) - 1;
  const uint32_t page_stride = (uint32_t)(pool.n_kv * (int)head_bytes<D>(pool));
  const int part_c = (D / 2) << shift, part_sb = (D / 16) << shift;

  AttnPart at;
  if (!find_part<64>(a, pool, cut, blockIdx.x, s_first, reinterpret_cast<int*>(s_m), at)) return;
  const int r = at.r, h = at.h;
  int start, n;
  const int rows = rows_of(a, r, start, n), tiles = (rows * group + 63) / 64;
  const int tile = tiles - 1 - at.tile, row0 = tile * 64, rows_here = min(64, rows * group - row0);      // the tiles that see most keys first
  const long keys = seen_keys(a, pool, r);
  long last;
  int parts, per;
  tile_cut<64>(keys, n, rows * group, tile, group, at.share, last, parts, per);
  if (at.part >= parts) return;
  const long slot = parts > 1 ? (long)blockIdx.x : -1;
  const int key0 = at.part * per * AT_UNIT, key1 = (int)min((long)(at.part + 1) * per * AT_UNIT, last);

  uint2 raw[4][D / 64];
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int in = pass * 16 + (tid >> 4), row = row0 + (in < rows_here ? in : 0), tok = row / group, head = h * group + (row - tok * group);
    const uint16_t* src = (const uint16_t*)a.q + (long)(start + tok) * a.q_token + (long)head * a.q_head + (D / 16) * (tid & 15);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) raw[pass][c] = *reinterpret_cast<const uint2*>(src + 4 * c);
  }

  // A step's bytes: 16 each of keys and values by every thread, scales and biases by the first wave.
  const int32_t* table = a.table + (size_t)r * a.table_width;
  const int end_page = key1 > 0 ? (key1 - 1) >> shift : 0;
  const unsigned char* head_base = pool.pages + (size_t)h * head_bytes<D>(pool);
  auto base = [&](int page) { return head_base + (uint64_t)((unsigned)page < (unsigned)pool.n_pages ? (uint32_t)page : 0u) * page_stride; };
  auto page_of = [&](int key) { return table[min(key >> shift, end_page)]; };
  uint32_t wk[KW], wv[KW], sb[G];
  bool there = false;
  const int key_token = tid & 31, key_part = tid >> 5;
  constexpr int V_UNITS = D / 16 / KW;                                 // threads to a lane's 8 keys
  const int v_blk = tid / (16 * V_UNITS), v_m = (tid / V_UNITS) & 15, v_sub = tid % V_UNITS;
  auto pages = [&](int k0) {
    KvPages p;
    p.k = page_of(k0 + key_token); p.v = page_of(k0 + 8 * v_blk); p.sb = wave == 0 ? page_of(k0 + (lane & 31)) : 0;
    return p;
  };
  auto load = [&](int k0, const KvPages& p) {
    load_words<KW>(wk, base(p.k) + ((k0 + key_token) & page_mask) * (D / 2) + 4 * KW * key_part);
    load_words<KW>(wv, base(p.v) + part_c + part_sb + (((k0 + 8 * v_blk) & page_mask) >> 3) * (4 * D) + (tid % (16 * V_UNITS)) * (4 * KW));
    if (wave == 0) {
      load_words<G>(sb, base(p.sb) + (lane < 32 ? part_c : 2 * part_c + part_sb) + ((k0 + (lane & 31)) & page_mask) * (D / 16));
      there = (unsigned)p.sb < (unsigned)pool.n_pages && k0 + (lane & 31) < key1;
    }
  };
  auto step_lds = [&](int buf) { return lds + buf * L::STEP; };
  struct Note { unsigned there; ValueUnit<D> unit; BadValues<D> bad; };
  Note* s_note = reinterpret_cast<Note*>(s_m);                         // by buffer: the keys that are there, the values' unit; free until the end
  ValueUnit<D> unit_put = first_unit<D>(), unit = unit_put;            // of the first wave's last step in LDS, of this wave's sums
  // keys: [operand][half of the row's quarter][quarter][row of the operand]; values: pieces of 4 dims, two keys a word
  const int k_to = ((((key_token >> 2) & 1) * HALVES + key_part % HALVES) * 64 + key_part / HALVES * 16 + (key_token >> 3) * 4 + (key_token & 3)) * 4 * KW;
  const int v_to = v_m / (16 / G) * V_STRIDE + (v_blk * 16 + G * (v_m % (16 / G))) * 16 + v_sub * 4;
  auto put = [&](int buf) {
    unsigned char* to = step_lds(buf);
    const StepLds st = StepLds::at<D>(to + L::KEYS);
    st16(to + k_to, make_uint4(wk[0], wk[1], wk[2], wk[3]));
#pragma unroll
    for (int c = 0; c < 4; ++c)            // two keys of 8 bytes: a word of four pieces
      *reinterpret_cast<uint32_t*>(st.v + v_to + 16 * c) = __builtin_amdgcn_perm(wv[2 + c / 2], wv[c / 2], c & 1 ? 0x07060302u : 0x05040100u);
    if (wave == 0) {
      const BadValues<D> bad = put_scales<D>(sb, there, st, unit_put);
      const unsigned mask = (unsigned)__ballot(there);
      if (lane == 0) {
        s_note[buf].there = mask; s_note[buf].unit = unit_put; s_note[buf].bad.any = bad.any;
        if (bad.any) s_note[buf].bad = bad;
      }
    }
  };

  const int steps = key1 > key0 ? (key1 - key0 + AT_STEP - 1) / (AT_STEP) : 0;
  int k0 = key0;
  KvPages ahead{};
  if (steps > 0) { load(k0, pages(k0)); ahead = pages(k0 + AT_STEP); }
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int in = pass * 16 + (tid >> 4);
    put_query<D, BF>(raw[pass], in, in < rows_here, in < rows_here ? (int)max(0l, keys - n + (row0 + in) / group + 1) : NO_LIMIT, a.scale, sq);
  }
  lds_barrier();
  if (steps > 0) put(0);
  if (steps > 1) { load(k0 + AT_STEP, ahead); ahead = pages(k0 + 2 * AT_STEP); }
  h8 qs[NT];
  float mul[NT];
  int limit[NT], most = 0;                             // keys that row n16 of tile nt sees, and that any row of this wave sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int in = wave * 16 + n16;
    mul[nt] = s_mul[in]; limit[nt] = s_lim[in];
    qs[nt] = __builtin_bit_cast(h8, kg == 0 ? s_qsum[in] : make_uint4(0, 0, 0, 0));
  }
  if (wave * 16 < rows_here) most = (int)max(0l, min(keys, keys - n + (row0 + min((wave + 1) * 16, rows_here) - 1) / group + 1));
  const OnesRows<D> ones = ones_rows<D>();
  f4 o[NT][G][4], ob[NT];
  float m[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -__builtin_inff(); ob[nt] = f4{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][g][i] = f4{0, 0, 0, 0};
  }
  lds_barrier();
  auto turn = [&](int i) {                             // the next step's bytes into LDS, those of the one after it asked for
    if (i + 1 < steps) put((i & 1) ^ 1);
    if (i + 2 < steps) { load(k0 + 2 * AT_STEP, ahead); ahead = pages(k0 + 3 * AT_STEP); }
    lds_barrier();
  };
  const int mine = min(steps, max(0, (most - key0 + AT_STEP - 1) / AT_STEP));     // steps that any row of this wave sees
  int i = 0;
  for (; i < mine; ++i, k0 += AT_STEP) {
    const int buf = i & 1;
    const unsigned char* from = step_lds(buf);
    const StepLds st = StepLds::at<D>((unsigned char*)from + L::KEYS);
    uint32_t k[2][D / 32];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        uint32_t w[KW];
        load_words<KW>(w, from + ((c * HALVES + half) * 64 + lane) * 4 * KW);
#pragma unroll
        for (int j = 0; j < KW; ++j) k[c][half * KW + j] = w[j];
      }
    const unsigned here = s_note[buf].there, any_bad = __builtin_amdgcn_readfirstlane(s_note[buf].bad.any);
    ValueUnit<D> now = s_note[buf].unit;
#pragma unroll
    for (uint32_t& f : now.f) f = __builtin_amdgcn_readfirstlane(f);
    if (now != unit) { if (i > 0) change_unit<D, NT>(unit, now, o, ob); unit = now; }              // (no sums yet in the first step)
    float s[NT][8];
    step_scores<D, NT>(k, [&](int nt, int w) { return __builtin_bit_cast(h8, s_q[(wave * (D / 32) + w) * 64 + lane]); }, qs, st, s);
    uint32_t pw[NT][G + 1][4];
    step_weights<D, NT, NT>(s, here, k0, limit, mul, st, m, o, ob, pw);
    step_values<D, NT, NT>(pw, st, ones, o, ob);
    if (any_bad) mark_bad<D, NT, NT>(s_note[buf].bad, k0, limit, ob);
    turn(i);
  }
  for (; i < steps; ++i, k0 += AT_STEP) turn(i);

  // ---- rows out through LDS ----
  m[0] = m[0] * mul[0];
  const float total = sum_of<D>(ob[0]);
  if (kg == 0) { s_m[wave * 16 + n16] = m[0]; s_l[wave * 16 + n16] = total; }
  float* s_o = reinterpret_cast<float*>(lds);
  put_sums<D>(o[0], ob[0], unit, 1.0f, s_o + wave * 16 * (D + 4));
  lds_barrier();
  for (int i = tid; i < 64 * (D / 4); i += 256) {
    const int in = i / (D / 4), d = 4 * (i % (D / 4));
    if (in >= rows_here) break;
    const int row = row0 + in, tok = row / group;
    put_row<D, BF>(a, cut, slot, in, start + tok, h * group + (row - tok * group), d, *reinterpret_cast<const float4*>(s_o + in * (D + 4) + d), s_m[in], s_l[in]);
  }
}

// Partial sums joined.  WIDE: a workgroup per row; its waves read 256 / D partial rows at once, 16 bytes a lane, four such loads
// in flight, and meet in LDS.  Otherwise a wave per row, 16 rows a workgroup.  A launch and three dependent trips: 4-5.5 us.
template <int D, bool BF, int TILE, bool WIDE>
__global__ __launch_bounds__(256) void k_kv4_attn_merge(Pool pool, sl_kv4_attn_args a, AttnCut cut) {
  constexpr int LANES = D / 4, PER_WAVE = 64 / LANES, WAVES = WIDE ? 4 : 1, PER = WAVES * PER_WAVE;
  __shared__ float s_red[4];
  __shared__ float4 s_y[4 * PER_WAVE][LANES];
  __shared__ float s_sum[4 * PER_WAVE];
  const int h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = a.n_heads / pool.n_kv;
  int start, n;
  const int rows = rows_of(a, r, start, n), row_first = WIDE ? blockIdx.x : blockIdx.x * 16;
  if (row_first >= rows * group) return;
  const int tile = row_first / TILE, tiles = (rows * group + TILE - 1) / TILE, share = cut.first[a.n_req + 1];
  const long keys = seen_keys(a, pool, r);
  long last;
  int count, per;
  tile_cut<TILE>(keys, n, rows * group, tile, group, share, last, count, per);
  if (count == 1) return;                               // one workgroup had all of it and wrote the rows
  const int most = parts_of(rounds_for(min(keys, keys - n + rows)), round_cost(TILE, rows * group), share);      // parts that each item is numbered with
  // as find_part numbers them: part i of the item stands at first + i * side
  const int items = tiles * pool.n_kv, item = (TILE > 16 ? tiles - 1 - tile : tile) * pool.n_kv + h, full = items & ~7, side = item < full ? 8 : items - full;
  const long first = cut.first[r] + (item < full ? (long)(item & ~7) * most + (item & 7) : (long)full * most + (item - full));
  if (cut.first[r] + (long)items * most > cut.slots) return;      // (row offsets that overlap: more parts than rows allow)
  const float* stat = cut.part + cut.slots * cut.rows * D;
  const int d = 4 * (lane % LANES), mine = (WIDE ? wave * PER_WAVE : 0) + lane / LANES;
  for (int j = 0; j < (WIDE ? 1 : 4); ++j) {
    const int row = WIDE ? row_first : row_first + wave * 4 + j, in = row % TILE;
    if (row >= rows * group) return;
    float best = -__builtin_inff();
    for (int i = WIDE ? tid : lane; i < count; i += 64 * WAVES) best = fmaxf(best, stat[(first + (long)i * side) * cut.rows + in]);
    best = tree_max<64>(best);
    if constexpr (WIDE) {
      if (lane == 0) s_red[wave] = best;
      __syncthreads();
      best = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    }
    float4 y = make_float4(0, 0, 0, 0);
    float sum = 0.0f;
    for (int i = mine; i < count; i += 4 * PER) {
      float4 p[4];
      float m[4], l[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool in_range = i + u * PER < count;
        const long slot = first + (long)(in_range ? i + u * PER : i) * side;
        p[u] = *reinterpret_cast<const float4*>(cut.part + (slot * cut.rows + in) * D + d);
        m[u] = in_range ? stat[slot * cut.rows + in] : -__builtin_inff();
        l[u] = in_range ? stat[(cut.slots + slot) * cut.rows + in] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (m[u] == -__builtin_inff() && l[u] == 0.0f) continue;         // a part in which the row sees no key; one whose scores are all NaN has that sum
        const float f = __builtin_amdgcn_exp2f(m[u] - best);
        sum = fmaf(f, l[u], sum);
        y.x = fmaf(f, p[u].x, y.x); y.y = fmaf(f, p[u].y, y.y); y.z = fmaf(f, p[u].z, y.z); y.w = fmaf(f, p[u].w, y.w);
      }
    }
    const int slot_y = WIDE ? mine : wave * PER_WAVE + lane / LANES;
    s_y[slot_y][lane % LANES] = y;
    if (lane % LANES == 0) s_sum[slot_y] = sum;
    if constexpr (WIDE) __syncthreads(); else wave_lds_order();
    const int lead = WIDE ? tid : lane;
    if (lead < LANES) {
      sum = 0.0f; y = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int from = (WIDE ? 0 : wave * PER_WAVE) + i;
        const float4 x = s_y[from][lead];
        sum += s_sum[from]; y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
      }
      const int tok = row / group;
      finish_row<BF>(a, start + tok, h * group + (row - tok * group), 4 * lead, y, sum);
    }
    if constexpr (!WIDE) wave_lds_order();
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------
int launch_status() { return hipGetLastError() == hipSuccess ? SL_OK : SL_ERR_DEVICE; }
int page_shift_of(int page_size) {
  for (int s = 4; s <= 8; ++s) if (page_size == 1 << s) return s;
  return -1;
}
bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }
bool layout_ok(int page_size, int n_kv, int head_dim) {
  return page_shift_of(page_size) >= 0 && n_kv >= 1 && n_kv <= 1024 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}
int pool_of(const sl_kv4_pool* p, Pool& out) {
  if (!p || !p->pages || !aligned(p->pages, 16) || p->n_pages < 1 || p->n_kv < 1) return SL_ERR_ARG;
  if (!layout_ok(p->page_size, p->n_kv, p->head_dim)) return SL_ERR_UNSUPPORTED;
  if ((int64_t)p->n_pages * p->page_size > 0x7fffffffLL) return SL_ERR_TOO_LARGE;
  out = Pool{(unsigned char*)p->pages, p->n_pages, page_shift_of(p->page_size), p->n_kv};
  return SL_OK;
}
// How a call is cut, from what the host knows.
struct AttnShape {
  AttnCut cut{};
  int tile = 16;              // rows of a workgroup
  int grid = 0;
  bool wide = true;           // many parts to a row: a workgroup joins one
  int64_t part_bytes = 0, bytes = 0;
};
constexpr int64_t MAX_GROUPS = 0xffffffffLL / 256;      // workgroups of 256 along one axis: a launch has fewer than 2^32 threads there
int compute_units() {         // of the current device
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
int attn_shape(const sl_kv4_pool* p, const sl_kv4_attn_args* a, AttnShape& sh) {
  if (!p || !a || a->n_heads < 1 || p->n_kv < 1 || a->n_heads % p->n_kv || a->n_req < 1 || a->max_rows < 1 || !layout_ok(p->page_size, p->n_kv, p->head_dim)) return SL_ERR_ARG;
  const int64_t group = a->n_heads / p->n_kv, rows = (int64_t)std::min(a->max_rows, std::max(a->n_tokens, 1)) * group;
  const int64_t widest = (int64_t)a->table_width * p->page_size;
  if (a->n_req > AT_MAX_REQ || a->n_heads > 65535 || rows > MAX_GROUPS || widest > 0x7fffffffLL - 4096) return SL_ERR_TOO_LARGE;
  // 256 dims: 16 rows a workgroup, from 49 rows on 64 (32 lanes of 32 rows 66 against 98 us, of 64 rows 140 against 103); fewer dims: a
  // second row tile as soon as there are rows for it (128 dims, six requests of 32 rows at 20-32K: 71 against 83 us).
  sh.tile = p->head_dim == 256 ? (rows <= 48 ? 16 : 64) : (rows <= 16 ? 16 : 32);
  const int tile = sh.tile;
  // items: by the most rows of a request, and by all rows of the call
  const int64_t items = p->n_kv * std::min(a->n_req * ((rows + tile - 1) / tile), a->n_tokens * group / tile + a->n_req);
  const int64_t resident = (int64_t)compute_units() * (tile == 64 ? 2 : attn_places(p->head_dim, tile / 16));
  const int64_t rounds = items * (std::min<int64_t>(widest, a->max_keys) / AT_UNIT + 1);
  if (p->n_kv * a->n_req * ((rows + tile - 1) / tile) + 4 * resident > MAX_GROUPS) return SL_ERR_TOO_LARGE;
  // How many parts.  Up to three quarters of the chip's places in items: as many parts as places, no more (128 lanes of 256 dims 83 us,
  // two turns of parts 91, unchecked 102; 40 verify requests 63, 69, 72).  More items: single tokens are cut for two
  // turns, from one and a half turns of items on for one (200 lanes 121 and 133, 500 lanes 224 and 210).  Row tiles of a prompt that
  // begins here see from nothing to all of it: the longest first and uncut, the chip takes them as it gets free (2048 rows of
  // 256 dims 140 us, parts of the mean 160; of 64 dims 34 and 46), unless there are fewer than two thirds of the places (1024 rows
  // 84 and 67).  Chunks behind a long context are alike: uncut where whole turns of items fill the chip to 85 % (2048 rows behind
  // 4096 390 us, cut for three turns 434), else cut (2333 rows in three requests 1520 and 975; of 64 dims 243, for two turns 189,
  // for three 193).
  const int64_t whole = (items + resident - 1) / resident;
  const bool alike = a->max_keys > 2ll * a->max_rows;
  int64_t want = resident;
  if (tile != 16 && !alike && 3 * items >= 2 * resident) want = items / 2;
  else if (4 * items <= 3 * resident) sh.cut.turns = 4;
  else if (tile == 16) { want = 2 * items <= 3 * resident ? 2 * resident : resident; sh.cut.turns = 4; }
  else want = items * 20 >= whole * resident * 17 ? items / 2 : (tile == 64 ? 3 : 2) * resident;
  sh.cut.want = (int)std::min(want, std::max<int64_t>(rounds, 1));
  // a request's items are numbered with the parts of its longest row tile: at most twice the mean of longest and shortest
  sh.grid = (int)(2 * sh.cut.want + items);
  // Joining: a workgroup per row while there are few rows or many parts to each, else a wave per row (2333 rows of 64 dims on 16K keys
  // 213 us with the first, 183 with the second; 128 lanes of 8 rows 102 and 105, 64 rows on 32K keys 97 and 113).
  sh.wide = rows * p->n_kv * a->n_req <= 4096 || sh.cut.want > 8 * items;
  sh.cut.slots = sh.grid; sh.cut.rows = (int)std::min<int64_t>(rows, tile);
  sh.part_bytes = sh.cut.slots * sh.cut.rows * (p->head_dim + 2) * 4;
  sh.part_bytes = (sh.part_bytes + 15) & ~15ll;
  sh.bytes = sh.part_bytes + ((a->n_req + 2) * 4 + 15) / 16 * 16;
  return SL_OK;
}
template <class K>
void launch_attn_kernel(K kernel, int lds, const Pool& pool, const sl_kv4_attn_args& a, const AttnCut& cut, int grid, hipStream_t st) {
  lds += a.n_req <= 64 ? 0 : (a.n_req + 1) * 4;
  if (lds > 65536) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, st, pool, a, cut);
}
template <int D, bool BF>
void launch_attn(const Pool& pool, const sl_kv4_attn_args& a, const AttnCut& cut, const AttnShape& sh, hipStream_t st) {
  const int rows = std::min(a.max_rows, a.n_tokens) * (a.n_heads / pool.n_kv);
#define KV4_ATTN(TILE, KERNEL, LDS)                                                                            \
  do {                                                                                                         \
    launch_attn_kernel(KERNEL, LDS, pool, a, cut, sh.grid, st);                                                \
    if (sh.wide) hipLaunchKernelGGL((k_kv4_attn_merge<D, BF, TILE, true>), dim3(rows, pool.n_kv, a.n_req), dim3(256), 0, st, pool, a, cut);               \
    else hipLaunchKernelGGL((k_kv4_attn_merge<D, BF, TILE, false>), dim3((rows + 15) / 16, pool.n_kv, a.n_req), dim3(256), 0, st, pool, a, cut);          \
  } while (0)
  if (sh.tile == 16) KV4_ATTN(16, (k_kv4_attn<D, BF, 1>), (AttnLds<D, 1>::BYTES));
  else if constexpr (D == 256) KV4_ATTN(64, (k_kv4_attn_tile<D, BF>), TileLds<D>::BYTES);
  else KV4_ATTN(32, (k_kv4_attn<D, BF, 2>), (AttnLds<D, 2>::BYTES));
#undef KV4_ATTN
}
// f<D, BF>() for the pool's head_dim and an element type
#define KV4_BY_LAYOUT(dim, bf, CALL)                                        \
  do {                                                                      \
    if ((dim) == 256) { if (bf) { CALL(256, true); } else { CALL(256, false); } }      \
    else if ((dim) == 128) { if (bf) { CALL(128, true); } else { CALL(128, false); } } \
    else { if (bf) { CALL(64, true); } else { CALL(64, false); } }          \
  } while (0)

}  // namespace

extern "C" {

int64_t sl_kv4_page_bytes(int page_size, int n_kv, int head_dim) {
  return layout_ok(page_size, n_kv, head_dim) ? (int64_t)page_size * n_kv * (9 * head_dim / 8) : 0;
}

int sl_kv4_plan(const sl_kv4_plan_args* a, void* stream) {
  if (!a || a->n_req < 0 || a->table_width < 0 || a->n_free < 0 || a->max_tokens < 0) return SL_ERR_ARG;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0) return SL_ERR_UNSUPPORTED;
  if (a->n_req > PLAN_MAX_REQ || (int64_t)a->n_req * a->table_width + a->n_free > 0x7fffffffLL || a->max_tokens > (1 << 30)) return SL_ERR_TOO_LARGE;
  const bool table = a->n_req > 0 && a->table_width > 0;
  if ((a->n_req > 0 && (!a->ctx_len || !a->new_len || !a->held_in || !a->held_out || !a->kv_len)) || (table && (!a->table_in || !a->table_out)) ||
      (a->n_free > 0 && (!a->free_in || !a->free_out)) || !a->free_count_in || !a->free_count_out || !a->q_start || !a->unserved ||
      (a->max_tokens > 0 && (!a->slot || !a->pos))) return SL_ERR_ARG;
  // (a step planned into the tensors that it is planned from: workgroups would read what others have written)
  const int32_t* ins[] = {a->n_req ? a->ctx_len : nullptr, a->n_req ? a->new_len : nullptr, a->n_req ? a->held_in : nullptr, table ? a->table_in : nullptr,
                          a->n_free ? a->free_in : nullptr, a->free_count_in};
  const int32_t* outs[] = {a->n_req ? a->held_out : nullptr, a->n_req ? a->kv_len : nullptr, table ? a->table_out : nullptr, a->n_free ? a->free_out : nullptr,
                           a->free_count_out, a->q_start, a->max_tokens ? a->slot : nullptr, a->max_tokens ? a->pos : nullptr, a->unserved};
  for (const int32_t* in : ins) for (const int32_t* out : outs) if (in && in == out) return SL_ERR_ARG;
  const int64_t most = std::max(a->n_free, a->max_tokens);
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(512, std::max<int64_t>(a->n_req, (most + PLAN_THREADS - 1) / PLAN_THREADS)));
  (void)hipGetLastError();            // an error an unrelated earlier call of this thread left behind is not this call's
  hipLaunchKernelGGL(k_kv4_plan, dim3((unsigned)blocks), dim3(PLAN_THREADS), 0, (hipStream_t)stream, *a, shift);
  return launch_status();
}

int sl_kv4_append(const sl_kv4_pool* p, const sl_kv4_append_args* a, void* stream) {
  Pool pool;
  int r = pool_of(p, pool); if (r) return r;
  if (!a || a->n_tokens < 0 || (a->dtype != SL_F16 && a->dtype != SL_BF16) || !(a->eps >= 0.0)) return SL_ERR_ARG;
  if (a->rot_dim < 0 || a->rot_dim % 8 || a->rot_dim > p->head_dim || (a->rot_dim && a->max_pos < 1)) return SL_ERR_ARG;
  if (a->n_tokens == 0) return SL_OK;
  if (!a->k || !a->v || !a->slot || (a->q && (!a->q_out || a->n_heads < 1)) || (a->rot_dim && (!a->cos || !a->sin || !a->pos))) return SL_ERR_ARG;
  const void* eight[] = {a->q, a->k, a->v, a->q_out, a->q_weight, a->k_weight};
  for (const void* x : eight) if (!aligned(x, 8)) return SL_ERR_ARG;
  const int64_t strides[] = {a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head, a->out_token, a->out_head};
  for (int i = a->q ? 0 : 2; i < (a->q ? 8 : 6); ++i) if (strides[i] % 4) return SL_ERR_ARG;
  if (a->rot_dim && (!aligned(a->cos, 16) || !aligned(a->sin, 16))) return SL_ERR_ARG;
  if (a->n_heads > 32768 || a->n_tokens > 4 * (MAX_GROUPS - 8)) return SL_ERR_TOO_LARGE;
  const int heads = 256 / p->head_dim, q_units = a->q ? (a->n_heads + heads - 1) / heads : 0;
  const int kv_units = (p->n_kv + heads - 1) / heads;
  // enough waves to fill the chip come first, then longer runs of heads (2048 tokens of 16 + 2 heads with their read-back: 22.3 us
  // with runs from 16384 waves on, 20.8 from 4096 on; 7.6K tokens of 32 + 8 heads: runs of 1, 2, 4, 8, 16 units 110, 86, 77, 73, 73)
  const int64_t waves = (int64_t)a->n_tokens * (q_units + 2 * kv_units);
  const int per = (int)std::max<int64_t>(1, std::min<int64_t>(8, waves / 2048));
  const int runs = (q_units + per - 1) / per + 2 * ((kv_units + per - 1) / per);
  (void)hipGetLastError();
#define KV4_CALL(D, BF) hipLaunchKernelGGL((k_kv4_append<D, BF>), dim3((a->n_tokens + 31) / 32 * 8, runs), dim3(256), 0, (hipStream_t)stream, pool, *a, q_units, kv_units, per)
  KV4_BY_LAYOUT(p->head_dim, a->dtype == SL_BF16, KV4_CALL);
#undef KV4_CALL
  return launch_status();
}

int64_t sl_kv4_attention_workspace(const sl_kv4_pool* p, const sl_kv4_attn_args* a) {
  AttnShape sh;
  return attn_shape(p, a, sh) == SL_OK ? sh.bytes : 0;
}

int sl_kv4_attention(const sl_kv4_pool* p, const sl_kv4_attn_args* a, void* stream) {
  Pool pool;
  int r = pool_of(p, pool); if (r) return r;
  if (!a || a->n_req < 0 || a->n_tokens < 0 || a->table_width < 0 || (a->dtype != SL_F16 && a->dtype != SL_BF16)) return SL_ERR_ARG;
  if (a->n_heads < 1 || a->n_heads % p->n_kv || a->max_rows < 0 || a->max_keys < 1 || !std::isfinite(a->scale)) return SL_ERR_ARG;
  if (a->n_req == 0 || a->n_tokens == 0 || a->max_rows == 0) return SL_OK;
  if (!a->q || !a->out || !a->q_start || !a->kv_len || (!a->table && a->table_width > 0)) return SL_ERR_ARG;
  const void* sixteen[] = {a->q, a->gate, a->out};
  for (const void* x : sixteen) if (!aligned(x, 16)) return SL_ERR_ARG;
  const int64_t strides[] = {a->q_token, a->q_head, a->out_token, a->out_head, a->gate ? a->gate_token : 0, a->gate ? a->gate_head : 0};
  for (int64_t x : strides) if (x % 8) return SL_ERR_ARG;
  AttnShape sh;
  r = attn_shape(p, a, sh); if (r) return r;
  if (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < sh.bytes) return SL_ERR_ARG;
  AttnCut cut = sh.cut;
  cut.part = (float*)a->workspace;
  cut.first = (int32_t*)((unsigned char*)a->workspace + sh.part_bytes);
  (void)hipGetLastError();
#define KV4_CALL(D, BF) launch_attn<D, BF>(pool, *a, cut, sh, (hipStream_t)stream)
  KV4_BY_LAYOUT(p->head_dim, a->dtype == SL_BF16, KV4_CALL);
#undef KV4_CALL
  return launch_status();
}

int sl_kv4_read(const sl_kv4_pool* p, const int32_t* slots, int n, int dtype, void* k_out, void* v_out, void* stream) {
  Pool pool;
  int r = pool_of(p, pool); if (r) return r;
  if (n < 0 || (dtype != SL_F32 && dtype != SL_F16) || !aligned(k_out, 16) || !aligned(v_out, 16)) return SL_ERR_ARG;
  if (n == 0 || (!k_out && !v_out)) return SL_OK;
  if (!slots) return SL_ERR_ARG;
  const int64_t blocks = ((int64_t)n + 4 * (1024 / p->head_dim) - 1) / (4 * (1024 / p->head_dim));
  if (blocks > MAX_GROUPS) return SL_ERR_TOO_LARGE;
  (void)hipGetLastError();
#define KV4_CALL(D, F16) hipLaunchKernelGGL((k_kv4_read<D, F16>), dim3((unsigned)blocks, p->n_kv), dim3(256), 0, (hipStream_t)stream, pool, slots, n, k_out, v_out)
  KV4_BY_LAYOUT(p->head_dim, dtype == SL_F16, KV4_CALL);
#undef KV4_CALL
  return launch_status();
}

}  // extern "C"
