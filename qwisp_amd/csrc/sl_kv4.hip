// Paged key/value cache held in 4 bits: page tables and slots from request lengths, norm + rotation + quantised store,
// attention over the pages, rows back as values.  Layout and rules: include/seedless_hip.h.
//
// Everything here only enqueues on the caller's stream.  What is read on the device (lengths, tables, slots) is checked
// on the device: an index that leaves its array is never followed.
#include "sl_device.cuh"
#include "../../include/seedless_hip.h"
#include <algorithm>

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
SL_DEV uint16_t f2bf(float x) {                       // to nearest, ties to even
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x7fc0;
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
template <bool BF>
SL_DEV float elem_f(uint16_t u) { return BF ? bf2f(u) : h2f(u); }
template <bool BF>
SL_DEV uint16_t f_elem(float x) { return BF ? f2bf(x) : f2h(x); }
template <bool BF>
SL_DEV void load4(const uint16_t* p, float* x) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  x[0] = elem_f<BF>((uint16_t)r.x); x[1] = elem_f<BF>((uint16_t)(r.x >> 16));
  x[2] = elem_f<BF>((uint16_t)r.y); x[3] = elem_f<BF>((uint16_t)(r.y >> 16));
}

// ---- page tables, slots and row offsets -----------------------------------------------------------------------------------
constexpr int PLAN_MAX_REQ = 4096;
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_PER = PLAN_MAX_REQ / PLAN_THREADS;

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

// Every workgroup forms the three running sums over the requests (rows, pages missing, pages given back) for itself, in
// LDS, and then fills its share of the outputs, an element per thread and step: one launch, no exchange between
// workgroups.  The requests' numbers are 12 bytes each and come from L2.
__global__ __launch_bounds__(PLAN_THREADS) void k_kv4_plan(sl_kv4_plan_args a, int page_shift) {
  __shared__ int s_row[PLAN_MAX_REQ + 1], s_need[PLAN_MAX_REQ + 1], s_give[PLAN_MAX_REQ + 1];
  __shared__ unsigned s_wave[PLAN_THREADS / 64];
  __shared__ unsigned s_fit[PLAN_MAX_REQ / 32];     // the request is served
  const int tid = threadIdx.x, n = a.n_req, per = (n + PLAN_THREADS - 1) / PLAN_THREADS, page = 1 << page_shift;
  const int W = a.table_width;
  for (int i = tid; i < (n + 31) / 32; i += PLAN_THREADS) s_fit[i] = 0;

  unsigned rows = 0, cap = (unsigned)a.max_tokens;
  for (int j = 0; j < per; ++j) {
    const int r = tid * per + j;
    if (r < n) rows = min(cap, rows + min(cap, (unsigned)max(a.new_len[r], 0)));
  }
  unsigned all_rows;
  unsigned row = scan_before(rows, cap, s_wave, all_rows);
  int need[PLAN_PER], give[PLAN_PER];
  bool sane[PLAN_PER];
  unsigned need_sum = 0, give_sum = 0;
  for (int j = 0; j < per; ++j) {
    const int r = tid * per + j;
    need[j] = give[j] = 0; sane[j] = false;
    if (r >= n) continue;
    const int ctx = a.ctx_len[r], nw = a.new_len[r], held = a.held_in[r];
    s_row[r] = (int)row;
    const long total = (long)ctx + nw;
    const bool fits = (unsigned)max(nw, 0) <= cap - row;
    sane[j] = ctx >= 0 && nw >= 0 && fits && held >= 0 && held <= W && total <= ((long)W << page_shift) && ctx <= ((long)held << page_shift);
    if (sane[j]) {
      const int want = (int)((total + page - 1) >> page_shift);
      need[j] = max(want - held, 0); give[j] = max(held - want, 0);
    }
    row = min(cap, row + min(cap, (unsigned)max(nw, 0)));
    need_sum += need[j]; give_sum += give[j];
  }
  unsigned all_need, all_give;
  unsigned nb = scan_before(need_sum, 0x7fffffffu, s_wave, all_need);
  unsigned gb = scan_before(give_sum, 0x7fffffffu, s_wave, all_give);
  const unsigned count = (unsigned)min(max(a.free_count_in[0], 0), a.n_free), have = count + all_give;
  // pages taken = what the served requests miss; they are the first ones of the running sum
  unsigned taken = 0;
  int unserved = 0;
  for (int j = 0; j < per; ++j) {
    const int r = tid * per + j;
    if (r >= n) continue;
    s_need[r] = (int)nb; s_give[r] = (int)gb;
    const bool fit = sane[j] && (need[j] == 0 || nb + need[j] <= have);
    if (fit) { atomicOr(&s_fit[r >> 5], 1u << (r & 31)); taken += need[j]; }
    else ++unserved;
    nb += need[j]; gb += give[j];
  }
  unsigned all_taken, all_unserved;
  scan_before(taken, 0x7fffffffu, s_wave, all_taken);
  scan_before((unsigned)unserved, 0x7fffffffu, s_wave, all_unserved);
  if (tid == 0) { s_row[n] = (int)all_rows; s_need[n] = (int)all_need; s_give[n] = (int)all_give; }
  __syncthreads();

  const int left = (int)(have - all_taken);
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
    if (c >= held && c < held + need_r && fit(r)) return free_at((int)have - 1 - s_need[r] - (c - held));
    return -1;
  };
  const int step = gridDim.x * PLAN_THREADS, at = blockIdx.x * PLAN_THREADS + tid;
  for (long i = at; i < (long)n * W; i += step) {
    const int r = (int)(i / W), c = (int)(i - (long)r * W), held = min(max(a.held_in[r], 0), W);
    a.table_out[i] = page_at(r, c, held);
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
  for (int r = at; r < n; r += step) {
    const bool f = fit(r);
    const int held = min(max(a.held_in[r], 0), W);
    a.held_out[r] = held - (s_give[r + 1] - s_give[r]) + (f ? s_need[r + 1] - s_need[r] : 0);
    a.kv_len[r] = f ? a.ctx_len[r] + a.new_len[r] : 0;
    a.q_start[r] = s_row[r];
  }
  if (at == 0) { a.q_start[n] = (int)all_rows; a.free_count_out[0] = min(left, a.n_free); a.unserved[0] = (int)all_unserved; }
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
SL_DEV float inv_sqrt(float x) { return 1.0f / sqrtf(x); }
SL_DEV double inv_sqrt(double x) { return 1.0 / sqrt(x); }

// A head row over D/4 lanes, four consecutive dims each: norm and rotation in precision F.
template <class F, int D, bool BF>
SL_DEV void turn_row(F* x, const uint16_t* weight, const float* cos_t, const float* sin_t, int half, int pos, double eps, int l) {
  if (weight) {
    const F ss = sum_lanes<D / 4>((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]));
    const F inv = inv_sqrt(ss / (F)D + (F)eps);
    float w[4];
    load4<BF>(weight + 4 * l, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * (F)w[i];
  }
  if (half) {
    const int hl = half / 4;                          // a half of the rotated dims, in lanes
    const bool low = l < hl, turns = l < 2 * hl;
    const int lane = threadIdx.x & 63, from = turns ? (low ? lane + hl : lane - hl) : lane;
    F y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __shfl(x[i], from);
    if (turns) {
      const size_t row = (size_t)pos * half + 4 * (low ? l : l - hl);
      const float4 c = *reinterpret_cast<const float4*>(cos_t + row), s = *reinterpret_cast<const float4*>(sin_t + row);
      const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = low ? x[i] * (F)cv[i] - y[i] * (F)sv[i] : x[i] * (F)cv[i] + y[i] * (F)sv[i];
    }
  }
}

// The four codes of this lane (16 lanes = one group of 64 dims), low nibble first, and the group's scale and bias.
// Double precision throughout: a value next to the border of two codes takes the side that exact arithmetic takes.
SL_DEV uint32_t quantise4(const double* v, uint32_t& sb) {
  const double lim = 65504.0;
  double x[4];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bad = bad || !(fabs(v[i]) <= 1.7976931348623157e308);
    x[i] = fmin(fmax(v[i], -lim), lim);
  }
  double mn = fmin(fmin(x[0], x[1]), fmin(x[2], x[3])), mx = fmax(fmax(x[0], x[1]), fmax(x[2], x[3]));
  mn = row16(mn, [](double a, double b) { return fmin(a, b); });
  mx = row16(mx, [](double a, double b) { return fmax(a, b); });
  const unsigned long long bads = __ballot(bad);
  if ((bads >> (threadIdx.x & 48)) & 0xffffull) { sb = 0x7e007e00u; return 0; }
  const bool low = fabs(mn) > fabs(mx);
  double scale = fmax((mx - mn) / 15.0, 1e-7);
  scale = low ? scale : -scale;
  const double edge = low ? mn : mx, steps = rint(edge / scale);
  double bias = 0.0;
  if (steps != 0.0) { scale = edge / steps; bias = edge; }
  const uint16_t hs = f2h((float)scale), hb = f2h((float)bias);
  const double s = (double)h2f(hs), b = (double)h2f(hb);
  sb = (uint32_t)hs | ((uint32_t)hb << 16);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) codes |= (uint32_t)fmin(fmax(rint((x[i] - b) / s), 0.0), 15.0) << (4 * i);
  return codes;
}

// A wave per (token, 256/D heads): D/4 lanes carry a head row.  Query heads first, then key heads, then value heads.
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_kv4_append(Pool pool, sl_kv4_append_args a, int q_units, int units) {
  constexpr int LANES = D / 4, HEADS = 64 / LANES;
  const int lane = threadIdx.x & 63, l = lane % LANES, sub = lane / LANES;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)a.n_tokens * units) return;
  const int t = (int)(item / units);
  int u = (int)(item - (long)t * units);
  const int pos = a.rot_dim ? a.pos[t] : 0, half = a.rot_dim / 2;
  const bool placed = !a.rot_dim || (pos >= 0 && pos < a.max_pos);
  if (u < q_units) {
    const int h = u * HEADS + sub;
    const bool there = h < a.n_heads;                 // (lanes without a head still take part in the exchanges)
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (there) load4<BF>((const uint16_t*)a.q + t * a.q_token + h * a.q_head + 4 * l, x);
    if (placed) turn_row<float, D, BF>(x, (const uint16_t*)a.q_weight, a.cos, a.sin, half, pos, a.eps, l);
    else { x[0] = x[1] = x[2] = x[3] = 0.0f; }
    if (there)
      *reinterpret_cast<uint2*>((uint16_t*)a.q_out + t * a.out_token + h * a.out_head + 4 * l) =
          make_uint2((uint32_t)f_elem<BF>(x[0]) | ((uint32_t)f_elem<BF>(x[1]) << 16), (uint32_t)f_elem<BF>(x[2]) | ((uint32_t)f_elem<BF>(x[3]) << 16));
    return;
  }
  u -= q_units;
  const int slot = a.slot[t];
  if (!placed || slot < 0 || (slot >> pool.page_shift) >= pool.n_pages) return;
  const int kv_units = (units - q_units) / 2;
  const bool key = u < kv_units;
  const int h = (key ? u : u - kv_units) * HEADS + sub;
  const bool there = h < pool.n_kv;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (there) load4<BF>(key ? (const uint16_t*)a.k + t * a.k_token + h * a.k_head + 4 * l : (const uint16_t*)a.v + t * a.v_token + h * a.v_head + 4 * l, x);
  double y[4] = {x[0], x[1], x[2], x[3]};
  if (key) turn_row<double, D, BF>(y, (const uint16_t*)a.k_weight, a.cos, a.sin, half, pos, a.eps, l);
  uint32_t sb;
  const uint32_t codes = quantise4(y, sb);
  if (!there) return;
  const int off = slot & ((1 << pool.page_shift) - 1), part = (D / 2) << pool.page_shift, sbs = (D / 16) << pool.page_shift;
  unsigned char* at = head_at<D>(pool, slot >> pool.page_shift, h) + (key ? 0 : part + sbs);
  *reinterpret_cast<uint16_t*>(at + (key ? key_codes_at<D>(off, 4 * l) : value_codes_at<D>(off, 4 * l))) = (uint16_t)codes;
  if (l % 16 == 0) reinterpret_cast<uint32_t*>(at + part)[off * (D / 64) + l / 16] = sb;
}

// ---- rows as values -----------------------------------------------------------------------------------------------------
template <int D, bool F16>
__global__ __launch_bounds__(256) void k_kv4_read(Pool pool, const int32_t* slots, long items, void* k_out, void* v_out) {
  constexpr int LANES = D / 4;
  const int l = (threadIdx.x & 63) % LANES;
  const long item = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;     // (row, head)
  if (item >= items) return;
  const int row = (int)(item / pool.n_kv), h = (int)(item - (long)row * pool.n_kv);
  const int slot = slots[row];
  const bool in = slot >= 0 && (slot >> pool.page_shift) < pool.n_pages;
  const int off = slot & ((1 << pool.page_shift) - 1), part = (D / 2) << pool.page_shift, sbs = (D / 16) << pool.page_shift;
  const unsigned char* base = head_at<D>(pool, in ? slot >> pool.page_shift : 0, h);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    void* out = kv ? v_out : k_out;
    if (!out) continue;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
      const unsigned char* at = base + (kv ? part + sbs : 0);
      const uint32_t codes = *reinterpret_cast<const uint16_t*>(at + (kv ? value_codes_at<D>(off, 4 * l) : key_codes_at<D>(off, 4 * l)));
      const uint32_t sb = reinterpret_cast<const uint32_t*>(at + part)[off * (D / 64) + l / 16];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaf(lo_h(sb), (float)((codes >> (4 * i)) & 15u), hi_h(sb));
    }
    const size_t to = (size_t)item * D + 4 * l;
    if (F16) *reinterpret_cast<uint2*>((uint16_t*)out + to) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
    else *reinterpret_cast<float4*>((float*)out + to) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// ---- attention ------------------------------------------------------------------------------------------------------------
// One wave per (row, query head), a key after the other: running maximum m and sum l of the softmax, o rescaled when m
// moves.
template <int D, bool BF>
__global__ __launch_bounds__(64) void k_kv4_attn_rows(Pool pool, sl_kv4_attn_args a) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y;
  if (t >= a.q_start[a.n_req]) return;
  const int r = owner_of(a.q_start, a.n_req, t), i = t - a.q_start[r], n = a.q_start[r + 1] - a.q_start[r];
  if (i < 0 || i >= n || i >= a.max_rows) return;
  const int kvh = h / (a.n_heads / pool.n_kv);
  const long seen = min((long)a.kv_len[r], (long)a.table_width << pool.page_shift) - n + i + 1;
  float q[PER], o[PER], m = -__builtin_inff(), sum = 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    q[j] = a.scale * elem_f<BF>(((const uint16_t*)a.q)[t * a.q_token + h * a.q_head + lane + 64 * j]);
    o[j] = 0.0f;
  }
  const int part = (D / 2) << pool.page_shift, sbs = (D / 16) << pool.page_shift;
  for (long key = 0; key < seen; ++key) {
    const int page = a.table[(size_t)r * a.table_width + (key >> pool.page_shift)], off = (int)key & ((1 << pool.page_shift) - 1);
    if (page < 0 || page >= pool.n_pages) continue;
    const unsigned char* at = head_at<D>(pool, page, kvh);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int d = lane + 64 * j;
      const uint32_t sb = reinterpret_cast<const uint32_t*>(at + part)[off * (D / 64) + j];
      const uint32_t c = (at[key_codes_at<D>(off, d)] >> (4 * (d & 1))) & 15u;
      s = fmaf(q[j], fmaf(lo_h(sb), (float)c, hi_h(sb)), s);
    }
    s = tree_sum<64>(s);
    const float top = fmaxf(m, s), back = m == top ? 1.0f : expf(m - top), p = s == top ? 1.0f : expf(s - top);
    m = top;
    sum = sum * back + p;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int d = lane + 64 * j;
      const uint32_t sb = reinterpret_cast<const uint32_t*>(at + part + sbs + part)[off * (D / 64) + j];
      const uint32_t c = (at[part + sbs + value_codes_at<D>(off, d)] >> (4 * (d & 1))) & 15u;
      o[j] = fmaf(p, fmaf(lo_h(sb), (float)c, hi_h(sb)), o[j] * back);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = lane + 64 * j;
    float y = sum != 0.0f ? o[j] / sum : 0.0f;
    if (a.gate) y = y * (1.0f / (1.0f + expf(-elem_f<BF>(((const uint16_t*)a.gate)[t * a.gate_token + h * a.gate_head + d]))));
    ((uint16_t*)a.out)[t * a.out_token + h * a.out_head + d] = f_elem<BF>(y);
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
  if (a->n_req > PLAN_MAX_REQ || (int64_t)a->n_req * a->table_width > 0x7fffffffLL || a->max_tokens > (1 << 30)) return SL_ERR_TOO_LARGE;
  const bool table = a->n_req > 0 && a->table_width > 0;
  if ((a->n_req > 0 && (!a->ctx_len || !a->new_len || !a->held_in || !a->held_out || !a->kv_len)) || (table && (!a->table_in || !a->table_out)) ||
      (a->n_free > 0 && (!a->free_in || !a->free_out)) || !a->free_count_in || !a->free_count_out || !a->q_start || !a->unserved ||
      (a->max_tokens > 0 && (!a->slot || !a->pos))) return SL_ERR_ARG;
  if ((table && a->table_in == a->table_out) || (a->n_free > 0 && a->free_in == a->free_out) || a->free_count_in == a->free_count_out ||
      (a->n_req > 0 && a->held_in == a->held_out)) return SL_ERR_ARG;
  const int64_t most = std::max<int64_t>((int64_t)a->n_req * a->table_width, std::max(a->n_free, a->max_tokens));
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(512, (most + PLAN_THREADS - 1) / PLAN_THREADS));
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
  if (a->n_heads > 65536) return SL_ERR_TOO_LARGE;
  const int heads = 256 / p->head_dim, q_units = a->q ? (a->n_heads + heads - 1) / heads : 0;
  const int units = q_units + 2 * ((p->n_kv + heads - 1) / heads);
  const int64_t blocks = ((int64_t)a->n_tokens * units + 3) / 4;
  if (blocks > 0x7fffffffLL) return SL_ERR_TOO_LARGE;
  (void)hipGetLastError();
#define KV4_CALL(D, BF) hipLaunchKernelGGL((k_kv4_append<D, BF>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, pool, *a, q_units, units)
  KV4_BY_LAYOUT(p->head_dim, a->dtype == SL_BF16, KV4_CALL);
#undef KV4_CALL
  return launch_status();
}

int64_t sl_kv4_attention_workspace(const sl_kv4_pool* p, const sl_kv4_attn_args* a) {
  (void)p; (void)a;
  return 0;
}

int sl_kv4_attention(const sl_kv4_pool* p, const sl_kv4_attn_args* a, void* stream) {
  Pool pool;
  int r = pool_of(p, pool); if (r) return r;
  if (!a || a->n_req < 0 || a->n_tokens < 0 || a->table_width < 0 || (a->dtype != SL_F16 && a->dtype != SL_BF16)) return SL_ERR_ARG;
  if (a->n_heads < 1 || a->n_heads % p->n_kv || a->max_rows < 0 || a->max_keys < 1) return SL_ERR_ARG;
  if (a->n_req == 0 || a->n_tokens == 0 || a->max_rows == 0) return SL_OK;
  if (!a->q || !a->out || !a->table || !a->q_start || !a->kv_len) return SL_ERR_ARG;
  const void* sixteen[] = {a->q, a->gate, a->out};
  for (const void* x : sixteen) if (!aligned(x, 16)) return SL_ERR_ARG;
  const int64_t strides[] = {a->q_token, a->q_head, a->out_token, a->out_head, a->gate ? a->gate_token : 0, a->gate ? a->gate_head : 0};
  for (int64_t x : strides) if (x % 8) return SL_ERR_ARG;
  if (a->n_heads > 65535) return SL_ERR_TOO_LARGE;
  (void)hipGetLastError();
#define KV4_CALL(D, BF) hipLaunchKernelGGL((k_kv4_attn_rows<D, BF>), dim3(a->n_tokens, a->n_heads), dim3(64), 0, (hipStream_t)stream, pool, *a)
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
  const int64_t items = (int64_t)n * p->n_kv, blocks = (items * (p->head_dim / 4) + 255) / 256;
  if (blocks > 0x7fffffffLL) return SL_ERR_TOO_LARGE;
  (void)hipGetLastError();
#define KV4_CALL(D, F16) hipLaunchKernelGGL((k_kv4_read<D, F16>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, pool, slots, (long)items, k_out, v_out)
  KV4_BY_LAYOUT(p->head_dim, dtype == SL_F16, KV4_CALL);
#undef KV4_CALL
  return launch_status();
}

}  // extern "C"
