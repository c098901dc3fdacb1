// bank8_attn.hip -- attention of each request's rows over its pages of the 8-bit bank.
//
// Both products run "swapped" on v_mfma_f32_32x32x16_f16, as in mha.hip:
//   S^T[token][row] = K_tile . Q^T          O^T[dim][row] += V^T_tile . P^T
// so a row's softmax statistics live in one lane (and its lane^32 partner) and the accumulators of S^T are the B operand of the
// second product.  `row` is a (query token, query head of the group) pair: the heads that share a kv head share its tiles.
// Codes become fp16 exactly (8 bits fit into 11), so the key scale is applied to the scores, once per element beside the softmax
// scale, and the value scale rides in the exponent: w = 2^(y - m), y = scale log2e ks s + log2 vs, O = sum w code, and the
// denominator takes each tile's sum of weights times 1 / vs.  No dequantised value exists anywhere.
// Queries enter as fp16 times a power of two per row that puts the row's largest element at 2^14: fp16 and bf16 rows are exact
// down to 2^-38 of that element; fp32 rows keep 22 bits in two planes (NS = 2: two products against the same codes).
// Weights are 2^10 times their usual size (the maximum is 2^10, not 1), which leaves 24 instead of 14 binades of normal fp16
// numbers below the maximum; fp32 calls keep them in two planes.  Sums are fp32, of the unrounded weights.
#include "bank8.h"

using namespace bank8;

namespace {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float LIFT = 10.f;             // log2 of the largest weight
constexpr float LOWEST = -3.0e38f;       // running maximum of a row that has seen nothing
constexpr float VS_MIN = 1.262177448e-29f;   // 2^-96: 1 / vs times 2^10 times 2^20 tokens stays finite

// ---------------------------------------------------------------------------------------------------- division into units
// A unit of work is (request, tile of ROWS rows, one of ns equal parts of the tokens that the tile sees) for one kv head.  Every
// part has at most `chunk` 32-token tiles, chunk = (all row tiles' token tiles) / want, so the parts of long and short requests
// cost the same and nothing is decided on the host, which does not know the lengths.  Each wave computes the same division from
// cu and lens: 64 requests at a time, two passes (total, then position).
struct Unit {
  int r, rt, part, ns;    // request, row tile, part of ns
  int q0, n, len;         // first row, rows, tokens
  int slot;               // index of the partial result of part 0 (ns > 1)
};

struct Req {
  int q0, n, len, rt, tiles;
};

template <int ROWS>
__device__ __forceinline__ Req request(const rmem_bank8_attn_args& a, int r, int G) {
  Req x = {0, 0, 0, 0, 0};
  if (r >= a.reqs) return x;
  int q0 = a.cu[r], q1 = a.cu[r + 1], len = a.lens[r];
  q0 = q0 < 0 ? 0 : q0 > a.rows ? a.rows : q0;
  q1 = q1 < q0 ? q0 : q1 > a.rows ? a.rows : q1;
  const long cap = (long)a.cols * a.bank.page;
  x.q0 = q0;
  x.n = q1 - q0;
  x.len = len < 0 ? 0 : len > cap ? (int)cap : len;
  x.rt = (int)(((long)x.n * G + ROWS - 1) / ROWS);
  x.tiles = (x.len + 31) >> 5;
  return x;
}

__device__ __forceinline__ long wave_sum_long(long v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const unsigned lo = __shfl_xor((unsigned)v, o), hi = __shfl_xor((unsigned)((unsigned long)v >> 32), o);
    v += (long)(((unsigned long)hi << 32) | lo);
  }
  return v;
}

// by_parts: index counts (request, row tile, part); otherwise (request, row tile) of requests in more than one part (the merge).
template <int ROWS>
__device__ bool find_unit(const rmem_bank8_attn_args& a, int G, long index, bool by_parts, int want, int chunk_min, Unit& u) {
  const int lane = threadIdx.x & 63;
  Req x = request<ROWS>(a, lane, G);
  long total = (long)x.rt * x.tiles;
  for (int b = 64; b < a.reqs; b += 64) {
    const Req y = request<ROWS>(a, b + lane, G);
    total += (long)y.rt * y.tiles;
  }
  total = wave_sum_long(total);
  long chunk = (total + want - 1) / want;
  chunk = chunk < chunk_min ? chunk_min : chunk;
  long seen = 0, slots = 0;
  for (int b = 0; b < a.reqs; b += 64) {
    if (b) x = request<ROWS>(a, b + lane, G);
    const int ns = x.tiles > chunk ? (int)((x.tiles + chunk - 1) / chunk) : 1;
    const int split = ns > 1 ? x.rt * ns : 0;
    int cnt = by_parts ? x.rt * ns : ns > 1 ? x.rt : 0;
    int c = cnt, s = split;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int cu = __shfl_up(c, o), su = __shfl_up(s, o);
      if (lane >= o) {
        c += cu;
        s += su;
      }
    }
    const unsigned long long hit = __ballot(index < seen + c);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      u.ns = __builtin_amdgcn_readlane(ns, l);
      int k = (int)(index - seen) - (__builtin_amdgcn_readlane(c, l) - __builtin_amdgcn_readlane(cnt, l));
      u.r = b + l;
      u.rt = by_parts ? k / u.ns : k;
      u.part = by_parts ? k - u.rt * u.ns : 0;
      u.q0 = __builtin_amdgcn_readlane(x.q0, l);
      u.n = __builtin_amdgcn_readlane(x.n, l);
      u.len = __builtin_amdgcn_readlane(x.len, l);
      u.slot = (int)slots + __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(split, l) + u.rt * u.ns;
      return true;
    }
    seen += __builtin_amdgcn_readlane(c, 63);
    slots += __builtin_amdgcn_readlane(s, 63);
  }
  return false;
}

// ------------------------------------------------------------------------------------------------------------ one key tile
// Query fragments of one row: step 2 t + e covers dims 32 t + 16 hi + 8 e .. + 7, the order in which a lane's 16 key bytes lie.
template <int D, int NS>
struct Query {
  frag8_t f[NS][D / 16];
  float mul;               // scores' factor: softmax scale * log2 e / row's power of two
};

template <int D, int NS>
__device__ __forceinline__ void load_query(Query<D, NS>& q, const void* p, long at, int type, bool on, int hi, float scale) {
  float x[D / 32][16];
  float mx = 0.f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      x[t][e] = on ? load1(p, at + 32 * t + 16 * hi + e, type) : 0.f;
      mx = fmaxf(mx, fabsf(x[t][e]));
    }
  float lo, up;
  xor32_pair(mx, lo, up);
  mx = fmaxf(lo, up);
  // 2^(14 - exponent of the largest element), within fp32; rows of infinities are left as they are
  int e = 268 - (int)(__float_as_uint(mx) >> 23);
  e = e > 254 ? 254 : e;
  if (type == FP16) e = 127;               // exact as it is
  const float f = __uint_as_float((unsigned)e << 23);
  q.mul = scale * LOG2E * __uint_as_float((unsigned)(254 - e) << 23);
  if (e == 254) q.mul = scale * LOG2E * 5.877471754e-39f;      // 2^-127
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      frag8_t h, l;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = x[t][8 * s + k] * f;
        h[k] = (_Float16)y;
        l[k] = (_Float16)(y - (float)h[k]);
      }
      q.f[0][2 * t + s] = h;
      if constexpr (NS == 2) q.f[NS - 1][2 * t + s] = l;
    }
}

template <int D>
struct Acc {
  f32x16_t o[D / 32];
  float m, l;
};

template <int D>
__device__ __forceinline__ void clear(Acc<D>& c) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) c.o[d][r] = 0.f;
  c.m = LOWEST;
  c.l = 0.f;
}

// tokens tok0 .. tok0 + 31 against this lane's row, which sees tokens < lim; kf(step), vf(dim tile, step) give the fragments
template <int D, int NS, class KF, class VF>
__device__ __forceinline__ void tile(Acc<D>& c, const Query<D, NS>& q, int tok0, int lim, float ks, float lvs, float ivs, int hi, bool masked,
                                     KF kf, VF vf) {
  f32x16_t s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
    const frag8_t k = kf(t);
    if constexpr (NS == 2) s = RMEM_MFMA(k, q.f[NS - 1][t], s);
    s = RMEM_MFMA(k, q.f[0][t], s);
  }
  const float mul = q.mul * ks;
  float top;
  const int left = lim - tok0 - 4 * hi;      // register r holds token tok0 + 4 hi + (r & 3) + 8 (r >> 2)
  if (!masked) {
    top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaf(top, mul, lvs);
  } else {
    top = LOWEST;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, (r & 3) + 8 * (r >> 2) < left ? fmaf(s[r], mul, lvs) : LOWEST);
  }
  float lo, up;
  xor32_pair(top, lo, up);
  const float m = fmaxf(c.m, fmaxf(lo, up));
  const float add = lvs - m + LIFT;
  float w[16], sum = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, add));
    if (masked) w[r] = (r & 3) + 8 * (r >> 2) < left ? w[r] : 0.f;
    sum += w[r];
  }
  xor32_pair(sum, lo, up);
  sum = (lo + up) * ivs;
  if (__any(m != c.m)) {
    const float alpha = __builtin_amdgcn_exp2f(c.m - m);
    c.l *= alpha;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) c.o[d][r] *= alpha;
    c.m = m;
  }
  c.l += sum;
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    frag8_t p, pl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = (_Float16)w[8 * st + e];
      if constexpr (NS == 2) pl[e] = (_Float16)(w[8 * st + e] - (float)p[e]);
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const frag8_t v = vf(d, st);
      if constexpr (NS == 2) c.o[d] = RMEM_MFMA(v, pl, c.o[d]);
      c.o[d] = RMEM_MFMA(v, p, c.o[d]);
    }
  }
}

// e4m3 bytes behind the request's last token may be NaN, and 0 * NaN is not 0: words m of a lane's 16 value bytes hold tokens
// 8 m + 4 hi .. + 3 of the tile
__device__ __forceinline__ u32x4_t keep_first(u32x4_t v, int valid, int hi) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int n = valid - 8 * m - 4 * hi;
    v[m] = n >= 4 ? v[m] : n <= 0 ? 0u : v[m] & ((1u << (8 * n)) - 1u);
  }
  return v;
}

__device__ __forceinline__ float readlane(float x, int l) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
}

// ------------------------------------------------------------------------------------------------------------ result rows
__device__ __forceinline__ void store4(void* p, long at, float a, float b, float c, float d, int type, bool wide) {
  if (!wide) {
    store1(p, at, a, type);
    store1(p, at + 1, b, type);
    store1(p, at + 2, c, type);
    store1(p, at + 3, d, type);
  } else if (type == FP32) {
    const f32x4_t w = {a, b, c, d};
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(p) + at) = w;
  } else if (type == FP16) {
    typedef __attribute__((ext_vector_type(4))) _Float16 h4;
    const h4 w = {(_Float16)a, (_Float16)b, (_Float16)c, (_Float16)d};
    *reinterpret_cast<h4*>(static_cast<_Float16*>(p) + at) = w;
  } else {
    typedef __attribute__((ext_vector_type(4))) __bf16 b4;
    const b4 w = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    *reinterpret_cast<b4*>(static_cast<__bf16*>(p) + at) = w;
  }
}

__device__ __forceinline__ bool wide_stores(const rmem_bank8_attn_args& a) {
  const long es = a.type == FP32 ? 4 : 2;
  return (((unsigned long)a.out | (unsigned long)(a.o_row * es) | (unsigned long)(a.o_head * es)) & (4 * es - 1)) == 0;
}

// a lane's share of its row: registers 4 k .. 4 k + 3 of tile d are dims 32 d + 8 k + 4 hi .. + 3
template <int D>
__device__ __forceinline__ void write_row(const rmem_bank8_attn_args& a, const Acc<D>& c, int hq, long row, int hi) {
  const float inv = c.l > 0.f ? 1.0f / c.l : c.l != c.l ? c.l : 0.f;
  const bool wide = wide_stores(a);
  const long at = row * a.o_row + hq * a.o_head;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      store4(a.out, at + 32 * d + 8 * k + 4 * hi, c.o[d][4 * k] * inv, c.o[d][4 * k + 1] * inv, c.o[d][4 * k + 2] * inv, c.o[d][4 * k + 3] * inv,
             a.type, wide);
  if (a.lse && hi == 0) a.lse[row * a.heads_q + hq] = (__log2f(c.l) + c.m - LIFT) * LN2;
}

// partial results of split units: [slot][kv head][ROWS][D] fp32, then [slot][kv head][ROWS][2] (maximum, sum)
struct Parts {
  float* o;
  float* ml;
  int slots;              // units that fit
};

template <int D, int ROWS>
__device__ __forceinline__ void write_part(const Parts& w, const Acc<D>& c, int slot, int h, int heads, int j, int hi) {
  const long row = ((long)slot * heads + h) * ROWS + j;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4_t x = {c.o[d][4 * k], c.o[d][4 * k + 1], c.o[d][4 * k + 2], c.o[d][4 * k + 3]};
      *reinterpret_cast<f32x4_t*>(w.o + row * D + 32 * d + 8 * k + 4 * hi) = x;
    }
  if (hi == 0) {
    w.ml[row * 2] = c.m;
    w.ml[row * 2 + 1] = c.l;
  }
}

// ------------------------------------------------------------------------------------------------------- few rows per head
// Four waves share a unit of 32 rows: wave w takes token tiles w, w + 4, ..., straight from memory into operand registers, the
// next tile's loads in flight behind the present one's arithmetic; the four partial results are joined through LDS.
// Page ids and scales of a wave's next 64 tiles sit one per lane.
template <int D, int CODE, int NS>
__global__ __launch_bounds__(256, 2) void attn_narrow(rmem_bank8_attn_args a, Parts parts, int G, int ps, int want, int chunk_min) {
  constexpr int DT = D / 32;
  __shared__ __attribute__((aligned(16))) f32x4_t s_o[2][DT * 4][64];
  __shared__ float s_m[4][64], s_l[4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hi = lane >> 5, j = lane & 31;
  const int heads = a.bank.heads, h = blockIdx.x % heads;
  Unit u;
  if (!find_unit<32>(a, G, blockIdx.x / heads, true, want, chunk_min, u)) return;
  const int row = u.rt * 32 + j, qt = row / G, hq = h * G + row % G;
  const bool on = qt < u.n;
  const int lim = !on ? 0 : a.causal ? min(u.len, u.len - u.n + qt + 1) : u.len;     // may be <= 0
  // tokens that the tile's last row sees, and this part of them
  const int last = min(u.n - 1, (u.rt * 32 + 31) / G);
  const int sees = max(0, a.causal ? u.len - u.n + last + 1 : u.len);
  const int first = max(0, a.causal ? u.len - u.n + u.rt * 32 / G + 1 : u.len);     // seen by every row of the tile
  const int tiles = (sees + 31) >> 5, per = (tiles + u.ns - 1) / u.ns;
  const int t0 = u.part * per, t1 = min(tiles, t0 + per);

  Query<D, NS> q;
  load_query<D, NS>(q, a.q, (long)(u.q0 + qt) * a.q_row + (long)hq * a.q_head, a.type, on, hi, a.scale);

  const int page = a.bank.page;
  const long block = (long)page * D;        // bytes of one (page, head)
  const int32_t* table = a.table + (long)u.r * a.ld_table;
  const uint8_t* kb = a.bank.k + h * block;
  const uint8_t* vb = a.bank.v + h * block;
  const long pstride = heads * block;
  const unsigned koff = (unsigned)(hi * page + j) * 16u, kstep = (unsigned)page * 32u, voff = (unsigned)(hi * D + j) * 16u;
  const int sub_mask = (1 << (ps - 5)) - 1;

  Acc<D> c;
  clear(c);
  for (int base = t0 + wave; base < t1; base += 256) {
    const int nt = min(64, (t1 - base + 3) >> 2);
    int pid = -1;
    float ks = 0.f, vs = 1.f;
    if (lane < nt) {
      const int id = table[(base + 4 * lane) >> (ps - 5)];
      if (id >= 0 && id < a.bank.pages) {
        pid = id;
        ks = a.bank.k_scale[(long)id * heads + h];
        vs = fmaxf(a.bank.v_scale[(long)id * heads + h], VS_MIN);
      }
    }
    const float lvs = __log2f(vs), ivs = 1.0f / vs;
    u32x4_t kr[2][DT], vr[2][DT];
    auto load = [&](int i, u32x4_t* k, u32x4_t* v) __attribute__((always_inline)) {
      const int id = __builtin_amdgcn_readlane(pid, i), sub = (base + 4 * i) & sub_mask;
      const long at = (id < 0 ? 0 : id) * pstride;
      const uint8_t* kp = kb + at + (unsigned)sub * 512u;
      const uint8_t* vp = vb + at + (unsigned)sub * (32u * D);
#pragma unroll
      for (int t = 0; t < DT; ++t) k[t] = *reinterpret_cast<const u32x4_t*>(kp + koff + t * kstep);
#pragma unroll
      for (int t = 0; t < DT; ++t) v[t] = *reinterpret_cast<const u32x4_t*>(vp + voff + t * 512u);
    };
    auto step = [&](int i, u32x4_t* k, u32x4_t* v) __attribute__((always_inline)) {
      const int tok0 = (base + 4 * i) * 32;
      const bool absent = __builtin_amdgcn_readlane(pid, i) < 0;
      const int end = absent ? tok0 : u.len;
      if (CODE == E4M3 && tok0 + 32 > end) {
#pragma unroll
        for (int t = 0; t < DT; ++t) v[t] = keep_first(v[t], end - tok0, hi);
      }
      tile<D, NS>(c, q, tok0, min(lim, end), readlane(ks, i), readlane(lvs, i), readlane(ivs, i), hi, tok0 + 32 > min(first, end),
                  [&](int t) { return decode8<CODE>(k[t >> 1][2 * (t & 1)], k[t >> 1][2 * (t & 1) + 1]); },
                  [&](int d, int st) { return decode8<CODE>(v[d][2 * st], v[d][2 * st + 1]); });
    };
    load(0, kr[0], vr[0]);
    for (int i = 0; i < nt; i += 2) {
      if (i + 1 < nt) load(i + 1, kr[1], vr[1]);
      step(i, kr[0], vr[0]);
      if (i + 1 >= nt) break;
      if (i + 2 < nt) load(i + 2, kr[0], vr[0]);
      step(i + 1, kr[1], vr[1]);
    }
  }

  // join the four waves
  s_m[wave][lane] = c.m;
  s_l[wave][lane] = c.l;
  __syncthreads();
  const float m = fmaxf(fmaxf(s_m[0][lane], s_m[1][lane]), fmaxf(s_m[2][lane], s_m[3][lane]));
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) l += s_l[w][lane] * __builtin_amdgcn_exp2f(s_m[w][lane] - m);
  const float alpha = __builtin_amdgcn_exp2f(c.m - m);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) c.o[d][r] *= alpha;
  c.m = m;
  c.l = l;
  auto put = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4_t x = {c.o[d][4 * k], c.o[d][4 * k + 1], c.o[d][4 * k + 2], c.o[d][4 * k + 3]};
        s_o[to][d * 4 + k][lane] = x;
      }
  };
  auto get = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4_t x = s_o[from][d * 4 + k][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) c.o[d][4 * k + e] += x[e];
      }
  };
  if (wave >= 2) put(wave - 2);
  __syncthreads();
  if (wave < 2) get(wave);
  __syncthreads();
  if (wave == 1) put(0);
  __syncthreads();
  if (wave != 0) return;
  get(0);
  if (!on) return;
  if (u.ns == 1) write_row<D>(a, c, hq, u.q0 + qt, hi);
  else if (u.slot + u.part < parts.slots) write_part<D, 32>(parts, c, u.slot + u.part, h, heads, j, hi);
}

// ------------------------------------------------------------------------------------------------------------------- merge
// One workgroup per (row tile of a split request, kv head, row): the parts of a row in order, D / 4 threads per part.
template <int ROWS>
__global__ __launch_bounds__(256) void attn_merge(rmem_bank8_attn_args a, Parts parts, int G, int want, int chunk_min) {
  __shared__ f32x4_t s_o[256];
  const int D = a.bank.dim, heads = a.bank.heads, tid = threadIdx.x;
  const int h = blockIdx.x % heads, j = blockIdx.y;
  Unit u;
  if (!find_unit<ROWS>(a, G, blockIdx.x / heads, false, want, chunk_min, u)) return;
  const int row = u.rt * ROWS + j, qt = row / G, hq = h * G + row % G;
  if (qt >= u.n || u.slot + u.ns > parts.slots) return;
  const long first = ((long)u.slot * heads + h) * ROWS + j, step = (long)heads * ROWS;
  float m = LOWEST;
  for (int p = tid & 63; p < u.ns; p += 64) m = fmaxf(m, parts.ml[(first + p * step) * 2]);
  m = wave_max_xor(m);
  const int width = D / 4, groups = 256 / width, g = tid / width, d4 = tid % width;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int p = g; p < u.ns; p += groups) {
    const long at = first + p * step;
    const float f = __builtin_amdgcn_exp2f(parts.ml[at * 2] - m);
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(parts.o + at * D + d4 * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    l = fmaf(parts.ml[at * 2 + 1], f, l);
  }
  __shared__ float s_l[32];
  s_o[tid] = o;
  if (d4 == 0) s_l[g] = l;
  __syncthreads();
  if (g) return;
  for (int k = 1; k < groups; ++k) {
    const f32x4_t x = s_o[k * width + d4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e];
    l += s_l[k];
  }
  const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
  const long out = (u.q0 + qt) * a.o_row + hq * a.o_head;
  store4(a.out, out + d4 * 4, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, a.type, wide_stores(a));
  if (a.lse && d4 == 0) a.lse[(u.q0 + qt) * (long)a.heads_q + hq] = (__log2f(l) + m - LIFT) * LN2;
}

// -------------------------------------------------------------------------------------------------------------------- host
constexpr int NARROW_UNITS = 2048;      // parts of all kv heads that a read is divided into
constexpr int NARROW_CHUNK = 16;        // fewest 32-token tiles worth a part

struct Plan {
  int G, ps, want;
  long units, slots;      // per kv head: grid bound, partial results' bound
};

bool valid_attn(const rmem_bank8_attn_args* a) {
  if (!a || !valid_bank(&a->bank) || !valid_type(a->type) || a->reqs <= 0 || a->rows < 0 || a->cols <= 0 || a->ld_table < a->cols ||
      (int64_t)a->cols * a->bank.page > 0x7fffffff || a->heads_q <= 0 || a->heads_q % a->bank.heads || !(a->scale > 0.f) ||
      !(a->scale < 3.0e38f))
    return false;
  return (int64_t)a->rows * (a->heads_q / a->bank.heads) <= 0x7fffffff;
}

Plan make_plan(const rmem_bank8_attn_args* a) {
  Plan p;
  p.G = a->heads_q / a->bank.heads;
  p.ps = log2_of(a->bank.page);
  p.want = NARROW_UNITS / a->bank.heads;
  if (p.want < 1) p.want = 1;
  const long row_tiles = ((long)a->rows * p.G) / 32 + (a->reqs < a->rows ? a->reqs : a->rows);
  // parts: at most total / chunk + one per row tile; of requests in several parts, at most twice total / chunk
  p.units = p.want + row_tiles;
  p.slots = 2L * p.want;
  return p;
}

long part_bytes(const rmem_bank8_attn_args* a, const Plan& p) {
  return p.slots * a->bank.heads * 32 * (a->bank.dim + 2) * 4;
}

template <int D, int CODE>
void launch_narrow(const rmem_bank8_attn_args& a, const Parts& parts, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.units * a.bank.heads));
  if (a.type == FP32) hipLaunchKernelGGL((attn_narrow<D, CODE, 2>), grid, dim3(256), 0, s, a, parts, p.G, p.ps, p.want, NARROW_CHUNK);
  else hipLaunchKernelGGL((attn_narrow<D, CODE, 1>), grid, dim3(256), 0, s, a, parts, p.G, p.ps, p.want, NARROW_CHUNK);
}

}  // namespace

extern "C" int64_t rmem_bank8_attn_workspace(const rmem_bank8_attn_args* a) {
  if (!valid_attn(a)) return -1;
  return part_bytes(a, make_plan(a));
}

extern "C" int rmem_bank8_attn(const rmem_bank8_attn_args* a, void* stream) {
  if (!valid_attn(a)) return RMEM_ERR_INVALID;
  if (a->rows == 0) return RMEM_OK;
  const Plan p = make_plan(a);
  if (!a->q || !a->out || !a->cu || !a->lens || !a->table || !a->workspace || ((uintptr_t)a->workspace % 16) ||
      a->workspace_bytes < part_bytes(a, p) || p.units * a->bank.heads >= 1 << 24)
    return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Parts parts;
  parts.o = static_cast<float*>(a->workspace);
  parts.ml = parts.o + p.slots * a->bank.heads * 32 * a->bank.dim;
  parts.slots = (int)p.slots;
  const bool e4m3 = a->bank.code == E4M3;
  switch (a->bank.dim) {
    case 32: e4m3 ? launch_narrow<32, E4M3>(*a, parts, p, s) : launch_narrow<32, INT8>(*a, parts, p, s); break;
    case 64: e4m3 ? launch_narrow<64, E4M3>(*a, parts, p, s) : launch_narrow<64, INT8>(*a, parts, p, s); break;
    default: e4m3 ? launch_narrow<128, E4M3>(*a, parts, p, s) : launch_narrow<128, INT8>(*a, parts, p, s); break;
  }
  RMEM_CHECK_LAUNCH();
  // a request whose row of the table holds no more than the smallest part is never divided
  if (((long)a->cols * a->bank.page + 31) / 32 > NARROW_CHUNK) {
    const long tiles = p.slots / 2;       // row tiles in at least two parts
    hipLaunchKernelGGL((attn_merge<32>), dim3((unsigned)(tiles * a->bank.heads), 32), dim3(256), 0, s, *a, parts, p.G, p.want, NARROW_CHUNK);
    RMEM_CHECK_LAUNCH();
  }
  return RMEM_OK;
}
