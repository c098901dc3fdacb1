// bank8_attn.hip -- attention of each request's rows over its pages of the 8-bit bank.
//
// Both products run "swapped" on v_mfma_f32_32x32x16_f16, as in mha.hip:
//   S^T[token][row] = K_tile . Q^T          O^T[dim][row] += V^T_tile . P^T
// so a row's softmax statistics live in one lane (and its lane^32 partner) and the accumulators of S^T are the B operand of the
// second product.  `row` is a (query token, query head of the group) pair: the heads that share a kv head share its tiles.
// Codes become fp16 exactly (8 bits fit into 11), so the key scale is applied to the scores, once per element beside the softmax
// scale, and the value scale rides in the exponent: w = 2^(y - m), y = scale log2e ks s + log2 vs, O = sum w code, and the
// denominator takes each tile's sum of weights times 1 / vs.  No dequantised value exists anywhere.
// Queries enter as fp16.  fp16 rows as they are; bf16 and fp32 rows times a power of two that puts the row's largest element between
// 2^14 and 2^15, where fp16's smallest step, 2^-24, is 2^-38 of 2^14: bf16 elements (8 bits) are exact down to 2^-31 of the largest
// and below that off by at most half a step, 2^-39 of it; fp32 elements go into two planes (NS = 2: two products against the same
// codes) and are off by at most 2^-22 of themselves or those 2^-39 of the row's largest, whichever is more.
// Weights are 2^10 times their usual size (2^10 at the row's reference, not 1), which leaves 24 instead of 14 binades of normal
// fp16 numbers below it; fp32 calls keep them in two planes.  Sums are fp32, of the unrounded weights.
#include "bank8.h"

#include <algorithm>
#include <type_traits>

using namespace bank8;

#define MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0)

namespace {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float LIFT = 10.f;             // log2 of a weight at the row's reference
constexpr float SLACK = 5.f;             // how far the maximum may get ahead of it
constexpr float LOWEST = -3.0e38f;       // running maximum of a row that has seen nothing
constexpr float VS_MIN = 3.23117427e-27f;    // 2^-88: 1 / vs times 2^15 times 2^24 tokens stays finite

// ---------------------------------------------------------------------------------------------------- division into units
// A unit of work is (request, tile of ROWS rows, one of ns equal parts of the tokens that the tile sees) for one kv head.  Every
// part has at most `chunk` 32-token tiles, chunk = (all row tiles' token tiles) / want, so the parts of long and short requests
// cost the same and nothing is decided on the host, which does not know the lengths.  Each wave computes the same division from
// cu and lens, a request per lane.
struct Unit {
  int r, rt, part, ns;    // request, row tile, part of ns
  int q0, n, len;         // first row, rows, tokens
  int slot, ord;          // of a row tile in several parts: index of part 0's partial result, index among such tiles
};

struct Req {
  int q0, n, len, rt, tiles;
};

// How a read is divided: `want` parts per kv head, none of fewer than `chunk_min` tiles, over the requests of `lo` .. `hi` rows per
// kv head (a call may give short and long requests to different kernels).
struct Split {
  int G, ps, want, chunk_min;
  int lo, hi;
};

template <int ROWS>
__device__ __forceinline__ Req request(const rmem_bank8_attn_args& a, int r, const Split& sp) {
  Req x = {0, 0, 0, 0, 0};
  if (r >= a.reqs) return x;
  int q0 = a.cu[r], q1 = a.cu[r + 1], len = a.lens[r];
  q0 = q0 < 0 ? 0 : q0 > a.rows ? a.rows : q0;
  q1 = q1 < q0 ? q0 : q1 > a.rows ? a.rows : q1;
  const long cap = (long)a.cols * a.bank.page;
  x.q0 = q0;
  x.n = q1 - q0;
  x.len = len < 0 ? 0 : len > cap ? (int)cap : len;
  const long rows = (long)x.n * sp.G;
  x.rt = rows < sp.lo || rows > sp.hi ? 0 : (int)((rows + ROWS - 1) / ROWS);
  x.tiles = (x.len + 31) >> 5;
  return x;
}

// Inclusive sums over the lanes in six DPP additions (shifts by 1, 2, 4, 8 within rows of 16, then the rows' last lanes): the same by
// __shfl_up is six LDS round trips, and every workgroup begins with it.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);       // lane 15 of rows 0 and 2 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);       // lane 31 to rows 2 and 3
  return v;
}
// sum over the lanes; exact below 2^53, and the same everywhere
__device__ __forceinline__ long wave_sum_long(long v) { return (long)wave_sum_xor_t<32>((double)v); }

// tiles of a part (up to 64 requests, one per lane)
__device__ __forceinline__ int chunk_of(const Req& x, const Split& sp) {
  const long total = (wave_sum_long((long)x.rt * x.tiles) + sp.want - 1) / sp.want;
  return total < sp.chunk_min ? sp.chunk_min : total > 0x3fffffff ? 0x3fffffff : (int)total;
}

// With more requests than lanes the division is computed once, by a launch of its own (index_kernel), and looked up: what lies in
// front of each request, and last the totals.  (Requests of one row and up to 1000 tokens, 64 at a time scanned by every workgroup:
// 1000 of them 280 us, looked up 175 us; 200 of up to 4000 tokens 100 and 98.)
struct Before {
  int units, slots, ords, chunk;
};

template <int ROWS>
__device__ __forceinline__ bool look_up(const rmem_bank8_attn_args& a, const Split& sp, const Before* index, long at, Unit& u) {
  const int lane = threadIdx.x & 63;
  if (at >= index[a.reqs].units) return false;
  int lo = 0, len = a.reqs;                    // the last request with no more than `at` units in front of it, 64 places at a time
  while (len > 1) {
    const int step = (len + 63) >> 6, r = lo + lane * step;
    const bool le = lane * step < len && index[r].units <= at;
    const int n = __popcll(__ballot(le));
    lo += (n - 1) * step;
    len = min(step, len - (n - 1) * step);
  }
  const Before b = index[lo];
  const Req x = request<ROWS>(a, lo, sp);
  const int k = (int)(at - b.units);
  u.ns = x.tiles > b.chunk ? (x.tiles + b.chunk - 1) / b.chunk : 1;
  u.r = lo;
  u.rt = x.rt - 1 - k / u.ns;
  u.part = k % u.ns;
  u.q0 = x.q0;
  u.n = x.n;
  u.len = x.len;
  u.slot = b.slots + u.rt * u.ns;
  u.ord = b.ords + u.rt;
  return k >= 0 && u.rt >= 0;                  // (sums that row offsets which are none have wrapped)
}

template <int ROWS>
__global__ __launch_bounds__(1024) void index_kernel(rmem_bank8_attn_args a, Split sp, Before* index) {
  __shared__ double s_sum[16];
  __shared__ int s_part[3][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  double total = 0;
  for (int r = tid; r < a.reqs; r += 1024) {
    const Req x = request<ROWS>(a, r, sp);
    total += (double)x.rt * x.tiles;
  }
  total = wave_sum_xor_t<32>(total);
  if (lane == 0) s_sum[wave] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < 16; ++w) total += s_sum[w];
  const long even = ((long)total + sp.want - 1) / sp.want;
  const int chunk = even < sp.chunk_min ? sp.chunk_min : even > 0x3fffffff ? 0x3fffffff : (int)even;
  int seen[3] = {0, 0, 0};
  for (int base = 0; base < a.reqs; base += 1024) {
    const Req x = request<ROWS>(a, base + tid, sp);
    const int ns = x.tiles > chunk ? (x.tiles + chunk - 1) / chunk : 1;
    const int own[3] = {x.rt * ns, ns > 1 ? x.rt * ns : 0, ns > 1 ? x.rt : 0};
    int sum[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sum[i] = wave_scan(own[i]);
      if (lane == 63) s_part[i][wave] = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      int front = seen[i];
      for (int w = 0; w < 16; ++w) {
        const int p = s_part[i][w];
        if (w < wave) front += p;
        seen[i] += p;
      }
      sum[i] += front - own[i];
    }
    if (base + tid < a.reqs) {
      const Before b = {sum[0], sum[1], sum[2], chunk};
      index[base + tid] = b;
    }
    __syncthreads();
  }
  if (tid == 0) {
    const Before b = {seen[0], seen[1], seen[2], chunk};
    index[a.reqs] = b;
  }
}

template <int ROWS>
__device__ bool find_unit(const rmem_bank8_attn_args& a, const Split& sp, const Before* before, long index, Unit& u) {
  if (before) return look_up<ROWS>(a, sp, before, index, u);
  const int lane = threadIdx.x & 63;
  const Req x = request<ROWS>(a, lane, sp);
  const int chunk = chunk_of(x, sp);
  const int ns = x.tiles > chunk ? (x.tiles + chunk - 1) / chunk : 1;
  const int cnt = x.rt * ns, split = ns > 1 ? cnt : 0, ord = ns > 1 ? x.rt : 0;
  const int c = wave_scan(cnt), s = wave_scan(split), o = wave_scan(ord);
  const unsigned long long hit = __ballot(index < c);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit);
  u.ns = __builtin_amdgcn_readlane(ns, l);
  const int k = (int)index - (__builtin_amdgcn_readlane(c, l) - __builtin_amdgcn_readlane(cnt, l));
  u.r = l;
  u.rt = __builtin_amdgcn_readlane(x.rt, l) - 1 - k / u.ns;      // the last row tile first: under a causal mask it sees most
  u.part = k % u.ns;
  u.q0 = __builtin_amdgcn_readlane(x.q0, l);
  u.n = __builtin_amdgcn_readlane(x.n, l);
  u.len = __builtin_amdgcn_readlane(x.len, l);
  u.slot = __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(split, l) + u.rt * u.ns;
  u.ord = __builtin_amdgcn_readlane(o, l) - __builtin_amdgcn_readlane(ord, l) + u.rt;
  return k >= 0 && u.rt >= 0;
}

// row tiles in several parts
template <int ROWS>
__device__ __forceinline__ long count_split(const rmem_bank8_attn_args& a, const Split& sp, const Before* before) {
  if (before) return before[a.reqs].ords;
  const Req x = request<ROWS>(a, threadIdx.x & 63, sp);
  const int chunk = chunk_of(x, sp);
  return wave_sum_long(x.tiles > chunk ? x.rt : 0);
}

// ---------------------------------------------------------------------------------------------------------- one token tile
// Two shapes of the matrix instruction, by the rows of a tile (R).  `g` = lane / R is the lane's part of what its row's lanes share.
//   R = 32 (32x32x16): S^T of 32 tokens in one product chain; lane (row, g) holds tokens (r & 3) + 8 (r >> 2) + 4 g in register r
//   R = 16 (16x16x32): two chains of 16 tokens each; lane (row, g) holds tokens 16 (g & 1) + 4 (g >> 1) + (r & 3) + 8 (r >> 2),
//          r = 0 .. 7: a group of up to 16 query heads on one token needs half the softmax arithmetic and half the registers
// In both a lane's values in V^T's byte order are its P operand.
template <int R>
__device__ __forceinline__ float row_max(float x) {
  float lo, up;
  xor32_pair(x, lo, up);
  x = fmaxf(lo, up);
  if constexpr (R == 16) {
    xor16_pair(x, lo, up);
    x = fmaxf(lo, up);
  }
  return x;
}
template <int R>
__device__ __forceinline__ float row_sum(float x) {
  float lo, up;
  xor32_pair(x, lo, up);
  x = lo + up;
  if constexpr (R == 16) {
    xor16_pair(x, lo, up);
    x = lo + up;
  }
  return x;
}

// Query fragments of one row.  A lane's 16 key bytes are 16 consecutive dims: chunk C t + g of 16 (C = 64 / R lanes per row), the
// first 8 for step 2 t, the others for step 2 t + 1; with R = 16 and 32 dims a lane has 8 bytes, dims 8 g .. + 7, and one step.
template <int R, int D, int NS>
struct Query {
  static constexpr int STEPS = R == 32 ? D / 16 : D / 32;
  frag8_t f[NS][STEPS];
  float mul;               // scores' factor: softmax scale * log2 e / row's power of two
};

template <int R, int D>
__device__ __forceinline__ int step_dim(int step, int g) {
  if (R == 16 && D == 32) return 8 * g;
  return ((64 / R) * (step >> 1) + g) * 16 + 8 * (step & 1);
}

// one branch on type and alignment around all of a lane's loads: a branch per element makes each wait for the one before
template <int R, int D, int S, class T>
__device__ __forceinline__ void load_row(float (&x)[S][8], const T* p, int g, bool wide) {
  typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T vec_t;
  constexpr int V = 16 / sizeof(T);
  if (wide) {
    vec_t y[S][8 / V];
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
      for (int k = 0; k < 8 / V; ++k) y[t][k] = *reinterpret_cast<const vec_t*>(p + step_dim<R, D>(t, g) + k * V);
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[t][e] = (float)y[t][e / V][e % V];
  } else {
    T y[S][8];
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[t][e] = p[step_dim<R, D>(t, g) + e];
#pragma unroll
    for (int t = 0; t < S; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[t][e] = (float)y[t][e];
  }
}

template <int R, int D, int NS>
__device__ __forceinline__ void load_query(Query<R, D, NS>& q, const rmem_bank8_attn_args& a, long row, int hq, bool on, int g) {
  constexpr int S = Query<R, D, NS>::STEPS;
  const int type = a.type;
  const float scale = a.scale;
  const long at = row * a.q_row + hq * a.q_head, es = type == FP32 ? 4 : 2;
  const bool wide = (((unsigned long)a.q | (unsigned long)(a.q_row * es) | (unsigned long)(a.q_head * es)) & 15) == 0;
  float x[S][8];
#pragma unroll
  for (int t = 0; t < S; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[t][e] = 0.f;
  if (on) {
    if constexpr (NS == 2) load_row<R, D>(x, static_cast<const float*>(a.q) + at, g, wide);
    else if (type == FP16) load_row<R, D>(x, static_cast<const _Float16*>(a.q) + at, g, wide);
    else load_row<R, D>(x, static_cast<const __bf16*>(a.q) + at, g, wide);
  }
  float mx = 0.f;
#pragma unroll
  for (int t = 0; t < S; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[t][e]));
  mx = row_max<R>(mx);
  // 2^(14 - exponent of the largest element), within fp32; rows of infinities are left as they are
  int e = 268 - (int)(__float_as_uint(mx) >> 23);
  e = e > 254 ? 254 : e;
  if (type == FP16) e = 127;               // exact as it is
  const float f = __uint_as_float((unsigned)e << 23);
  q.mul = scale * LOG2E * __uint_as_float((unsigned)(254 - e) << 23);
  if (e == 254) q.mul = scale * LOG2E * 5.877471754e-39f;      // 2^-127
#pragma unroll
  for (int t = 0; t < S; ++t) {
    frag8_t h, l;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float y = x[t][k] * f;
      h[k] = (_Float16)y;
      l[k] = (_Float16)(y - (float)h[k]);
    }
    q.f[0][t] = h;
    if constexpr (NS == 2) q.f[NS - 1][t] = l;
  }
}

// O^T of the lane's row, four consecutive dims at a time: quad i holds dims (256 / R) i + 4 g .. + 3
template <int R, int D>
struct Acc {
  static constexpr int QUADS = D * R / 256, STRIDE = 256 / R;
  typedef typename std::conditional<R == 32, f32x16_t, f32x4_t>::type tile_t;
  tile_t o[D / R];
  float m, l;
  __device__ __forceinline__ f32x4_t quad(int i) const {
    if constexpr (R == 16) return o[i];
    else {
      const f32x4_t x = {o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]};
      return x;
    }
  }
  __device__ __forceinline__ void add(int i, f32x4_t x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (R == 16) o[i][e] += x[e];
      else o[i >> 2][4 * (i & 3) + e] += x[e];
    }
  }
  __device__ __forceinline__ void mul(float f) {
#pragma unroll
    for (int d = 0; d < D / R; ++d)
#pragma unroll
      for (int r = 0; r < R / 2 * (R == 32) + 4 * (R == 16); ++r) o[d][r] *= f;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < D / R; ++d)
#pragma unroll
      for (int r = 0; r < R / 2 * (R == 32) + 4 * (R == 16); ++r) o[d][r] = 0.f;
    m = LOWEST;
    l = 0.f;
  }
};

// T tiles of 32 tokens from tok0 on, against this lane's row, which sees the tokens below lim[t] of tile t; kf(t, step, chain) and
// vf(t, dim tile, step) give fragments.  One maximum and one look at the accumulators for all T: a row's reference m follows the
// maximum only when that gets SLACK ahead, because weights up to 2^(LIFT + SLACK) fit into fp16 -- after the first few tiles the
// accumulators are hardly ever scaled again.
template <int T, int R, int D, int NS, class KF, class VF>
__device__ __forceinline__ void attend_tiles(Acc<R, D>& c, const Query<R, D, NS>& q, int tok0, const int (&lim)[T], const float (&ks)[T],
                                      const float (&lvs)[T], const float (&ivs)[T], int g, bool masked, KF kf, VF vf) {
  constexpr int N = R / 2;                  // tokens per lane and tile
  float s[T][N];
#pragma unroll
  for (int i = 0; i < T; ++i) {
    if constexpr (R == 32) {
      f32x16_t x;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const frag8_t k = kf(i, t, 0);
        if constexpr (NS == 2) x = RMEM_MFMA(k, q.f[NS - 1][t], x);
        x = RMEM_MFMA(k, q.f[0][t], x);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] = x[r];
    } else {
      f32x4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const frag8_t f = kf(i, t, k);
          if constexpr (NS == 2) x[k] = MFMA16(f, q.f[NS - 1][t], x[k]);
          x[k] = MFMA16(f, q.f[0][t], x[k]);
        }
#pragma unroll
      for (int r = 0; r < 8; ++r) s[i][r] = x[r >> 2][r & 3];
    }
  }
  if (masked) {
    // register r holds token (r & 3) + 8 (r >> 2) of these; the pin keeps this a branch (as selects it costs every tile)
    int at = R == 32 ? 4 * g : 16 * (g & 1) + 4 * (g >> 1);
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int r = 0; r < N; ++r) s[i][r] = (r & 3) + 8 * (r >> 2) < lim[i] - tok0 - 32 * i - at ? s[i][r] : -INFINITY;
  }
  float mul[T], top = LOWEST;
#pragma unroll
  for (int i = 0; i < T; ++i) {
    mul[i] = fmaxf(q.mul * ks[i], 1.4e-45f);      // positive: times -infinity it stays that
    float x = s[i][0];
#pragma unroll
    for (int r = 1; r < N; ++r) x = fmaxf(x, s[i][r]);
    top = fmaxf(top, fmaf(x, mul[i], lvs[i]));
  }
  top = row_max<R>(top);
  if (__any(top > c.m + SLACK)) {
    const float m = top > c.m + SLACK ? top : c.m;
    const float alpha = __builtin_amdgcn_exp2f(c.m - m);
    c.l *= alpha;
    c.mul(alpha);
    c.m = m;
  }
#pragma unroll
  for (int i = 0; i < T; ++i) {
    const float add = lvs[i] - c.m + LIFT;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < N; ++r) {
      s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], mul[i], add));
      sum[r & 1] += s[i][r];
    }
    c.l = fmaf(sum[0] + sum[1], ivs[i], c.l);     // this lane's tokens; joined with its row's other lanes at the end
#pragma unroll
    for (int st = 0; st < N / 8; ++st) {
      frag8_t p, pl;
      if constexpr (NS == 2) {
        u32x4_t h, l;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t hh, ll;
          split_pair_f16(s[i][8 * st + 2 * e], s[i][8 * st + 2 * e + 1], hh, ll);
          h[e] = hh;
          l[e] = ll;
        }
        p = __builtin_bit_cast(frag8_t, h);
        pl = __builtin_bit_cast(frag8_t, l);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = (_Float16)s[i][8 * st + e];
      }
#pragma unroll
      for (int d = 0; d < D / R; ++d) {
        const frag8_t v = vf(i, d, st);
        if constexpr (R == 32) {
          if constexpr (NS == 2) c.o[d] = RMEM_MFMA(v, pl, c.o[d]);
          c.o[d] = RMEM_MFMA(v, p, c.o[d]);
        } else {
          if constexpr (NS == 2) c.o[d] = MFMA16(v, pl, c.o[d]);
          c.o[d] = MFMA16(v, p, c.o[d]);
        }
      }
    }
  }
}

// the first n of a word's four bytes
__device__ __forceinline__ uint32_t keep_first(uint32_t v, int n) { return n >= 4 ? v : n <= 0 ? 0u : v & ((1u << (8 * n)) - 1u); }

__device__ __forceinline__ float readlane(float x, int l) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
}

// ------------------------------------------------------------------------------------------------------------ result rows
template <class T>
__device__ __forceinline__ void store4(T* p, f32x4_t x, bool wide) {
  typedef __attribute__((ext_vector_type(4))) T vec_t;
  const vec_t w = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
  if (wide) *reinterpret_cast<vec_t*>(p) = w;
  else {
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = w[e];
  }
}
template <class F>
__device__ __forceinline__ void by_type(int type, void* p, F f) {
  if (type == FP32) f(static_cast<float*>(p));
  else if (type == FP16) f(static_cast<_Float16*>(p));
  else f(static_cast<__bf16*>(p));
}

__device__ __forceinline__ bool wide_stores(const rmem_bank8_attn_args& a) {
  const long es = a.type == FP32 ? 4 : 2;
  return (((unsigned long)a.out | (unsigned long)(a.o_row * es) | (unsigned long)(a.o_head * es)) & (4 * es - 1)) == 0;
}

template <int R, int D>
__device__ __forceinline__ void write_row(const rmem_bank8_attn_args& a, const Acc<R, D>& c, int hq, long row, int g) {
  const float inv = c.l > 0.f ? 1.0f / c.l : c.l != c.l ? c.l : 0.f;
  const bool wide = wide_stores(a);
  const long at = row * a.o_row + hq * a.o_head;
  by_type(a.type, a.out, [&](auto* p) {
#pragma unroll
    for (int i = 0; i < Acc<R, D>::QUADS; ++i) store4(p + at + Acc<R, D>::STRIDE * i + 4 * g, c.quad(i) * inv, wide);
  });
  if (a.lse && g == 0) a.lse[row * a.heads_q + hq] = (__log2f(c.l) + c.m - LIFT) * LN2;
}

// partial results of split units: [slot][kv head][ROWS][D] fp32, [slot][kv head][ROWS][2] (reference, sum), and for each row tile
// in several parts what the merge needs to know of it
struct Split_tile {
  int q0, n, rt, ns, slot, pad[3];
};
struct Parts {
  float* o;
  float* ml;
  Split_tile* tiles;
  const Before* before;   // the division, looked up (null: computed)
  int slots, ords;        // units and tiles that fit
};

template <int ROWS, int R, int D>
__device__ __forceinline__ void write_part(const Parts& w, const Acc<R, D>& c, const Unit& u, int h, int heads, int j, int g) {
  const int slot = u.slot + u.part;
  if (slot < 0 || slot >= w.slots) return;
  if (h == 0 && u.part == 0 && j == 0 && g == 0 && u.ord >= 0 && u.ord < w.ords) {
    const Split_tile t = {u.q0, u.n, u.rt, u.ns, u.slot, {0, 0, 0}};
    w.tiles[u.ord] = t;
  }
  const long row = ((long)slot * heads + h) * ROWS + j;
#pragma unroll
  for (int i = 0; i < Acc<R, D>::QUADS; ++i) *reinterpret_cast<f32x4_t*>(w.o + row * D + Acc<R, D>::STRIDE * i + 4 * g) = c.quad(i);
  if (g == 0) {
    w.ml[row * 2] = c.m;
    w.ml[row * 2 + 1] = c.l;
  }
}

// ------------------------------------------------------------------------------------------------------- few rows per head
// Four waves share a unit of R rows: wave w takes token tiles w, w + 4, ..., straight from memory into operand registers, the
// next tile's loads in flight behind the present one's arithmetic; the four partial results are joined through LDS.
// Page ids and scales of a wave's next 64 tiles sit one per lane.  Bound by the bytes: one row of 64 heads over 250 k tokens of 8 x 128,
// 512 MB, 92 us, 5.6 TB/s; 64 ragged rows of 32 heads, 451 MB, 91 us, 5.0 TB/s.  With 32 rows per tile the vector instructions bound
// it, since each wave decodes what it multiplies: 64 requests of 16 tokens and 4 x 8 heads over 4 k tokens 110 us, 610 TFLOP/s,
// vector pipe 66 % busy, matrix pipe 28 %.
template <int R, int D>
struct Raw;                               // a lane's codes of a tile
template <int D>
struct Raw<32, D> {
  u32x4_t k[D / 32], v[D / 32];
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int page, int j, int g) {
    const unsigned ko = (unsigned)(g * page + j) * 16u, vo = (unsigned)(g * D + j) * 16u;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) k[t] = *reinterpret_cast<const u32x4_t*>(kp + ko + (unsigned)(t * page) * 32u);
    asm volatile("" ::: "memory");          // keys are wanted first: loads return in the order of their issue
#pragma unroll
    for (int t = 0; t < D / 32; ++t) v[t] = *reinterpret_cast<const u32x4_t*>(vp + vo + t * 512u);
  }
  // e4m3 bytes behind the request's last token may be NaN, and 0 * NaN is not 0
  __device__ __forceinline__ void cut(int valid, int g) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) v[t][m] = keep_first(v[t][m], valid - 8 * m - 4 * g);
  }
  template <int CODE>
  __device__ __forceinline__ frag8_t kf(int t, int) const { return decode8<CODE>(k[t >> 1][2 * (t & 1)], k[t >> 1][2 * (t & 1) + 1]); }
  template <int CODE>
  __device__ __forceinline__ frag8_t vf(int d, int st) const { return decode8<CODE>(v[d][2 * st], v[d][2 * st + 1]); }
};
template <int D>
struct Raw<16, D> {
  static constexpr int KC = D == 32 ? 1 : D / 64;      // 16-byte (32 dims: 8-byte) loads per token
  u32x4_t k[2][KC];
  u32x2_t v[D / 16];
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int page, int j, int g) {
    const int tok = 4 * (j >> 3) + 16 * ((j >> 2) & 1) + (j & 3);    // of chain 0, row j of S^T; chain 1: 8 further on
    if constexpr (D == 32) {
      const unsigned ko = (unsigned)((g >> 1) * page + tok) * 16u + 8u * (g & 1);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const u32x2_t x = *reinterpret_cast<const u32x2_t*>(kp + ko + c * 128u);
        k[c][0][0] = x[0];
        k[c][0][1] = x[1];
      }
    } else {
      const unsigned ko = (unsigned)(g * page + tok) * 16u;
#pragma unroll
      for (int t = 0; t < KC; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) k[c][t] = *reinterpret_cast<const u32x4_t*>(kp + ko + (unsigned)(t * page) * 64u + c * 128u);
    }
    asm volatile("" ::: "memory");          // keys are wanted first: loads return in the order of their issue
    const unsigned vo = (unsigned)((g >> 1) * D + j) * 16u + 8u * (g & 1);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) v[d] = *reinterpret_cast<const u32x2_t*>(vp + vo + d * 256u);
  }
  __device__ __forceinline__ void cut(int valid, int g) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int m = 0; m < 2; ++m) v[d][m] = keep_first(v[d][m], valid - 8 * m - 16 * (g & 1) - 4 * (g >> 1));
  }
  template <int CODE>
  __device__ __forceinline__ frag8_t kf(int t, int c) const {
    if constexpr (D == 32) return decode8<CODE>(k[c][0][0], k[c][0][1]);
    else return decode8<CODE>(k[c][t >> 1][2 * (t & 1)], k[c][t >> 1][2 * (t & 1) + 1]);
  }
  template <int CODE>
  __device__ __forceinline__ frag8_t vf(int d, int) const { return decode8<CODE>(v[d][0], v[d][1]); }
};

// ROWS rows of a unit from first_row on: sees = tokens seen by some of them, all = by every one
struct Sees {
  int sees, all;
};
template <int ROWS>
__device__ __forceinline__ Sees rows_see(const Unit& u, int first_row, int causal, int G) {
  const int first = first_row / G, last = min(u.n - 1, (first_row + ROWS - 1) / G);
  Sees x;
  x.sees = first >= u.n ? 0 : max(0, causal ? u.len - u.n + last + 1 : u.len);
  x.all = max(0, causal ? u.len - u.n + first + 1 : u.len);
  return x;
}

template <int R, int D, int CODE, int NS>
__global__ __launch_bounds__(256, 2) void attn_narrow(rmem_bank8_attn_args a, Parts parts, Split sp) {
  const int G = sp.G, ps = sp.ps;
  constexpr int QUADS = Acc<R, D>::QUADS;
  __shared__ __attribute__((aligned(16))) f32x4_t s_o[2][QUADS][64];
  __shared__ float s_m[4][64], s_l[4][64];
  const int tid = threadIdx.x, lane = tid & 63, g = lane / R, j = lane % R;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);       // uniform: tile counts and page addresses stay scalar
  const int heads = a.bank.heads, h = blockIdx.x % heads;
  Unit u;
  if (!find_unit<R>(a, sp, parts.before, blockIdx.x / heads, u)) return;
  const int row = u.rt * R + j, qt = row / G, hq = h * G + row % G;
  const bool on = qt < u.n;
  const int lim = !on ? 0 : a.causal ? min(u.len, u.len - u.n + qt + 1) : u.len;     // may be <= 0
  const Sees see = rows_see<R>(u, u.rt * R, a.causal, G);
  const int tiles = (see.sees + 31) >> 5, per = (tiles + u.ns - 1) / u.ns;
  const int t0 = u.part * per, t1 = min(tiles, t0 + per);

  Query<R, D, NS> q;
  load_query<R, D, NS>(q, a, u.q0 + qt, hq, on, g);

  const int page = a.bank.page;
  const long block = (long)page * D;        // bytes of one (page, head)
  const int32_t* table = a.table + (long)u.r * a.ld_table;
  const uint8_t* kb = a.bank.k + h * block;
  const uint8_t* vb = a.bank.v + h * block;
  const long pstride = heads * block;
  const int sub_mask = (1 << (ps - 5)) - 1;

  Acc<R, D> c;
  c.clear();
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
    Raw<R, D> raw[2];
    auto load = [&](int i, Raw<R, D>& x) __attribute__((always_inline)) {
      const int id = __builtin_amdgcn_readlane(pid, i), sub = (base + 4 * i) & sub_mask;
      const long at = (id < 0 ? 0 : id) * pstride;
      x.load(kb + at + (unsigned)sub * 512u, vb + at + (unsigned)sub * (32u * D), page, j, g);
    };
    auto step = [&](int i, Raw<R, D>& x) __attribute__((always_inline)) {
      const int tok0 = (base + 4 * i) * 32;
      const bool absent = __builtin_amdgcn_readlane(pid, i) < 0;
      const int end = absent ? tok0 : u.len;
      if (CODE == E4M3 && tok0 + 32 > end) x.cut(end - tok0, g);
      const int lims[1] = {min(lim, end)};
      const float k1[1] = {readlane(ks, i)}, l1[1] = {readlane(lvs, i)}, i1[1] = {readlane(ivs, i)};
      attend_tiles<1, R, D, NS>(c, q, tok0, lims, k1, l1, i1, g, tok0 + 32 > min(see.all, end),
                         [&](int, int t, int k) { return x.template kf<CODE>(t, k); }, [&](int, int d, int st) { return x.template vf<CODE>(d, st); });
    };
    // The loads are unconditional (the last tile again where there is no next one): with a way around them the compiler would have
    // to wait for all that may be in flight before it touches the present tile.
    load(0, raw[0]);
    for (int i = 0;; i += 2) {
      load(min(i + 1, nt - 1), raw[1]);
      step(i, raw[0]);
      if (i + 1 >= nt) break;
      load(min(i + 2, nt - 1), raw[0]);
      step(i + 1, raw[1]);
      if (i + 2 >= nt) break;
    }
  }

  // join the lanes of a row, then the four waves
  c.l = row_sum<R>(c.l);
  s_m[wave][lane] = c.m;
  s_l[wave][lane] = c.l;
  __syncthreads();
  const float m = fmaxf(fmaxf(s_m[0][lane], s_m[1][lane]), fmaxf(s_m[2][lane], s_m[3][lane]));
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) l += s_l[w][lane] * __builtin_amdgcn_exp2f(s_m[w][lane] - m);
  c.mul(__builtin_amdgcn_exp2f(c.m - m));
  c.m = m;
  c.l = l;
  auto put = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) s_o[to][i][lane] = c.quad(i);
  };
  auto get = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QUADS; ++i) c.add(i, s_o[from][i][lane]);
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
  if (u.ns == 1) write_row<R, D>(a, c, hq, u.q0 + qt, g);
  else write_part<R, R, D>(parts, c, u, h, heads, j, g);
}

// ------------------------------------------------------------------------------------------------------ many rows per head
// Four waves of 32 rows each share a unit's tokens, 64 at a time: codes come through registers (the next stage's loads in flight
// during this stage's arithmetic), are decoded once per workgroup and lie in LDS as fp16 fragments, in the order in which the
// waves read them: 16 bytes per lane, contiguous.  Two buffers, one barrier per stage.
// Decoding ahead of LDS costs a wave a quarter of the conversions and doubles the LDS bytes: at 128 dims a wave reads 16 KB per 32
// tokens, 512 clocks for four waves at 128 B per clock, as long as their matrix instructions; decoding behind it would put 128
// conversions per 32 tokens beside every wave's softmax arithmetic, which is the longer pipe.
// 512 rows of 32 heads over 64 k tokens of 128 dims: 678 us, 814 TFLOP/s, matrix pipe busy 40 % of the time, vector pipe 56 %.  Computing a
// stage's scores beside the former's weights needs 230 registers, and loses more by the wave that then does not fit (790 us).
// fp32 rows, two planes of queries and weights: 4 x 1674 rows x 8 over 1.7 to 8.4 k tokens of 64 dims 173 us, matrix pipe 35 %, vector
// pipe 55 %; of 128 dims one wave per SIMD (219 + 96 registers), which hides little: 450 us, 24 % and 29 %; 2 x 2048 causal rows of 32
// heads over 10 k tokens 1.43 ms, 35 % and 38 %, against 702 us for bf16 rows.
constexpr int WROWS = 128;

template <int D, int CODE, int NS>
__global__ __launch_bounds__(256, NS == 2 && D == 128 ? 1 : 2) void attn_wide(rmem_bank8_attn_args a, Parts parts, Split sp) {
  constexpr int R = 32, CH = D / 32;             // 16-byte chunks per thread and stage: 8 D / 256
  constexpr int HALF = 64 * D / 8;               // fragments (16 bytes) of a stage's keys; as many of its values
  __shared__ __attribute__((aligned(16))) u32x4_t s_kv[2][2 * HALF];
  const int G = sp.G, ps = sp.ps;
  const int tid = threadIdx.x, lane = tid & 63, g = lane / R, j = lane % R;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = a.bank.heads, h = blockIdx.x % heads;
  Unit u;
  if (!find_unit<WROWS>(a, sp, parts.before, blockIdx.x / heads, u)) return;
  const int row0 = u.rt * WROWS + wave * R, row = row0 + j, qt = row / G, hq = h * G + row % G;
  const bool on = qt < u.n;
  const int lim = !on ? 0 : a.causal ? min(u.len, u.len - u.n + qt + 1) : u.len;
  const Sees see = rows_see<R>(u, row0, a.causal, G);                        // this wave's rows
  const int tiles = (rows_see<WROWS>(u, u.rt * WROWS, a.causal, G).sees + 31) >> 5, per = (tiles + u.ns - 1) / u.ns;
  const int t0 = u.part * per, t1 = min(tiles, t0 + per), stages = (t1 - t0 + 1) >> 1;

  Query<R, D, NS> q;
  load_query<R, D, NS>(q, a, u.q0 + qt, hq, on, g);

  const int page = a.bank.page;
  const long block = (long)page * D;
  const int32_t* table = a.table + (long)u.r * a.ld_table;
  const uint8_t* kb = a.bank.k + h * block;
  const uint8_t* vb = a.bank.v + h * block;
  const long pstride = heads * block;
  const int sub_mask = (1 << (ps - 5)) - 1;

  // page of tile t0 + 64 c + lane; -1: none
  auto pages_of = [&](int c) __attribute__((always_inline)) {
    const int t = t0 + 64 * c + lane;
    int id = -1;
    if (t < t1) id = table[t >> (ps - 5)];
    return id < a.bank.pages ? id : -1;
  };
  u32x4_t raw[CH];
  int page0 = -1, page1 = -1;                    // pages of the two tiles in `raw`
  int load_pid = -1;                             // pages of the 64 tiles around them
  auto load = [&](int st) __attribute__((always_inline)) {
    if ((st & 31) == 0) {
      load_pid = pages_of(st >> 5);
      asm volatile("" : "+v"(load_pid));         // waited for here: behind the branch every stage would wait for all loads in flight
    }
    const int i = (2 * st) & 63, ta = t0 + 2 * st;
    page0 = __builtin_amdgcn_readlane(load_pid, i);
    page1 = __builtin_amdgcn_readlane(load_pid, i + 1);
    const long a0 = (page0 < 0 ? 0 : page0) * pstride, a1 = (page1 < 0 ? 0 : page1) * pstride;
    const int s0 = ta & sub_mask, s1 = (ta + 1) & sub_mask;
#pragma unroll
    for (int it = 0; it < CH; ++it) {
      const int c = it * 256 + tid;
      const uint8_t* p;
      if (it * 256 + wave * 64 < 4 * D) {        // keys: a wave takes the 64 tokens of 16 dims
        const int tok = c & 63, cc = c >> 6;
        p = kb + (tok < 32 ? a0 + s0 * 512 : a1 + s1 * 512) + (unsigned)(cc * page + (tok & 31)) * 16u;
      } else {                                   // values: dims of half th & 1 of tile th >> 1, the same tile for a wave
        const int v = c - 4 * D, d = v % D, th = v / D;
        p = vb + (__builtin_amdgcn_readfirstlane(th >> 1) ? a1 + s1 * (32 * D) : a0 + s0 * (32 * D)) + (unsigned)((th & 1) * D + d) * 16u;
      }
      raw[it] = *reinterpret_cast<const u32x4_t*>(p);
    }
  };
  auto put = [&](int st, u32x4_t* to) __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < CH; ++it) {
      const int c = it * 256 + tid;
      u32x4_t x = raw[it];
      int at;
      if (it * 256 + wave * 64 < 4 * D) {
        const int tok = c & 63, cc = c >> 6;
        at = ((((tok >> 5) * (D / 16) + (cc & ~1)) * 2 + (cc & 1)) << 5) + (tok & 31);
      } else {
        const int v = c - 4 * D, d = v % D, th = v / D;
        at = HALF + ((((th >> 1) * (D / 32) + (d >> 5)) * 4 + (th & 1)) << 5) + (d & 31);
        if constexpr (CODE == E4M3) {            // NaN codes behind the last token, or of the page read for an absent one
          const int sub = __builtin_amdgcn_readfirstlane(th >> 1), left = (sub ? page1 : page0) < 0 ? 0 : u.len - (t0 + 2 * st + sub) * 32;
          if (left < 32) {
#pragma unroll
            for (int m = 0; m < 4; ++m) x[m] = keep_first(x[m], left - 8 * m - 4 * (th & 1));
          }
        }
      }
      to[at] = __builtin_bit_cast(u32x4_t, decode8<CODE>(x[0], x[1]));
      to[at + 64] = __builtin_bit_cast(u32x4_t, decode8<CODE>(x[2], x[3]));
    }
  };

  Acc<R, D> c;
  c.clear();
  int pid = -1;                                  // pages and scales of 64 tiles, one per lane
  float ks = 0.f, lvs = 0.f, ivs = 1.f;
  if (stages > 0) {
    load(0);
    put(0, s_kv[0]);
    load(min(1, stages - 1));
  }
  for (int st = 0; st < stages; ++st) {
    if ((st & 31) == 0) {
      pid = pages_of(st >> 5);
      float vs = 1.f;
      ks = 0.f;
      if (pid >= 0) {
        ks = a.bank.k_scale[(long)pid * heads + h];
        vs = fmaxf(a.bank.v_scale[(long)pid * heads + h], VS_MIN);
      }
      lvs = __log2f(vs);
      ivs = 1.0f / vs;
      asm volatile("" : "+v"(pid), "+v"(ks));    // as above
    }
    __syncthreads();                             // stage st is in its buffer, and every wave is done with the other one
    if (st + 1 < stages) put(st + 1, s_kv[(st + 1) & 1]);
    if (st + 2 < stages) load(st + 2);
    const u32x4_t* kv = s_kv[st & 1];
    const int t = t0 + 2 * st, i = (2 * st) & 63, tok0 = t * 32;
    if (tok0 >= see.sees) continue;
    const bool gone0 = __builtin_amdgcn_readlane(pid, i) < 0, gone1 = __builtin_amdgcn_readlane(pid, i + 1) < 0;   // (-1 from t1 on)
    const int lims[2] = {gone0 ? tok0 : lim, gone1 ? tok0 + 32 : lim};
    const float k2[2] = {readlane(ks, i), readlane(ks, i + 1)}, l2[2] = {readlane(lvs, i), readlane(lvs, i + 1)},
                i2[2] = {readlane(ivs, i), readlane(ivs, i + 1)};
    attend_tiles<2, R, D, NS>(c, q, tok0, lims, k2, l2, i2, g, gone0 || gone1 || tok0 + 64 > min(see.all, u.len),
                       [&](int sub, int k, int) { return __builtin_bit_cast(frag8_t, kv[(sub * (D / 16) + k) * 64 + lane]); },
                       [&](int sub, int d, int k) { return __builtin_bit_cast(frag8_t, kv[HALF + ((sub * (D / 32) + d) * 2 + k) * 64 + lane]); });
  }
  c.l = row_sum<R>(c.l);
  if (!on) return;
  if (u.ns == 1) write_row<R, D>(a, c, hq, u.q0 + qt, g);
  else write_part<WROWS, R, D>(parts, c, u, h, heads, wave * R + j, g);
}

// ------------------------------------------------------------------------------------------------------------------- merge
// One workgroup per (row tile in several parts, kv head, BLOCK rows of the tile), a fixed number of workgroups that step through
// them: a grid for the most there could be costs more than the work (most calls have few or none).  Few parts: one thread per
// four dims of a row, which walks them.  Many: a wave per row, the parts over its 256 / D groups of lanes.  64 rows of 32 heads of 128
// dims 6 us, 4 x 1674 rows of 8 x 32 13 us, 36 MB.
constexpr int merge_block(int rows) { return rows == 16 ? 4 : rows == 32 ? 8 : 16; }
constexpr int FEW_PARTS = 8;

template <int D>
__device__ __forceinline__ float over_groups(float x) {       // sum over the lanes that hold the same dims
  x += xor_lane<32>(x);
  if constexpr (D <= 64) x += xor_lane<16>(x);
  if constexpr (D <= 32) x += xor_lane<8>(x);
  return x;
}

template <int ROWS, int D>
__device__ __forceinline__ void merge(const rmem_bank8_attn_args& a, const Parts& parts, const Split& sp, int block, int blocks) {
  constexpr int WIDTH = D / 4, GROUPS = 64 / WIDTH, BLOCK = merge_block(ROWS), BLOCKS = ROWS / BLOCK;
  const int heads = a.bank.heads, lane = threadIdx.x & 63, G = sp.G;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool wide = wide_stores(a);
  const long tiles = count_split<ROWS>(a, sp, parts.before), items = (tiles < parts.ords ? tiles : parts.ords) * heads * BLOCKS;
  auto finish = [&](const Split_tile& t, int h, int j, int d4, f32x4_t o, float m, float l, bool mine) __attribute__((always_inline)) {
    const int row = t.rt * ROWS + j, hq = h * G + row % G;
    const long at = t.q0 + row / G;
    const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
    if (mine) {
      by_type(a.type, a.out, [&](auto* p) { store4(p + at * a.o_row + hq * a.o_head + d4 * 4, o * inv, wide); });
      if (a.lse && d4 == 0) a.lse[at * a.heads_q + hq] = (__log2f(l) + m - LIFT) * LN2;
    }
  };
  for (long item = block; item < items; item += blocks) {
    const long th = item / BLOCKS;
    const int h = (int)(th % heads), end = (int)(item % BLOCKS + 1) * BLOCK;
    const Split_tile t = parts.tiles[th / heads];
    // (row offsets that are none -- requests that overlap -- can leave a descriptor unwritten)
    if (t.slot < 0 || t.ns < 2 || t.ns > parts.slots - t.slot || t.q0 < 0 || t.n < 0 || t.n > a.rows - t.q0 || t.rt < 0 ||
        t.rt > 0x7fffffff / ROWS - 1)
      continue;
    const int rows = min(end, t.n * G - t.rt * ROWS);        // of the tile that exist (n * G < 2^31: checked on the host)
    const long step = (long)heads * ROWS;
    if (t.ns <= FEW_PARTS) {
      const int d4 = threadIdx.x % WIDTH;
      for (int j = end - BLOCK + threadIdx.x / WIDTH; j < rows; j += 256 / WIDTH) {
        const long first = ((long)t.slot * heads + h) * ROWS + j;
        float pm[FEW_PARTS], pl[FEW_PARTS], m = LOWEST, l = 0.f;
        f32x4_t x[FEW_PARTS], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < FEW_PARTS; ++p) {
          const long at = first + min(p, t.ns - 1) * step;
          pm[p] = parts.ml[at * 2];
          pl[p] = parts.ml[at * 2 + 1];
          x[p] = *reinterpret_cast<const f32x4_t*>(parts.o + at * D + d4 * 4);
        }
#pragma unroll
        for (int p = 0; p < FEW_PARTS; ++p) m = fmaxf(m, pm[p]);
#pragma unroll
        for (int p = 0; p < FEW_PARTS; ++p) {
          const float f = p < t.ns ? __builtin_amdgcn_exp2f(pm[p] - m) : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = p < t.ns ? fmaf(x[p][e], f, o[e]) : o[e];
          l = p < t.ns ? fmaf(pl[p], f, l) : l;
        }
        finish(t, h, j, d4, o, m, l, true);
      }
    } else {
      const int g = lane / WIDTH, d4 = lane % WIDTH;
      for (int j = end - BLOCK + wave; j < rows; j += 4) {
        const long first = ((long)t.slot * heads + h) * ROWS + j;
        float m = LOWEST;
        for (int p = lane; p < t.ns; p += 64) m = fmaxf(m, parts.ml[(first + p * step) * 2]);
        m = wave_max_xor(m);
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll 8
        for (int p = g; p < t.ns; p += GROUPS) {
          const long at = first + p * step;
          const float f = __builtin_amdgcn_exp2f(parts.ml[at * 2] - m);
          const f32x4_t x = *reinterpret_cast<const f32x4_t*>(parts.o + at * D + d4 * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
          l = fmaf(parts.ml[at * 2 + 1], f, l);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = over_groups<D>(o[e]);
        l = over_groups<D>(l);
        finish(t, h, j, d4, o, m, l, g == 0);
      }
    }
  }
}

template <int ROWS, int D>
__global__ __launch_bounds__(256) void attn_merge(rmem_bank8_attn_args a, Parts parts, Split sp) {
  merge<ROWS, D>(a, parts, sp, blockIdx.x, gridDim.x);
}
// of the wide kernel's parts (the first `first` workgroups) and the narrow kernel's beside it: one launch instead of two, 4 us
template <int D>
__global__ __launch_bounds__(256) void attn_merge_both(rmem_bank8_attn_args a, Parts wide, Split wide_sp, Parts narrow, Split narrow_sp, int first) {
  if ((int)blockIdx.x < first) merge<WROWS, D>(a, wide, wide_sp, blockIdx.x, first);
  else merge<32, D>(a, narrow, narrow_sp, blockIdx.x - first, gridDim.x - first);
}

// -------------------------------------------------------------------------------------------------------------------- host
constexpr int ROWS16 = 16;              // requests of at most this many rows per kv head take tiles of 16 rows
// Up to this many the narrow kernel, beyond the wide one.  Narrow and wide, with their merges, us: 4 requests of 32 tokens and 4 x 8
// heads (256 rows per kv head) over 16 k tokens of 128 dims 59, 70; 4 of 256 tokens and 8 heads over 8 k of 64 dims 41, 56; 20 of 130
// fp32 tokens and 8 heads over 2 k of 32 dims 40, 49; one of 60 tokens and 8 x 4 heads over 20 k of 128 dims 41, 50; 64 of 16 tokens and
// 4 x 8 heads over 4 k of 128 dims 115, 114.
constexpr int NARROW_ROWS = 256;
constexpr int NARROW_CHUNK = 8;         // fewest 32-token tiles worth a part
constexpr int WIDE_CHUNK = 16;

// Parts of all kv heads that a read is divided into: as many as there are workgroups on the chip at once (registers: two on each of 256
// CUs at 128 dims, four of the wide kernel below; more parts add starts and more to merge, fewer leave CUs idle).  With 512 / 1024 /
// 1536 / 2048 parts, us:
//   wide, 8 x 32:    2 x 1000 fp32 rows over 5 k tokens 55 / 53 / 59 / 61, 4 x 1674 over 1.7 to 8.4 k 144 / 131 / 123 / 129,
//                    6 x 500 causal rows of 4 x 2 heads over 3.5 k 53 / 50 / 52 / 52, 1 x 3600 over 18 k 220 / 218 / 217 / 224
//   wide, 64 dims:   2 x 400 causal rows of 4 heads in one over 30 k 78 / 67 / 75 / 77, 3 x 2400 fp32 rows x 8 over 2.4 to 9.6 k
//                    221 / 232 / 236 / 233
//   narrow, 8 x 32:  64 rows over 16 to 33 k 37 / 35 / 35 / 34, 4 x 100 fp32 rows over 8 k 30 / 30 / 35 / 36
// and with 256 / 512 / 1024 / 2048 parts at 128 dims:
//   wide:            3 x 2400 fp32 rows x 8 over 2.4 to 9.6 k 581 / 505 / 521 / 537, 16 x 300 fp16 over 1 k 61 / 74 / 75 / 76
//   narrow:          64 rows x 8 over 16 to 33 k 123 / 104 / 102 / 103, 4 x 100 fp32 rows over 8 k 52 / 53 / 60 / 72
int parts_of(int dim) { return dim == 128 ? 512 : 1024; }

struct Launch {
  Split sp;
  int rows;                       // rows of a tile
  long tiles, units, slots;       // per kv head: bounds of row tiles, units, partial results
};
struct Plan {
  Launch narrow, wide;            // units 0: not used
};

bool valid_attn(const rmem_bank8_attn_args* a) {
  if (!a || !valid_bank(&a->bank) || !valid_type(a->type) || a->reqs <= 0 || a->rows < 0 || a->cols <= 0 || a->ld_table < a->cols ||
      (int64_t)a->cols * a->bank.page > 0x7fffffff || a->heads_q <= 0 || a->heads_q % a->bank.heads || !(a->scale > 0.f) ||
      !(a->scale < 3.0e38f))
    return false;
  return (int64_t)a->rows * (a->heads_q / a->bank.heads) <= 0x7fffff00;
}

Launch make_launch(const rmem_bank8_attn_args* a, int rows, int units, int chunk_min, int lo, int hi) {
  Launch l;
  l.sp.G = a->heads_q / a->bank.heads;
  l.sp.ps = log2_of(a->bank.page);
  l.sp.want = units / a->bank.heads > 0 ? units / a->bank.heads : 1;
  l.sp.chunk_min = chunk_min;
  l.sp.lo = lo;
  l.sp.hi = hi;
  l.rows = rows;
  const long reqs = std::min(a->reqs, a->rows);            // with rows
  l.tiles = (long)a->rows * l.sp.G / rows + reqs;
  l.tiles = std::min(l.tiles, reqs * (((long)hi + rows - 1) / rows));
  // parts: at most total / chunk + one per row tile; of requests in several parts, at most twice total / chunk
  l.units = l.sp.want + l.tiles;
  // a request whose row of the table holds no more than the smallest part is never divided
  l.slots = ((long)a->cols * a->bank.page + 31) / 32 > chunk_min ? 2L * l.sp.want : 0;
  return l;
}

Plan make_plan(const rmem_bank8_attn_args* a) {
  const long most = (long)a->max_rows * (a->heads_q / a->bank.heads);
  const int all = 0x7fffffff;
  Plan p = {};
  if (most <= NARROW_ROWS) p.narrow = make_launch(a, most <= ROWS16 ? 16 : 32, parts_of(a->bank.dim), NARROW_CHUNK, 0, all);
  else {
    // one request: the wide kernel alone; several: the short ones among them in a launch of their own
    p.wide = make_launch(a, WROWS, parts_of(a->bank.dim), WIDE_CHUNK, a->reqs == 1 ? 0 : NARROW_ROWS + 1, all);
    if (a->reqs > 1) p.narrow = make_launch(a, 32, parts_of(a->bank.dim), NARROW_CHUNK, 0, NARROW_ROWS);
  }
  return p;
}

// A launch of 256 threads per workgroup counts its threads in 32 bits.
constexpr long MOST_GROUPS = 1L << 24;
bool fits_grids(const rmem_bank8_attn_args* a, const Plan& p) {
  return p.narrow.units * a->bank.heads < MOST_GROUPS && p.wide.units * a->bank.heads < MOST_GROUPS;
}

// floats of a launch's workspace: partial results, references and sums, tiles in several parts (at most `want`: two parts each),
// the division's index; each a multiple of 16 bytes
long part_floats(const rmem_bank8_attn_args* a, const Launch& l) {
  const long index = a->reqs > 64 ? (a->reqs + 1L) * (long)(sizeof(Before) / 4) : 0;
  return l.slots * a->bank.heads * l.rows * (a->bank.dim + 2) + (l.slots ? l.sp.want : 0) * (long)(sizeof(Split_tile) / 4) + index;
}

template <int D, int CODE, int NS>
void launch_attn(const rmem_bank8_attn_args& a, const Parts& parts, const Launch& l, hipStream_t s) {
  const dim3 grid((unsigned)(l.units * a.bank.heads));
  if (l.rows == 16) hipLaunchKernelGGL((attn_narrow<16, D, CODE, NS>), grid, dim3(256), 0, s, a, parts, l.sp);
  else if (l.rows == 32) hipLaunchKernelGGL((attn_narrow<32, D, CODE, NS>), grid, dim3(256), 0, s, a, parts, l.sp);
  else hipLaunchKernelGGL((attn_wide<D, CODE, NS>), grid, dim3(256), 0, s, a, parts, l.sp);
}

template <int D>
void launch_tiles(const rmem_bank8_attn_args& a, const Parts& parts, const Launch& l, hipStream_t s) {
  const bool e4m3 = a.bank.code == E4M3, two = a.type == FP32;
  if (e4m3) two ? launch_attn<D, E4M3, 2>(a, parts, l, s) : launch_attn<D, E4M3, 1>(a, parts, l, s);
  else two ? launch_attn<D, INT8, 2>(a, parts, l, s) : launch_attn<D, INT8, 1>(a, parts, l, s);
}

int merge_grid(const rmem_bank8_attn_args& a, const Launch& l) {
  const long tiles = l.tiles < l.sp.want ? l.tiles : l.sp.want;         // row tiles in at least two parts: at most `want`
  return (int)std::min(tiles * a.bank.heads * (l.rows / merge_block(l.rows)), 2048L);
}
template <int D>
void launch_merge(const rmem_bank8_attn_args& a, const Parts& parts, const Launch& l, hipStream_t s) {
  const dim3 grid(merge_grid(a, l));
  if (l.rows == 16) hipLaunchKernelGGL((attn_merge<16, D>), grid, dim3(256), 0, s, a, parts, l.sp);
  else if (l.rows == 32) hipLaunchKernelGGL((attn_merge<32, D>), grid, dim3(256), 0, s, a, parts, l.sp);
  else hipLaunchKernelGGL((attn_merge<WROWS, D>), grid, dim3(256), 0, s, a, parts, l.sp);
}

int place(const rmem_bank8_attn_args& a, float* ws, const Launch& l, Parts& parts, hipStream_t s) {
  parts.o = ws;
  parts.ml = ws + l.slots * a.bank.heads * l.rows * a.bank.dim;
  parts.tiles = reinterpret_cast<Split_tile*>(parts.ml + l.slots * a.bank.heads * l.rows * 2);
  parts.slots = (int)l.slots;
  parts.ords = l.slots ? l.sp.want : 0;
  parts.before = nullptr;
  if (a.reqs > 64) {
    Before* index = reinterpret_cast<Before*>(parts.tiles + parts.ords);
    if (l.rows == 16) hipLaunchKernelGGL(index_kernel<16>, dim3(1), dim3(1024), 0, s, a, l.sp, index);
    else if (l.rows == 32) hipLaunchKernelGGL(index_kernel<32>, dim3(1), dim3(1024), 0, s, a, l.sp, index);
    else hipLaunchKernelGGL(index_kernel<WROWS>, dim3(1), dim3(1024), 0, s, a, l.sp, index);
    RMEM_CHECK_LAUNCH();
    parts.before = index;
  }
  return RMEM_OK;
}

template <int D>
int launch_dim(const rmem_bank8_attn_args& a, float* ws, const Plan& p, hipStream_t s) {
  Parts wide, narrow;
  if (p.wide.units) {
    const int rc = place(a, ws, p.wide, wide, s);
    if (rc != RMEM_OK) return rc;
    launch_tiles<D>(a, wide, p.wide, s);
    RMEM_CHECK_LAUNCH();
    ws += part_floats(&a, p.wide);
  }
  if (p.narrow.units) {
    const int rc = place(a, ws, p.narrow, narrow, s);
    if (rc != RMEM_OK) return rc;
    launch_tiles<D>(a, narrow, p.narrow, s);
    RMEM_CHECK_LAUNCH();
  }
  const bool w = p.wide.units && p.wide.slots, n = p.narrow.units && p.narrow.slots;
  if (w && n) {
    const int first = merge_grid(a, p.wide);
    hipLaunchKernelGGL((attn_merge_both<D>), dim3(first + merge_grid(a, p.narrow)), dim3(256), 0, s, a, wide, p.wide.sp, narrow, p.narrow.sp, first);
  } else if (w) launch_merge<D>(a, wide, p.wide, s);
  else if (n) launch_merge<D>(a, narrow, p.narrow, s);
  RMEM_CHECK_LAUNCH();
  return RMEM_OK;
}

}  // namespace

extern "C" int64_t rmem_bank8_attn_workspace(const rmem_bank8_attn_args* a) {
  if (!valid_attn(a)) return -1;
  const Plan p = make_plan(a);
  if (!fits_grids(a, p)) return -1;
  return 4 * ((p.narrow.units ? part_floats(a, p.narrow) : 0) + (p.wide.units ? part_floats(a, p.wide) : 0));
}

extern "C" int rmem_bank8_attn(const rmem_bank8_attn_args* a, void* stream) {
  if (!valid_attn(a)) return RMEM_ERR_INVALID;
  if (a->rows == 0) return RMEM_OK;
  const Plan p = make_plan(a);
  const int64_t need = rmem_bank8_attn_workspace(a);
  if (need < 0 || !a->q || !a->out || !a->cu || !a->lens || !a->table ||
      (need && (!a->workspace || ((uintptr_t)a->workspace % 16) || a->workspace_bytes < need)))
    return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* ws = static_cast<float*>(a->workspace);
  return a->bank.dim == 32 ? launch_dim<32>(*a, ws, p, s) : a->bank.dim == 64 ? launch_dim<64>(*a, ws, p, s) : launch_dim<128>(*a, ws, p, s);
}
