// bank8.hip -- the paged 8-bit bank: block tables and slot maps (plan), writing tokens (append), reading them back (gather).
// Storage and semantics: include/rmem_hip.h and bank8.h; the read over the pages is bank8_attn.hip.
#include "bank8.h"

#include <algorithm>
#include <type_traits>

using namespace bank8;

namespace {

// ------------------------------------------------------------------------------------------------------------------- plan
// One workgroup: the requests are scanned (pages asked for, rows, pages going back) up to 1024 at a time, the page ids that
// move are spread over the threads by binary search in the scan.  Bound by the chain of dependent memory reads (lengths -> ring
// and table entries), not by bytes; one workgroup keeps it one launch and lets state and lengths be updated in place.
// 64 requests of one token 4.4 us; 500 with 17 k rows, 40 of them ending, 12 us and 4 us for the slot map.
constexpr int PT = 1024;

struct Scan3 {
  long long a, b, c;
};
__device__ __forceinline__ long long shfl_up64(long long x, int o) {
  const unsigned lo = __shfl_up((unsigned)x, o), hi = __shfl_up((unsigned)(x >> 32), o);
  return (long long)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ long long clamp_add(int x) { return x > 0 ? x : 0; }

__device__ __forceinline__ int upper_bound(const long long* cum, int n, long long x) {   // first i with cum[i] > x, n if none
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// rows up to which the planning workgroup writes the slot map itself
constexpr int SLOTS_INLINE = 4096;

// slot of a token; -1 where the table names no page that a slot could name
__device__ __forceinline__ int slot_of(int id, long long pos, int ps) {
  return (unsigned)id >> (31 - ps) ? -1 : (id << ps) + (int)(pos & ((1 << ps) - 1));
}

__global__ __launch_bounds__(PT) void plan_kernel(rmem_bank8_plan_args p, int ps) {
  __shared__ long long s_need[PT], s_rows[PT], s_back[PT];   // inclusive sums within the chunk
  __shared__ int s_held[PT], s_start[PT], s_rel[PT];
  __shared__ long long s_wave[3][PT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int page_mask = (1 << ps) - 1, threads = blockDim.x;
  int head = p.state_in[0], count = p.state_in[1];
  head %= p.ring;
  head += head < 0 ? p.ring : 0;
  count = count < 0 ? 0 : count > p.ring ? p.ring : count;
  auto ring_at = [&](long long i) { const long long at = head + i; return at >= p.ring ? at - p.ring : at; };   // i < ring
  long long c_need = 0, c_rows = 0, c_back = 0;              // carried from earlier chunks
  long long taken = 0, missing = 0;                          // this thread's requests
  const bool inline_slots = p.rows <= SLOTS_INLINE;
  for (int base = 0; base < p.reqs; base += threads) {
    const int r = base + tid;
    long long ctx = 0, add = 0, need = 0, asked = 0, back = 0, held = 0;
    bool fits = false;
    if (r < p.reqs) {
      ctx = clamp_add(p.ctx[r]);
      add = clamp_add(p.add[r]);
      const long long had = p.had ? clamp_add(p.had[r]) : 0;
      held = (ctx + page_mask) >> ps;
      need = ((ctx + add + page_mask) >> ps) - held;
      fits = held + need <= p.cols;
      asked = fits ? need : 0;
      long long was = (had + page_mask) >> ps;
      if (was > p.cols) was = p.cols;
      back = was > held ? was - held : 0;
    }
    long long x = asked, y = add, z = back;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long xu = shfl_up64(x, o), yu = shfl_up64(y, o), zu = shfl_up64(z, o);
      if (lane >= o) {
        x += xu;
        y += yu;
        z += zu;
      }
    }
    if (lane == 63) {
      s_wave[0][wave] = x;
      s_wave[1][wave] = y;
      s_wave[2][wave] = z;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      x += s_wave[0][w];
      y += s_wave[1][w];
      z += s_wave[2][w];
    }
    const bool granted = fits && (need == 0 || c_need + x <= count);
    s_need[tid] = x;
    s_rows[tid] = y;
    s_back[tid] = z;
    s_held[tid] = (int)(held < 0x7fffffff ? held : 0x7fffffff);
    s_start[tid] = granted ? (int)ctx : -1;
    s_rel[tid] = 0;
    if (r < p.reqs) {
      if (granted) taken += need; else missing += need;
      const long long row = c_rows + y;
      p.cu[r + 1] = (int)(row < 0x7fffffff ? row : 0x7fffffff);
      p.lens[r] = (int)(granted ? ctx + add : ctx);
      p.start[r] = s_start[tid];
      if (r == 0) p.cu[0] = 0;
    }
    __syncthreads();
    const int nr = min(p.reqs - base, threads);
    const long long n_need = s_need[nr - 1], n_rows = s_rows[nr - 1], n_back = s_back[nr - 1];
    // pages going back, before new entries can overwrite them in the table
    for (long long i = tid; i < n_back; i += threads) {
      const int k = upper_bound(s_back, nr, i);
      const long long j = i - (k ? s_back[k - 1] : 0);
      const long long at = count + c_back + i;
      if (at < p.ring)                                       // (more pages than the ring has places: dropped, and not counted)
        p.free_ring[ring_at(at)] = p.table[(base + k) * p.ld_table + s_held[k] + j];
    }
    if (n_back) __syncthreads();
    for (long long i = tid; i < n_need; i += threads) {
      const int k = upper_bound(s_need, nr, i);
      const long long j = i - (k ? s_need[k - 1] : 0);
      if (s_start[k] >= 0) p.table[(base + k) * p.ld_table + s_held[k] + j] = p.free_ring[ring_at(c_need + i)];
    }
    if (inline_slots) {
      // rows of this chunk; entries are taken from where they come from, so nothing waits for the table's writes
      const long long end = c_rows + n_rows < p.rows ? c_rows + n_rows : p.rows;
      for (long long t = c_rows + tid; t < end; t += threads) {
        const int k = upper_bound(s_rows, nr, t - c_rows);
        const int start = s_start[k];
        int slot = -1;
        if (start >= 0) {
          const long long pos = start + (t - c_rows) - (k ? s_rows[k - 1] : 0);
          const long long pi = pos >> ps;
          const int id = pi >= s_held[k] ? p.free_ring[ring_at(c_need + (k ? s_need[k - 1] : 0) + pi - s_held[k])]
                                         : p.table[(base + k) * p.ld_table + pi];
          slot = slot_of(id, pos, ps);
        }
        p.slots[t] = slot;
      }
    }
    c_need += n_need;
    c_rows += n_rows;
    c_back += n_back;
    __syncthreads();                                         // the chunk's sums are overwritten next
  }
  if (inline_slots)
    for (long long t = c_rows + tid; t < p.rows; t += threads) p.slots[t] = -1;
  // totals
  long long x = taken, y = missing;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long xu = shfl_up64(x, o), yu = shfl_up64(y, o);
    if (lane >= o) {
      x += xu;
      y += yu;
    }
  }
  if (lane == 63) {
    s_wave[0][wave] = x;
    s_wave[1][wave] = y;
  }
  __syncthreads();
  if (tid == 0) {
    long long t = 0, m = 0;
    for (int w = 0; w < threads / 64; ++w) {
      t += s_wave[0][w];
      m += s_wave[1][w];
    }
    // what was written above: the places that this step's grants leave hold granted pages, which must not be counted as free
    const long long held = count + c_back < p.ring ? count + c_back : p.ring;
    p.state_out[0] = (int)(head + t >= p.ring ? head + t - p.ring : head + t);
    p.state_out[1] = (int)(held - t);
    p.status[0] = (int)t;
    p.status[1] = (int)(m < 0x7fffffff ? m : 0x7fffffff);
  }
}

// the slot map of a long step, from the finished table
__global__ __launch_bounds__(256) void slots_kernel(rmem_bank8_plan_args p, int ps) {
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t >= p.rows) return;
  int lo = 0, hi = p.reqs;                                   // first r with cu[r + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  int slot = -1;
  if (lo < p.reqs) {
    const int start = p.start[lo];
    if (start >= 0) {
      const long long pos = start + t - p.cu[lo];
      slot = slot_of(p.table[lo * p.ld_table + (pos >> ps)], pos, ps);
    }
  }
  p.slots[t] = slot;
}

// ----------------------------------------------------------------------------------------------------------------- append
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;                      // NaN and infinities do not set a scale
}

// Rows of a call may reach a page in any order, so a page's rows are gathered first: the workgroup of the page's first row finds
// them all and writes the page, the others leave.  Up to SCAN_ROWS rows every workgroup that begins a run reads the whole slot map
// (16 KB at most, from the L2); beyond, two small launches mark each page's first row and count its runs, and only a page that is
// reached by several runs is searched for.
constexpr int SCAN_ROWS = 4096;
constexpr int GRID_Y = 32768;            // windows over the grid's y, further ones over z
constexpr int APPEND_GROUPS = 4096;      // workgroups from which on a workgroup takes several rows

__device__ __forceinline__ bool in_pool(int slot, const rmem_bank8& b) { return slot >= 0 && slot < b.pages * (long)b.page; }
// whether `row` goes on where the row before it ended, in the same page
__device__ __forceinline__ bool goes_on(const int32_t* slots, int row, int slot, int page) {
  return row && (slot & (page - 1)) && slots[row - 1] == slot - 1;
}

struct PageMark {
  int first, runs;
};
__global__ __launch_bounds__(256) void mark_clear_kernel(rmem_bank8_append_args a, PageMark* marks, int ps) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const int slot = a.slots[row];
  if (!in_pool(slot, a.bank) || goes_on(a.slots, row, slot, a.bank.page)) return;   // (each page that is reached has a run's begin)
  marks[slot >> ps].first = 0x7fffffff;
  marks[slot >> ps].runs = 0;
}
__global__ __launch_bounds__(256) void mark_kernel(rmem_bank8_append_args a, PageMark* marks, int ps) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const int slot = a.slots[row];
  if (!in_pool(slot, a.bank) || goes_on(a.slots, row, slot, a.bank.page)) return;
  atomicMin(&marks[slot >> ps].first, row);
  atomicAdd(&marks[slot >> ps].runs, 1);
}

// N elements as they lie in memory: one vector (or several of 16 bytes) with WIDE.  Loads are issued for all of a
// thread's places, rows that do not exist reading one that does: a branch around a load ends in a wait for it.
template <class T, int N, bool WIDE>
struct Run {
  static constexpr int V = !WIDE ? 1 : N < 16 / (int)sizeof(T) ? N : 16 / (int)sizeof(T);
  typedef __attribute__((ext_vector_type(V))) T vec_t;
  vec_t y[N / V];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < N / V; ++k) y[k] = *reinterpret_cast<const vec_t*>(p + k * V);
  }
  __device__ __forceinline__ float at(int e) const { return (float)y[e / V][e % V]; }
};
// Largest magnitude of many elements by their bits, two 16-bit ones at a time: without the sign they order as integers do, infinity
// and NaN above all numbers.
template <class T, int V>
struct Top {
  typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> bits_t;
  typedef __attribute__((ext_vector_type(V))) bits_t vec_t;
  static constexpr bits_t SIGN = (bits_t)(1u << (8 * sizeof(T) - 1)), ENDLESS = sizeof(T) == 4 ? 0x7f800000u : std::is_same_v<T, _Float16> ? 0x7c00u : 0x7f80u;
  vec_t top = (vec_t)(bits_t)0;
  template <int N, bool WIDE>
  __device__ __forceinline__ void take(const Run<T, N, WIDE>& x) {
#pragma unroll
    for (int k = 0; k < N / V; ++k) top = __builtin_elementwise_max(top, __builtin_bit_cast(vec_t, x.y[k]) & (bits_t)~SIGN);
  }
  __device__ __forceinline__ float largest() const {           // infinity where an element is not finite
    bits_t t = top[0];
#pragma unroll
    for (int e = 1; e < V; ++e) t = t > top[e] ? t : top[e];
    return t < ENDLESS ? (float)__builtin_bit_cast(T, t) : INFINITY;
  }
};
// element `at` of row r: with FAST a 32-bit byte offset from the (uniform) base, one register instead of two for each of a
// thread's loads in flight
template <class T, bool FAST>
__device__ __forceinline__ const T* element(const T* src, long ldr, int r, int at) {
  if constexpr (FAST) return reinterpret_cast<const T*>(reinterpret_cast<const char*>(src) + ((unsigned)r * (unsigned)ldr + (unsigned)at) * (unsigned)sizeof(T));
  else return src + r * ldr + at;
}

// One workgroup per (window of rows, head, keys or values); each page that begins in the window (its first row in the call lies
// there) is read twice, for its largest value and, from the caches, to be encoded: holding it in registers in between (64 to 128 of
// them) leaves too few workgroups to hide the chain slots -> rows -> maximum -> codes.  Keys: a thread takes 16 dims of a token,
// eight threads a token of 128 dims (256 bytes in, 128-byte pieces out).  Values: a thread takes 16 tokens (half a 32-token tile)
// of two dims, so that a wave reads whole rows and each thread writes the two chunks that hold its tokens.
// 25.6 k fp16 rows of 8 x 128 to e4m3: 48 us for 157 MB, 3.3 TB/s -- what is left is that chain, at 20 waves per CU (16: 50 us; 32
// spill, and at 20 the form for fp32 rows that are not 16-byte aligned, by two or three registers); 64 single tokens 5.4 to 5.9 us.
template <class T, int CODE, int D, bool FAST, int NT>
__global__ __launch_bounds__(NT, 5) void append_kernel(rmem_bank8_append_args a, const PageMark* marks, int ps, int window) {
  __shared__ float s_max[NT / 64];
  __shared__ __attribute__((aligned(16))) int s_row[128];   // row that fills each place of the page, -1: none; the last of several
  __shared__ int s_other;
  const rmem_bank8& b = a.bank;
  const int zs = gridDim.z / 2, h = blockIdx.x, part = blockIdx.z >= zs;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int page = b.page;
  const T* src = static_cast<const T*>(part ? a.v : a.k) + (long)h * (part ? a.v_head : a.k_head);
  const long ldr = part ? a.v_row : a.k_row;
  // every wave looks the window's rows over at once: which of them begin a page that is this workgroup's to write
  const int row0 = ((blockIdx.z - part * zs) * GRID_Y + blockIdx.y) * window;
  if (row0 >= a.rows) return;
  int w_slot = -1, w_runs = 0, w_ahead[2];             // slots of this lane's row and of those 64 and 128 behind it
  bool begins = false;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = row0 + lane + 64 * (k + 1);
    w_ahead[k] = a.slots[min(r, a.rows - 1)];
    if (r >= a.rows) w_ahead[k] = -1;
  }
  if (row0 + lane < a.rows) w_slot = a.slots[row0 + lane];
  if (lane < window && row0 + lane < a.rows) {
    begins = in_pool(w_slot, b) && !goes_on(a.slots, row0 + lane, w_slot, page);
    if (marks && begins) {
      const PageMark m = marks[w_slot >> ps];
      begins = m.first == row0 + lane;
      w_runs = m.runs;
    }
  }
  for (unsigned long long todo = __ballot(begins); todo; todo &= todo - 1) {
    const int at0 = __builtin_ctzll(todo), row = row0 + at0;
    const int slot = __builtin_amdgcn_readlane(w_slot, at0), runs = __builtin_amdgcn_readlane(w_runs, at0);
    const int pg32 = slot >> ps, off = slot & (page - 1);
    float* scale_p = (part ? b.v_scale : b.k_scale) + (long)pg32 * b.heads + h;
    const float before = *scale_p;
    __syncthreads();                      // the page before has been written
    if (runs == 1) {
      // the run goes on where the slots do; a row further on that fitted the pattern again would begin another run
      for (int i = tid; i < 128; i += NT) {
        const int ahead = at0 + i - off, from = ahead & 63;      // below 64 + 128
        const int s0 = __shfl(w_slot, from), s1 = __shfl(w_ahead[0], from), s2 = __shfl(w_ahead[1], from);
        const int s = ahead < 64 ? s0 : ahead < 128 ? s1 : s2;
        s_row[i] = i >= off && i < page && s >= 0 && s == slot + i - off ? row + i - off : -1;
      }
      if (tid == 0) s_other = 0;
    } else {
      for (int i = tid; i < 128; i += NT) s_row[i] = -1;
      if (tid == 0) s_other = 0;
      __syncthreads();
      for (int r = marks ? row + tid : tid; r < a.rows; r += NT) {
        const int s = a.slots[r];
        if (s < 0 || (s >> ps) != pg32) continue;
        if (r < row) s_other = 1;
        else atomicMax(&s_row[s & (page - 1)], r);
      }
    }
    __syncthreads();
    if (s_other) continue;
    // places filled: first, one past the last, whether there are gaps
    const unsigned long long f0 = __ballot(s_row[lane] >= 0), f1 = __ballot(s_row[64 + lane] >= 0);
    const int lo = f0 ? __builtin_ctzll(f0) : 64 + __builtin_ctzll(f1), hi = f1 ? 128 - __builtin_clzll(f1) : 64 - __builtin_clzll(f0);
    const bool holes = __popcll(f0) + __popcll(f1) < hi - lo;

    uint8_t* codes = (part ? b.v : b.k) + ((long)pg32 * b.heads + h) * ((long)page * D);
    // the new tokens' largest value, four loads of eight elements in flight per thread
    constexpr int W = D / 8;
    const int any = s_row[lo];             // a place that no row fills reads this row, and does not change the maximum
    Top<T, Run<T, 8, FAST>::V> top;
    for (int u0 = tid; u0 < (hi - lo) * W; u0 += 4 * NT) {
      Run<T, 8, FAST> y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + i * NT, place = lo + u / W, r = place < hi ? s_row[place] : -1;
        y[i].load(element<T, FAST>(src, ldr, r < 0 ? any : r, (u % W) * 8));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) top.take(y[i]);
    }
    auto over_block = [&](float x) __attribute__((always_inline)) {
      x = wave_max_xor(x);
      if (lane == 0) s_max[wave] = x;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) x = fmaxf(x, s_max[w]);
      return x;
    };
    float mx = over_block(top.largest());
    const bool odd = mx == INFINITY;
    if (odd) {                             // once more, leaving out what is not finite
      __syncthreads();
      mx = 0.f;
      for (int u = tid; u < (hi - lo) * D; u += NT) {
        const int r = s_row[lo + u / D];
        if (r >= 0) mx = fmaxf(mx, finite_abs((float)*element<T, FAST>(src, ldr, r, u % D)));
      }
      mx = over_block(mx);
    }
    const float was = lo ? before : 0.f, fresh = fmaxf(mx, 1e-30f) / (CODE == INT8 ? 127.f : 448.f);
    const bool grown = lo && fresh > was;
    const float scale = lo && !grown ? was : fresh;
    const float inv = 1.0f / scale, ratio = grown ? was / scale : 1.0f;
    if (tid == 0) *scale_p = scale;                 // (every thread has read it: the barriers above)

    // Places that no row fills: in front of and between new tokens of a page that kept some, their codes stay (rounded again where
    // the scale rose); in a page that begins anew they become 0.
    auto write = [&](auto clean) __attribute__((always_inline)) {
      constexpr bool ODD = decltype(clean)::value;
      if (!part) {
        constexpr int C = D / 16;
        auto at = [&](int key, int c) { return reinterpret_cast<u32x4_t*>(codes + ((long)c * page + key) * 16); };
        for (int u0 = tid; u0 < (hi - lo) * C; u0 += 2 * NT) {
          Run<T, 16, FAST> y[2];
          int r[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int u = u0 + i * NT, key = lo + u / C;
            r[i] = key < hi ? s_row[key] : -1;
            y[i].load(element<T, FAST>(src, ldr, r[i] < 0 ? row : r[i], (u % C) * 16));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int u = u0 + i * NT;
            if (r[i] < 0) continue;
            u32x4_t w;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = encode4<CODE, ODD>(y[i].at(4 * e) * inv, y[i].at(4 * e + 1) * inv, y[i].at(4 * e + 2) * inv, y[i].at(4 * e + 3) * inv);
            *at(lo + u / C, u % C) = w;
          }
        }
        if (grown || (holes && !lo))
          for (int u = tid; u < hi * C; u += NT) {
            const int key = u / C;
            if (s_row[key] >= 0) continue;
            u32x4_t w = *at(key, u % C);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = grown ? recode4<CODE>(w[e], ratio) : zeros4<CODE>();
            *at(key, u % C) = w;
          }
      } else {
        constexpr int P = D / 2;
        const int t0 = lo >> 5, t1 = (hi + 31) >> 5;
        auto at = [&](int th, int d) { return reinterpret_cast<u32x4_t*>(codes + ((long)th * D + d) * 16); };
        for (int u = 2 * t0 * P + tid; u < 2 * t1 * P; u += NT) {
          const int th = u / P, d = 2 * (u % P);
          Run<T, 2, FAST> y[16];
          uint32_t fill[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int4 r = *reinterpret_cast<const int4*>(&s_row[(th >> 1) * 32 + 8 * m + 4 * (th & 1)]);
            fill[m] = (r.x >= 0 ? 0xffu : 0u) | (r.y >= 0 ? 0xff00u : 0u) | (r.z >= 0 ? 0xff0000u : 0u) | (r.w >= 0 ? 0xff000000u : 0u);
            y[4 * m].load(element<T, FAST>(src, ldr, r.x < 0 ? row : r.x, d));
            y[4 * m + 1].load(element<T, FAST>(src, ldr, r.y < 0 ? row : r.y, d));
            y[4 * m + 2].load(element<T, FAST>(src, ldr, r.z < 0 ? row : r.z, d));
            y[4 * m + 3].load(element<T, FAST>(src, ldr, r.w < 0 ? row : r.w, d));
          }
          u32x4_t w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
          if (lo && ((th >> 1) * 32 < lo || holes)) {
            w[0] = *at(th, d);
            w[1] = *at(th, d + 1);
          }
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int n = hi - ((th >> 1) * 32 + 8 * m + 4 * (th & 1));      // places below hi of these four
            const uint32_t below = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u, keep = lo ? below & ~fill[m] : 0u;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t now = encode4<CODE, ODD>(y[4 * m].at(k) * inv, y[4 * m + 1].at(k) * inv, y[4 * m + 2].at(k) * inv, y[4 * m + 3].at(k) * inv);
              const uint32_t kept = grown ? recode4<CODE>(w[k][m], ratio) : w[k][m];
              w[k][m] = (now & fill[m]) | (kept & keep) | (zeros4<CODE>() & ~(fill[m] | keep));
            }
          }
          *at(th, d) = w[0];
          *at(th, d + 1) = w[1];
        }
        if (grown)
          for (int u = tid; u < 2 * t0 * D; u += NT) {
            u32x4_t w = *at(u / D, u % D);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = recode4<CODE>(w[e], ratio);
            *at(u / D, u % D) = w;
          }
      }
    };
    if (odd) write(std::true_type());
    else write(std::false_type());
  }
}

// ----------------------------------------------------------------------------------------------------------------- gather
// One wave per (32 rows, head, keys or values).  Keys: D / 16 lanes per row, 16 dims each.  Values lie by tokens, so consecutive
// rows of one 32-token tile are read together: a lane takes two dims of half the tile, 32 bytes, and writes its tokens' pairs.
// Bound by the bytes: 40 k rows of 8 x 128 from e4m3 to bf16, 246 MB, 46 us, 5.3 TB/s (54 us with a row's heads in turn).
template <class T, int CODE, int D>
__global__ __launch_bounds__(64) void gather_kernel(rmem_bank8_gather_args a, int ps) {
  const rmem_bank8& b = a.bank;
  const int lane = threadIdx.x, h = blockIdx.y, part = blockIdx.z, page = b.page;
  const int row0 = blockIdx.x * 32, nr = min(32, a.rows - row0);
  int slot = -1;
  if (lane < nr) {
    slot = a.slots[row0 + lane];
    if (!in_pool(slot, b)) slot = -1;
  }
  const long pstride = (long)b.heads * page * D;
  float scale = 0.f;
  if (slot >= 0) scale = (part ? b.v_scale : b.k_scale)[(long)(slot >> ps) * b.heads + h];
  if (part == 0) {
    constexpr int C = D / 16, R = 64 / C, N = 32 / R;         // lanes per row, rows at once, steps
    const int c = lane % C;
    const uint8_t* codes = b.k + (long)h * page * D;
    u32x4_t w[N];
    float sc[N];
    int s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * R + lane / C;
      s[i] = __shfl(slot, r);
      sc[i] = __shfl(scale, r);
      w[i] = u32x4_t{0, 0, 0, 0};
      if (s[i] >= 0) w[i] = *reinterpret_cast<const u32x4_t*>(codes + (s[i] >> ps) * pstride + (c * page + (s[i] & (page - 1))) * 16);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * R + lane / C;
      if (r >= nr) continue;
      typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T vec_t;
      constexpr int V = 16 / sizeof(T);
      vec_t y[16 / V];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4_t x = values4<CODE>(w[i][e]) * sc[i];
#pragma unroll
        for (int f = 0; f < 4; ++f) y[(4 * e + f) / V][(4 * e + f) % V] = (T)(s[i] >= 0 ? x[f] : 0.f);
      }
      T* out = static_cast<T*>(a.ko) + ((long)(row0 + r) * b.heads + h) * D + c * 16;
#pragma unroll
      for (int k = 0; k < 16 / V; ++k) *reinterpret_cast<vec_t*>(out + k * V) = y[k];
    }
  } else {
    typedef __attribute__((ext_vector_type(2))) T pair_t;
    const int before = __shfl_up(slot, 1);
    const bool first = lane == 0 || slot < 0 || before < 0 || slot != before + 1 || (slot & 31) == 0;
    unsigned long long starts = __ballot(first && lane < nr);
    const uint8_t* codes = b.v + (long)h * page * D;
    T* out = static_cast<T*>(a.vo) + ((long)row0 * b.heads + h) * D;
    const long ldo = (long)b.heads * D;
    while (starts) {
      const int i0 = __builtin_ctzll(starts);
      starts &= starts - 1;
      const int i1 = starts ? __builtin_ctzll(starts) : nr;
      const int s = __builtin_amdgcn_readlane(slot, i0);
      const float sc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale), i0));
      if (s < 0) {                                            // (rows outside the pool are segments of one)
        for (int d = 2 * lane; d < D; d += 128) *reinterpret_cast<pair_t*>(out + i0 * ldo + d) = pair_t{(T)0.f, (T)0.f};
        continue;
      }
      const int key0 = s & 31;
      const uint8_t* tile = codes + (s >> ps) * pstride + (long)((s & (page - 1)) >> 5) * (32 * D);
#pragma unroll
      for (int u0 = 0; u0 < D; u0 += 64) {
        const int u = u0 + lane, half = u / (D / 2), d = 2 * (u % (D / 2));
        if (u >= D) break;
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(tile + (half * D + d) * 16);
        const u32x4_t w0 = p[0], w1 = p[1];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const f32x4_t x = values4<CODE>(w0[m]) * sc, y = values4<CODE>(w1[m]) * sc;
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const int r = i0 + 8 * m + 4 * half + f - key0;
            if (r >= i0 && r < i1) *reinterpret_cast<pair_t*>(out + r * ldo + d) = pair_t{(T)x[f], (T)y[f]};
          }
        }
      }
    }
  }
}

// kernels by type, code and dim
template <template <class, int, int> class F, class... A>
void dispatch(int type, int code, int dim, A&&... args) {
  auto dims = [&](auto t, auto c) {
    typedef decltype(t) T;
    constexpr int CODE = decltype(c)::value;
    if (dim == 32) F<T, CODE, 32>::run(args...);
    else if (dim == 64) F<T, CODE, 64>::run(args...);
    else F<T, CODE, 128>::run(args...);
  };
  auto codes = [&](auto t) { code == INT8 ? dims(t, std::integral_constant<int, INT8>()) : dims(t, std::integral_constant<int, E4M3>()); };
  if (type == FP32) codes(float());
  else if (type == FP16) codes((_Float16)0.f);
  else codes((__bf16)0.f);
}
template <class T, int CODE, int D>
struct Append {
  static void run(const rmem_bank8_append_args& a, const PageMark* marks, int ps, int window, hipStream_t s) {
    // FAST: every row of every head begins on 16 bytes, and the rows span less than 4 GiB
    const unsigned long mis = (unsigned long)a.k | (unsigned long)a.v | (unsigned long)((a.k_row | a.k_head | a.v_row | a.v_head) * (long)sizeof(T));
    // a window's heads follow each other, so that what runs at a time reads whole rows; values after all keys (13 k rows of 8 x 32: 12.2 us,
    // 12.7 head by head; 1000 single tokens of 8 x 128: 48 us, 55 with a window's keys and values side by side)
    const int windows = (a.rows + window - 1) / window;
    const dim3 grid(a.bank.heads, std::min(windows, GRID_Y), 2 * ((windows + GRID_Y - 1) / GRID_Y));
    const long span = (a.rows - 1L) * std::max(a.k_row, a.v_row) + D;
    // Up to SCAN_ROWS rows most pages get a token or a few: workgroups of 128 keep more of their chains of reads in flight (1000
    // single tokens: 48 us, 71 with 256); long calls fill whole pages, which 256 write faster (25 k tokens into pages of 128: 45, 52).
    if ((mis & 15) || span * (long)sizeof(T) >= 1L << 32) hipLaunchKernelGGL((append_kernel<T, CODE, D, false, 128>), grid, dim3(128), 0, s, a, marks, ps, window);
    else if (!marks) hipLaunchKernelGGL((append_kernel<T, CODE, D, true, 128>), grid, dim3(128), 0, s, a, marks, ps, window);
    else hipLaunchKernelGGL((append_kernel<T, CODE, D, true, 256>), grid, dim3(256), 0, s, a, marks, ps, window);
  }
};
template <class T, int CODE, int D>
struct Gather {
  static void run(const rmem_bank8_gather_args& a, int ps, hipStream_t s) {
    hipLaunchKernelGGL((gather_kernel<T, CODE, D>), dim3((a.rows + 31) / 32, a.bank.heads, 2), dim3(64), 0, s, a, ps);
  }
};

}  // namespace

extern "C" int rmem_bank8_plan(const rmem_bank8_plan_args* a, void* stream) {
  if (!a || a->reqs <= 0 || !a->ctx || !a->add || !a->table || a->cols <= 0 || a->ld_table < a->cols || !a->free_ring || a->ring <= 0 ||
      !a->state_in || !a->state_out || !a->cu || !a->lens || !a->start || !a->status || a->rows < 0 || (a->rows && !a->slots) ||
      (a->page != 32 && a->page != 64 && a->page != 128) || (int64_t)a->cols * a->page > 0x7fffffff)
    return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int ps = log2_of(a->page);
  // as many threads as the requests, or a quarter of the rows, can use: a step of few requests is one wave and no barrier's wait
  const int use = std::max(a->reqs, a->rows <= SLOTS_INLINE ? a->rows / 4 : PT), threads = use >= PT ? PT : use <= 64 ? 64 : (use + 63) & ~63;
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(threads), 0, s, *a, ps);
  RMEM_CHECK_LAUNCH();
  if (a->rows > SLOTS_INLINE) {
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)(((long)a->rows + 255) / 256)), dim3(256), 0, s, *a, ps);
    RMEM_CHECK_LAUNCH();
  }
  return RMEM_OK;
}

static bool valid_append(const rmem_bank8_append_args* a) {
  return a && valid_bank(&a->bank) && valid_type(a->type) && a->rows >= 0 && a->rows < 1 << 24 && a->bank.heads <= 65535 && a->k_row >= 0 &&
         a->k_head >= 0 && a->v_row >= 0 && a->v_head >= 0;
}

extern "C" int64_t rmem_bank8_append_workspace(const rmem_bank8_append_args* a) {
  if (!valid_append(a)) return -1;
  return a->rows > SCAN_ROWS ? (int64_t)sizeof(PageMark) * a->bank.pages : 0;
}

extern "C" int rmem_bank8_append(const rmem_bank8_append_args* a, void* stream) {
  if (!valid_append(a)) return RMEM_ERR_INVALID;
  if (a->rows == 0) return RMEM_OK;
  const int64_t need = rmem_bank8_append_workspace(a);
  if (!a->k || !a->v || !a->slots || (need && (!a->workspace || ((uintptr_t)a->workspace % 16) || a->workspace_bytes < need)))
    return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int ps = log2_of(a->bank.page);
  PageMark* marks = need ? static_cast<PageMark*>(a->workspace) : nullptr;
  if (marks) {
    const dim3 grid((a->rows + 255) / 256);
    hipLaunchKernelGGL(mark_clear_kernel, grid, dim3(256), 0, s, *a, marks, ps);
    RMEM_CHECK_LAUNCH();
    hipLaunchKernelGGL(mark_kernel, grid, dim3(256), 0, s, *a, marks, ps);
    RMEM_CHECK_LAUNCH();
  }
  // rows of a workgroup: one while that leaves the chip room (a step of single tokens), up to 64 of a long call's, most of whose
  // rows begin no page (25 k rows of prompts: 58 us with up to 32, 48 us with up to 64)
  const long groups = (long)a->rows * a->bank.heads * 2;
  const int window = groups <= APPEND_GROUPS ? 1 : groups >= 64L * APPEND_GROUPS ? 64 : (int)((groups + APPEND_GROUPS - 1) / APPEND_GROUPS);
  dispatch<Append>(a->type, a->bank.code, a->bank.dim, *a, marks, ps, window, s);
  RMEM_CHECK_LAUNCH();
  return RMEM_OK;
}

extern "C" int rmem_bank8_gather(const rmem_bank8_gather_args* a, void* stream) {
  if (!a || !valid_bank(&a->bank) || !valid_type(a->type) || a->rows < 0 || a->rows >= 1 << 30 || a->bank.heads > 65535) return RMEM_ERR_INVALID;
  if (a->rows == 0) return RMEM_OK;
  if (!a->slots || !a->ko || !a->vo || ((uintptr_t)a->ko % 16) || ((uintptr_t)a->vo % 16)) return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  dispatch<Gather>(a->type, a->bank.code, a->bank.dim, *a, log2_of(a->bank.page), s);
  RMEM_CHECK_LAUNCH();
  return RMEM_OK;
}
