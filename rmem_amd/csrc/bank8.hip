// bank8.hip -- the paged 8-bit bank: block tables and slot maps (plan), writing tokens (append), reading them back (gather).
// Storage and semantics: include/rmem_hip.h and bank8.h; the read over the pages is bank8_attn.hip.
#include "bank8.h"

using namespace bank8;

namespace {

// ------------------------------------------------------------------------------------------------------------------- plan
// One workgroup: the requests are scanned (pages asked for, rows, pages going back) a chunk of 1024 at a time, the page ids that
// move are spread over the threads by binary search in the scan.  Bound by the chain of dependent memory reads (lengths -> ring
// and table entries), not by bytes; one workgroup keeps it one launch and lets state and lengths be updated in place.
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
  const int page_mask = (1 << ps) - 1;
  int head = p.state_in[0], count = p.state_in[1];
  head = p.ring > 0 ? (int)(((long long)head % p.ring + p.ring) % p.ring) : 0;
  count = count < 0 ? 0 : count > p.ring ? p.ring : count;
  long long c_need = 0, c_rows = 0, c_back = 0;              // carried from earlier chunks
  long long taken = 0, missing = 0;                          // this thread's requests
  const bool inline_slots = p.rows <= SLOTS_INLINE;
  for (int base = 0; base < p.reqs; base += PT) {
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
    const int nr = p.reqs - base < PT ? p.reqs - base : PT;
    const long long n_need = s_need[nr - 1], n_rows = s_rows[nr - 1], n_back = s_back[nr - 1];
    // pages going back, before new entries can overwrite them in the table
    for (long long i = tid; i < n_back; i += PT) {
      const int k = upper_bound(s_back, nr, i);
      const long long j = i - (k ? s_back[k - 1] : 0);
      const long long at = count + c_back + i;
      if (at < p.ring)                                       // (more pages than the ring holds: returned twice, dropped)
        p.free_ring[(head + at) % p.ring] = p.table[(base + k) * p.ld_table + s_held[k] + j];
    }
    if (n_back) __syncthreads();
    for (long long i = tid; i < n_need; i += PT) {
      const int k = upper_bound(s_need, nr, i);
      const long long j = i - (k ? s_need[k - 1] : 0);
      if (s_start[k] >= 0) p.table[(base + k) * p.ld_table + s_held[k] + j] = p.free_ring[(head + c_need + i) % p.ring];
    }
    if (inline_slots) {
      // rows of this chunk; entries are taken from where they come from, so nothing waits for the table's writes
      const long long end = c_rows + n_rows < p.rows ? c_rows + n_rows : p.rows;
      for (long long t = c_rows + tid; t < end; t += PT) {
        const int k = upper_bound(s_rows, nr, t - c_rows);
        const int start = s_start[k];
        int slot = -1;
        if (start >= 0) {
          const long long pos = start + (t - c_rows) - (k ? s_rows[k - 1] : 0);
          const long long pi = pos >> ps;
          const int id = pi >= s_held[k] ? p.free_ring[(head + c_need + (k ? s_need[k - 1] : 0) + pi - s_held[k]) % p.ring]
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
    for (long long t = c_rows + tid; t < p.rows; t += PT) p.slots[t] = -1;
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
    for (int w = 0; w < PT / 64; ++w) {
      t += s_wave[0][w];
      m += s_wave[1][w];
    }
    const long long left = count - t + c_back;
    p.state_out[0] = p.ring > 0 ? (int)((head + t) % p.ring) : 0;
    p.state_out[1] = (int)(left < p.ring ? left : p.ring);
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
  if (!in_pool(slot, a.bank)) return;
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

// One workgroup per (row, head, keys or values).
__global__ __launch_bounds__(256) void append_kernel(rmem_bank8_append_args a, const PageMark* marks, int ps) {
  __shared__ float s_max[4];
  __shared__ int s_row[128];              // row that fills each place of the page, -1: none; the last of several
  __shared__ int s_end[2];                // one past the last place filled, and the complement of the first
  __shared__ int s_other;
  const int row = blockIdx.x, h = blockIdx.y, part = blockIdx.z;
  const rmem_bank8& b = a.bank;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int page = b.page, dim = b.dim, code = b.code;
  const int slot = a.slots[row];
  if (!in_pool(slot, b) || goes_on(a.slots, row, slot, page)) return;
  const int pg32 = slot >> ps;
  int runs = 0;
  if (marks) {
    if (marks[pg32].first != row) return;
    runs = marks[pg32].runs;
  }
  if (tid < 128) s_row[tid] = -1;
  if (tid < 2) s_end[tid] = 0;
  if (tid == 0) s_other = 0;
  __syncthreads();
  if (runs == 1) {
    const long r = (long)row + tid;
    const int at = (slot & (page - 1)) + tid;
    if (at < page && r < a.rows) {
      // the run ends where the slots do not go on: later rows that fit the pattern again would be a second run
      if (a.slots[r] == slot + tid) s_row[at] = (int)r;
    }
  } else {
    for (int r = marks ? row + tid : tid; r < a.rows; r += 256) {
      const int s = a.slots[r];
      if (s < 0 || (s >> ps) != pg32) continue;
      if (r < row) s_other = 1;
      else atomicMax(&s_row[s & (page - 1)], r);
    }
  }
  __syncthreads();
  if (s_other) return;
  if (tid < page && s_row[tid] >= 0) {
    atomicMax(&s_end[0], tid + 1);
    atomicMax(&s_end[1], 128 - tid);
  }
  __syncthreads();
  const int hi = s_end[0], lo = 128 - s_end[1];

  const long pg = pg32;
  const void* src = part ? a.v : a.k;
  const long ldr = part ? a.v_row : a.k_row, base = (long)h * (part ? a.v_head : a.k_head);
  uint8_t* codes = (part ? b.v : b.k) + (pg * b.heads + h) * ((long)page * dim);
  float* scale_p = (part ? b.v_scale : b.k_scale) + pg * b.heads + h;

  float mx = 0.f;
  for (int i = tid; i < (hi - lo) * dim; i += 256) {
    const int r = s_row[lo + i / dim];
    if (r >= 0) mx = fmaxf(mx, finite_abs(load1(src, base + r * ldr + i % dim, a.type)));
  }
  mx = wave_max_xor(mx);
  if (lane == 0) s_max[wave] = mx;
  const float was = lo ? *scale_p : 0.f;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  const float fresh = fmaxf(mx, 1e-30f) / code_top(code);
  const bool grown = lo && fresh > was;
  const float scale = lo && !grown ? was : fresh;
  const float inv = 1.0f / scale, ratio = grown ? was / scale : 1.0f;
  if (tid == 0) *scale_p = scale;                             // (every thread has read it: the barrier above)

  // Places that no row fills: in front of and between new tokens of a page that kept some, their codes stay (rounded again where
  // the scale rose); in a page that begins anew they become 0.
  if (!part) {
    // unit: 16 dims of a token
    const int first = grown ? 0 : lo, n = hi - first;
    for (int i = tid; i < n * (dim / 16); i += 256) {
      const int key = first + i % n, c = i / n, r = s_row[key];
      if (r < 0 && lo && !grown) continue;
      u32x4_t* dst = reinterpret_cast<u32x4_t*>(codes + ((long)c * page + key) * 16);
      u32x4_t w;
      if (r >= 0) {
        const long at = base + r * ldr + c * 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t u = 0;
#pragma unroll
          for (int f = 0; f < 4; ++f) u |= encode1(load1(src, at + 4 * e + f, a.type) * inv, code) << (8 * f);
          w[e] = u;
        }
      } else if (lo) {
        w = *dst;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t u = 0;
#pragma unroll
          for (int f = 0; f < 4; ++f) u |= encode1(decode1((w[e] >> (8 * f)) & 0xff, code) * ratio, code) << (8 * f);
          w[e] = u;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = 0x01010101u * zero_code(code);
      }
      *dst = w;
    }
  } else {
    // unit: 16 tokens of a dim (half a 32-token tile)
    const int t0 = grown ? 0 : lo >> 5, t1 = (hi + 31) >> 5;
    for (int i = tid; i < (t1 - t0) * 2 * dim; i += 256) {
      const int d = i % dim, th = i / dim, tile = t0 + (th >> 1), half = th & 1;
      u32x4_t* dst = reinterpret_cast<u32x4_t*>(codes + (((long)tile * 2 + half) * dim + d) * 16);
      u32x4_t w = *dst;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        uint32_t u = 0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int key = tile * 32 + 8 * m + 4 * half + f, r = s_row[key];
          uint32_t x = (w[m] >> (8 * f)) & 0xff;
          if (r >= 0) x = encode1(load1(src, base + r * ldr + d, a.type) * inv, code);
          else if (key >= hi || !lo) x = zero_code(code);
          else if (grown) x = encode1(decode1(x, code) * ratio, code);
          u |= x << (8 * f);
        }
        w[m] = u;
      }
      *dst = w;
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------- gather
// One thread: 16 dims of a (row, head), keys and values.
__global__ __launch_bounds__(256) void gather_kernel(rmem_bank8_gather_args a, int ps) {
  const rmem_bank8& b = a.bank;
  const int chunks = b.dim / 16;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)a.rows * b.heads * chunks) return;
  const int c = (int)(i % chunks), h = (int)(i / chunks % b.heads);
  const long row = i / chunks / b.heads;
  const int slot = a.slots[row];
  const bool in = slot >= 0 && slot < b.pages * (long)b.page;
  const long pg = in ? slot >> ps : 0, at = pg * b.heads + h;
  const int key = in ? slot & (b.page - 1) : 0, q = key & 31;
  const float ks = in ? b.k_scale[at] : 0.f, vs = in ? b.v_scale[at] : 0.f;
  const uint8_t* k = b.k + at * ((long)b.page * b.dim) + ((long)c * b.page + key) * 16;
  const uint8_t* v = b.v + at * ((long)b.page * b.dim) + (((long)(key >> 5) * 2 + ((q >> 2) & 1)) * b.dim + c * 16) * 16 + 4 * (q >> 3) + (q & 3);
  const long o = i * 16;
  for (int e = 0; e < 16; ++e) {
    store1(a.ko, o + e, in ? decode1(k[e], b.code) * ks : 0.f, a.type);
    store1(a.vo, o + e, in ? decode1(v[e * 16], b.code) * vs : 0.f, a.type);
  }
}

}  // namespace

extern "C" int rmem_bank8_plan(const rmem_bank8_plan_args* a, void* stream) {
  if (!a || a->reqs <= 0 || !a->ctx || !a->add || !a->table || a->cols <= 0 || a->ld_table < a->cols || !a->free_ring || a->ring <= 0 ||
      !a->state_in || !a->state_out || !a->cu || !a->lens || !a->start || !a->status || a->rows < 0 || (a->rows && !a->slots) ||
      (a->page != 32 && a->page != 64 && a->page != 128) || (int64_t)a->cols * a->page > 0x7fffffff)
    return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int ps = log2_of(a->page);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(PT), 0, s, *a, ps);
  RMEM_CHECK_LAUNCH();
  if (a->rows > SLOTS_INLINE) {
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)(((long)a->rows + 255) / 256)), dim3(256), 0, s, *a, ps);
    RMEM_CHECK_LAUNCH();
  }
  return RMEM_OK;
}

static bool valid_append(const rmem_bank8_append_args* a) {
  return a && valid_bank(&a->bank) && valid_type(a->type) && a->rows >= 0 && a->rows < 1 << 24 && a->bank.heads <= 65535;
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
  hipLaunchKernelGGL(append_kernel, dim3(a->rows, a->bank.heads, 2), dim3(256), 0, s, *a, marks, ps);
  RMEM_CHECK_LAUNCH();
  return RMEM_OK;
}

extern "C" int rmem_bank8_gather(const rmem_bank8_gather_args* a, void* stream) {
  if (!a || !valid_bank(&a->bank) || !valid_type(a->type) || a->rows < 0) return RMEM_ERR_INVALID;
  if (a->rows == 0) return RMEM_OK;
  if (!a->slots || !a->ko || !a->vo || ((uintptr_t)a->ko % 16) || ((uintptr_t)a->vo % 16)) return RMEM_ERR_INVALID;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const long units = (long)a->rows * a->bank.heads * (a->bank.dim / 16), blocks = (units + 255) / 256;
  if (blocks >= 1 << 24) return RMEM_ERR_INVALID;
  hipLaunchKernelGGL(gather_kernel, dim3((unsigned)blocks), dim3(256), 0, s, *a, log2_of(a->bank.page));
  RMEM_CHECK_LAUNCH();
  return RMEM_OK;
}
