// tg_paged.cu -- kernels over a paged KV cache: keys and values appended with
// the position rotation applied on the way, decode attention through a block
// table (dense, or over listed pages), and the selection of pages by a bound
// on their scores.
//
// The reference keeps one contiguous [pos][n_kv*head_dim] cache per layer
// (g_k_cache / g_v_cache, tmac_gguf.cpp:200-201) and has no counterpart of
// any of these; the rotation is its apply_rope (tmac_gguf.cpp:990-1016) and
// the attention its GQA block (tmac_gguf.cpp:1093-1128).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tg_device.cuh"
#include "tg_launch.cuh"
#include "tg_paged.h"
#include "tg_shared.h"

namespace tg {

// ------------------------------------------------------------ append

// U consecutive elements of a row (2 or 4: one or two rotation pairs).
template <int U>
struct Unit {
  float x[U];
};

template <int U>
__device__ __forceinline__ Unit<U> load_unit(const float* p) {
  Unit<U> r;
  if constexpr (U == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    r.x[0] = a.x; r.x[1] = a.y; r.x[2] = a.z; r.x[3] = a.w;
  } else {
    const float2 a = *reinterpret_cast<const float2*>(p);
    r.x[0] = a.x; r.x[1] = a.y;
  }
  return r;
}

template <int U>
__device__ __forceinline__ Unit<U> load_unit(const __nv_bfloat16* p) {
  Unit<U> r;
#pragma unroll
  for (int i = 0; i < U; i += 2) {
    const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(p + i);
    r.x[i] = __low2float(b);
    r.x[i + 1] = __high2float(b);
  }
  return r;
}

template <int U>
__device__ __forceinline__ void store_unit(float* p, const Unit<U>& r) {
  if constexpr (U == 4)
    *reinterpret_cast<float4*>(p) = make_float4(r.x[0], r.x[1], r.x[2], r.x[3]);
  else
    *reinterpret_cast<float2*>(p) = make_float2(r.x[0], r.x[1]);
}

template <int U>
__device__ __forceinline__ void store_unit(__nv_bfloat16* p, const Unit<U>& r) {
  if constexpr (U == 4) {
    *reinterpret_cast<uint2*>(p) =
        make_uint2(pack_bf16x2(r.x[0], r.x[1]), pack_bf16x2(r.x[2], r.x[3]));
  } else {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(r.x[0], r.x[1]);
  }
}

// x0*c - x1*s, x0*s + x1*c with one rounding per product and sum
// (tmac_gguf.cpp:999-1000 without contraction).
template <int U>
__device__ __forceinline__ Unit<U> rotate_unit(const Unit<U>& v, const Unit<U>& cs) {
  Unit<U> r;
#pragma unroll
  for (int i = 0; i < U; i += 2) {
    r.x[i] = __fsub_rn(__fmul_rn(v.x[i], cs.x[i]), __fmul_rn(v.x[i + 1], cs.x[i + 1]));
    r.x[i + 1] = __fadd_rn(__fmul_rn(v.x[i], cs.x[i + 1]), __fmul_rn(v.x[i + 1], cs.x[i]));
  }
  return r;
}

// The value as the pool holds it (fp32, or rounded to nearest even bf16).
template <typename T>
__device__ __forceinline__ float as_stored(float v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(v));
  return v;
}

constexpr int kAppendWarps = 8;
constexpr int kAppendBatch = 8;  // loads a lane has in flight

// Whether table row i has tokens of this call on page `page`, which is entry j
// of some other row: its tokens on it are then [a, b) of its own, the first of
// them at row r0 of the page.
struct PageTokens {
  int a, b, r0;
};

__device__ __forceinline__ PageTokens tokens_on_page(const PagedAppendParams& p, int i, int j,
                                                     int page) {
  PageTokens x{0, 0, 0};
  const int pos0 = p.pos0[i];
  const int first = p.cu ? p.cu[i] : i, last = p.cu ? min(p.cu[i + 1], p.n_tokens) : i + 1;
  const long long lo = (long long)j << p.log2p, hi = min(lo + (1ll << p.log2p), (long long)p.table_len);
  const long long end = min((long long)pos0 + (last - first), hi);
  if (pos0 < 0 || pos0 >= hi || end <= lo || last <= first) return x;
  if (p.table[(size_t)i * p.max_blocks + j] != page) return x;
  const long long from = max((long long)pos0, lo);
  x.a = first + (int)(from - pos0);
  x.b = first + (int)(end - pos0);
  x.r0 = (int)(from - lo);
  return x;
}

// Bounds over one row more.  A NaN stays (fminf and fmaxf would drop it, and
// the page would rank by its other rows).
template <int U>
__device__ __forceinline__ void extend(Unit<U>& lo, Unit<U>& hi, const Unit<U>& x) {
#pragma unroll
  for (int e = 0; e < U; ++e) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo.x[e]) : "f"(x.x[e]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi.x[e]) : "f"(x.x[e]));
  }
}

// A new key as the pool holds it.
template <typename T, int U>
__device__ __forceinline__ Unit<U> new_row(const float* k, const float* cs) {
  Unit<U> x = rotate_unit<U>(load_unit<U>(k), load_unit<U>(cs));
#pragma unroll
  for (int e = 0; e < U; ++e) x.x[e] = as_stored<T>(x.x[e]);
  return x;
}

// The bounds of a page that row s and rows behind it write: row s's tokens
// [t, t_end) from position pos on, the others' found by looking at all rows
// behind it.  src: the token of each row of the page, -1 where it is in the
// pool.  By one warp.
template <typename T, int U>
__device__ __forceinline__ void bounds_of_rows(const PagedAppendParams& p, int s, int t, int t_end,
                                            int pos, int page, int* src) {
  const int lane = threadIdx.x & 31, hd = p.hd, row = p.n_kv * hd, P = 1 << p.log2p;
  const int slot = pos & (P - 1);
  int end = slot + (t_end - t);
  for (int r = lane; r < P; r += 32) src[r] = r >= slot && r < end ? t + (r - slot) : -1;
  __syncwarp();
  for (int i = s + 1 + lane; i < p.n_seqs; i += 32) {
    const PageTokens x = tokens_on_page(p, i, pos >> p.log2p, page);
    for (int a = x.a; a < x.b; ++a) atomicMax(&src[x.r0 + (a - x.a)], a);
    if (x.b > x.a) end = max(end, x.r0 + (x.b - x.a));
  }
  end = __reduce_max_sync(0xffffffffu, end);
  __syncwarp();
  const size_t base = (size_t)page * p.n_kv;
  T* bounds = static_cast<T*>(p.bounds);
  for (int i = lane * U; i < row; i += 32 * U) {
    const int g = i / hd, d = i - g * hd;
    Unit<U> lo, hi;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      lo.x[e] = INFINITY;
      hi.x[e] = -INFINITY;
    }
    const T* old = static_cast<const T*>(p.kp) + ((base + g) << p.log2p) * hd + d;
    for (int r = 0; r < end; ++r)
      extend(lo, hi, src[r] < 0 ? load_unit<U>(old + (size_t)r * hd)
                                : new_row<T, U>(p.k + (size_t)src[r] * row + i,
                                                p.cs + (size_t)(pos - slot + r) * hd + d));
    store_unit<U>(bounds + (base + g) * 2 * hd + d, lo);
    store_unit<U>(bounds + ((base + g) * 2 + 1) * hd + d, hi);
  }
}

// The page of a table row's first or last token of this call, -1 for none.
// Two rows that write one page both end on it: a row that writes all of a page
// leaves no position for another.  x counts rows, or with cu their ends.
__device__ __forceinline__ int end_page(const PagedAppendParams& p, int x) {
  const int i = p.cu ? x >> 1 : x, pos0 = p.pos0[i];
  const int limit = min(p.table_len, p.max_blocks << p.log2p);
  int n = 1;
  if (p.cu) n = min(p.cu[i + 1], p.n_tokens) - p.cu[i];
  if (n <= 0 || pos0 < 0 || pos0 >= limit) return -1;
  const int pos = p.cu && (x & 1) ? (int)min((long long)pos0 + n, (long long)limit) - 1 : pos0;
  return p.table[(size_t)i * p.max_blocks + (pos >> p.log2p)];
}

// One warp per token: its q row rotated, its k row rotated and written with
// its v row to the page of its position.  The warp of the first new token of
// a page also writes the page's bounds: min and max over the page's rows up
// to the last one of this call, the earlier rows from the pool and the new
// ones rotated again from k (the few extra reads come from L2), so that no
// warp waits for another and the bounds are the same however the rows were
// cut into calls.  Where several table rows write one page (tokens of one
// sequence as rows of their own), the first of them forms the bounds over the
// tokens of all: a warp that read the pool for a row that another warp of the
// launch writes would race with it.
template <typename T, int U>
__global__ void __launch_bounds__(32 * kAppendWarps, 4) paged_append_kernel(const PagedAppendParams p) {
  __shared__ int seq_of[kAppendWarps];
  __shared__ int open_page[kAppendWarps], open_seq[kAppendWarps];
  __shared__ int twins_of[kAppendWarps];
  __shared__ int source[kAppendWarps][kPagedMaxPage];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * kAppendWarps, t = t0 + warp;
  // Pages that the table rows end on, for the look at shared pages below: on
  // their way before anything waits.  Few are looked at by every warp for
  // itself, many by the CTA together.  The look costs 0.4 us of a step of 64
  // tokens (5.1 us in a graph without it) and of 16000 tokens of 16 prompts
  // (28.9 us), 2 us of a step of 1024 (5.8 us); with the loads behind those of
  // the token's own page it was 1.4, 1.5 and 6 us.
  constexpr int kAhead = 2;
  const int n_ends = !p.bounds ? 0 : p.cu ? 2 * p.n_seqs : p.n_seqs;
  const bool few = n_ends <= 32 * kAhead;   // every warp looks for itself
  int ends[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int x = few ? lane + 32 * u : threadIdx.x + 32 * kAppendWarps * u;
    ends[u] = x < n_ends ? end_page(p, x) : -1;
  }
  int s = -1;
  if (p.cu) {
    // The sequences of this CTA's tokens: every thread looks at some of the
    // sequences (one round of loads; a search would be a chain of them).
    if (threadIdx.x < kAppendWarps) seq_of[threadIdx.x] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < p.n_seqs; i += 32 * kAppendWarps) {
      const int lo = max(p.cu[i], t0), hi = min(p.cu[i + 1], t0 + kAppendWarps);
      for (int x = lo; x < hi; ++x) seq_of[x - t0] = i;
    }
    __syncthreads();
    s = seq_of[warp];
  } else if (t < p.n_seqs) {
    s = t;
  }
  const int P = 1 << p.log2p, hd = p.hd;
  bool live = t < p.n_tokens && s >= 0;   // padding tokens stay as they are
  int first = 0, last = 0, pos = 0, slot = 0, page = 0;
  if (live) {
    first = p.cu ? p.cu[s] : t;
    last = p.cu ? min(p.cu[s + 1], p.n_tokens) : t + 1;
    const long long pos_ll = (long long)p.pos0[s] + (t - first);
    if (p.pos0[s] < 0 || pos_ll >= p.table_len || (pos_ll >> p.log2p) >= p.max_blocks) {
      if (lane == 0) record_error(p.err, kDevErrBadPos);
      live = false;
    } else {
      pos = (int)pos_ll;
      slot = pos & (P - 1);
      page = p.table[(size_t)s * p.max_blocks + (pos >> p.log2p)];
      if (page < 0 || page >= p.n_pages) {
        if (lane == 0) record_error(p.err, kDevErrBadPage);
        live = false;
      }
    }
  }
  // The pages that this CTA opens, looked for among all table rows.
  const bool opens = live && p.bounds && (t == first || slot == 0);
  unsigned twins = 0;   // table rows that share the page: 1 before this one, 2 behind it
  if (few) {
    if (opens) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int x = lane + 32 * u, i = p.cu ? x >> 1 : x;
        if (ends[u] == page && i != s) twins |= i < s ? 1 : 2;
      }
      twins = __reduce_or_sync(0xffffffffu, twins);
    }
  } else {
    if (lane == 0) {
      open_page[warp] = opens ? page : -2;
      open_seq[warp] = s;
      twins_of[warp] = 0;
    }
    if (__syncthreads_or(opens)) {
      int open[kAppendWarps];
#pragma unroll
      for (int w = 0; w < kAppendWarps; ++w) open[w] = open_page[w];
      auto look = [&](int x, int end) {
        unsigned hits = 0;
#pragma unroll
        for (int w = 0; w < kAppendWarps; ++w) hits |= open[w] == end ? 1u << w : 0u;
        const int i = p.cu ? x >> 1 : x;
        for (; hits; hits &= hits - 1) {   // seldom: rows of this CTA, and twins
          const int w = __ffs(hits) - 1;
          if (open_seq[w] != i) atomicOr(&twins_of[w], i < open_seq[w] ? 1 : 2);
        }
      };
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (ends[u] >= 0) look(threadIdx.x + 32 * kAppendWarps * u, ends[u]);
#pragma unroll 4
      for (int x = threadIdx.x + 32 * kAppendWarps * kAhead; x < n_ends; x += 32 * kAppendWarps)
        look(x, end_page(p, x));
      __syncthreads();
      twins = twins_of[warp];
    }
  }
  if (!live) return;
  const float* cs = p.cs + (size_t)pos * hd;
  if (p.q) {
    const int nq = p.n_head * hd;
    const float* q = p.q + (size_t)t * nq;
    float* qo = p.q_out + (size_t)t * nq;
    for (int i0 = lane * U; i0 < nq; i0 += kAppendBatch * 32 * U) {
      Unit<U> x[kAppendBatch];
#pragma unroll
      for (int u = 0; u < kAppendBatch; ++u) {
        const int i = i0 + u * 32 * U;
        if (i < nq) x[u] = load_unit<U>(q + i);
      }
#pragma unroll
      for (int u = 0; u < kAppendBatch; ++u) {
        const int i = i0 + u * 32 * U;
        if (i < nq) store_unit<U>(qo + i, rotate_unit<U>(x[u], load_unit<U>(cs + i % hd)));
      }
    }
  }
  const int row = p.n_kv * hd;
  const float* k = p.k + (size_t)t * row;
  const float* v = p.v + (size_t)t * row;
  T* kp = static_cast<T*>(p.kp);
  T* vp = static_cast<T*>(p.vp);
  const size_t base = (size_t)page * p.n_kv;
  for (int i = lane * U; i < row; i += 32 * U) {
    const int g = i / hd, d = i - g * hd;
    const Unit<U> xk = load_unit<U>(k + i), xv = load_unit<U>(v + i), c = load_unit<U>(cs + d);
    const size_t at = (((base + g) << p.log2p) + slot) * hd + d;
    store_unit<U>(kp + at, rotate_unit<U>(xk, c));
    store_unit<U>(vp + at, xv);
  }
  if (!opens || (twins & 1)) return;
  if (twins) {
    bounds_of_rows<T, U>(p, s, t, t + min(last - t, min(P - slot, p.table_len - pos)), pos, page,
                         source[warp]);
    return;
  }
  // Rows [0, slot) of the page from the pool, [slot, end) from k.
  const int end = min(min(P, slot + (last - t)), slot + (p.table_len - pos));
  T* bounds = static_cast<T*>(p.bounds);
  for (int i = lane * U; i < row; i += 32 * U) {
    const int g = i / hd, d = i - g * hd;
    Unit<U> lo, hi;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      lo.x[e] = INFINITY;
      hi.x[e] = -INFINITY;
    }
    const T* old = kp + ((base + g) << p.log2p) * hd + d;
#pragma unroll 8
    for (int r = 0; r < slot; ++r) extend(lo, hi, load_unit<U>(old + (size_t)r * hd));
#pragma unroll 4
    for (int r = slot; r < end; ++r)
      extend(lo, hi, new_row<T, U>(k + (size_t)(r - slot) * row + i, cs + (size_t)(r - slot) * hd + d));
    store_unit<U>(bounds + (base + g) * 2 * hd + d, lo);
    store_unit<U>(bounds + ((base + g) * 2 + 1) * hd + d, hi);
  }
}

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.n_tokens + kAppendWarps - 1) / kAppendWarps)), block(32 * kAppendWarps);
  if (p.dtype == 1)
    return p.vec4 ? launch_chained(paged_append_kernel<__nv_bfloat16, 4>, grid, block, 0, st, p)
                  : launch_chained(paged_append_kernel<__nv_bfloat16, 2>, grid, block, 0, st, p);
  return p.vec4 ? launch_chained(paged_append_kernel<float, 4>, grid, block, 0, st, p)
                : launch_chained(paged_append_kernel<float, 2>, grid, block, 0, st, p);
}

// ------------------------------------------------------------ the schedule

// Pages that query i attends (before listing); a position outside the table
// counts as none and is reported.
__device__ __forceinline__ int query_blocks(const PagedAttnParams& p, int past, bool report) {
  if (past < 0) {
    if (past < -1 && report) record_error(p.err, kDevErrBadPos);
    return 0;
  }
  const int nb = (past >> p.log2p) + 1;
  if (nb > p.max_blocks) {
    if (report) record_error(p.err, kDevErrBadPos);
    return 0;
  }
  return nb;
}

// (Positions fit 31 bits, so 32 do for rows below.)
// First table entry of a query's list: those before it are attended elsewhere
// by the queries that attend all of them.
__device__ __forceinline__ int query_skip(const PagedAttnParams& p, int past) {
  return (unsigned)past + 1u >= (unsigned)p.skip << p.log2p ? p.skip : 0;
}

__device__ __forceinline__ int query_chunks(const PagedAttnParams& p, int past, int nb) {
  const int list = p.sel ? min(p.n_sel, nb) : nb - min(nb, query_skip(p, past));
  return (int)((((unsigned)list << p.log2p) + (1u << p.lchunk) - 1u) >> p.lchunk);
}

// CTAs that share the T chunks out: enough that each has a chunk for each of
// its warps, and in any case some for every stream.
__device__ __forceinline__ int paged_active(int grid, int T, int warps, int n_streams) {
  return min(min(grid, T), max((T + warps - 1) / warps, 3 * n_streams));
}

// A CTA's range is an equal share of the T chunks, its ends moved to the
// nearer end of the stream that they would cut if that stream is short
// (kWholeRounds steps of all warps or less).  A cut costs its two CTAs a
// record, an arrival and a merge, about 5000 cycles, as much as the chunks
// that a moved range has too many.  A range may be empty.  Measured with 0, 2,
// 4 and 8 rounds (us): 64 fp32 sequences of up to 256 rows 15.0, 10.7, 10.7,
// 10.7; 64 queries over 64 listed pages of 16 rows 16.2, 16.2, 13.6, 13.6; a
// batch of middling lengths 41.5, 41.5, 41.5, 45.1.
constexpr int kWholeRounds = 4;

struct PagedRange {
  int T, G;       // chunks of all streams, CTAs that share them
  int lo, hi;     // this CTA's chunks
  int s;          // a query at or before the one of chunk lo
};

// The schedule of a launch, in shared memory: prefix[s], the chunks of one
// stream of each query before s, and the queries' last positions (past_s).
// Every warp forms all of it, the same words as the others, and reads what it
// wrote itself: with the queries dealt out to the CTA's threads, the barriers
// that this took cost more than the work.
__device__ PagedRange paged_schedule(const PagedAttnParams& p, int* prefix, int* past_s,
                                     int streams, int warps) {
  const int lane = threadIdx.x & 31;
  const bool report = blockIdx.x == 0 && threadIdx.x < 32;
  const int per = (p.n + 31) / 32;
  const int b0 = min(lane * per, p.n), b1 = min(b0 + per, p.n);
  int sum = 0;
#pragma unroll 4
  for (int s = b0; s < b1; ++s) {
    const int past = p.mode == 2 ? p.prefix_past : p.past[s];
    const int nb = query_blocks(p, past, report);
    past_s[s] = nb > 0 ? past : -1;
    sum += query_chunks(p, past, nb);
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  PagedRange r;
  r.T = __shfl_sync(0xffffffffu, incl, 31) * streams;
  r.G = paged_active(gridDim.x, r.T, warps, p.n * streams);
  const int c = blockIdx.x;
  // floor(c T / G) and floor((c + 1) T / G) without 64 bits.
  int lo = 0, hi = 0;
  if (c < r.G) {
    const int q = r.T / r.G, rem = r.T - q * r.G, a = c * rem / r.G;
    lo = c * q + a;
    hi = lo + q + (c * rem - a * r.G + rem >= r.G);
  }
  int run = incl - sum;
  if (lane == 0) prefix[0] = 0;
#pragma unroll 4
  for (int s = b0; s < b1; ++s) {
    const int past = past_s[s];
    if (past >= 0) run += query_chunks(p, past, (past >> p.log2p) + 1);
    prefix[s + 1] = run;
  }
  __syncwarp();
  // The lane in whose queries the range begins or ends looks for the place.
  int at_lo = 0, at_hi = 0, s_lo = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int at = k ? hi : lo;
    if (at == 0 || at < (incl - sum) * streams || at >= incl * streams) continue;
    int s = b0;
    while (prefix[s + 1] * streams <= at) ++s;
    const int C = prefix[s + 1] - prefix[s], in = (at - prefix[s] * streams) % C;
    int cut = at;
    if (C <= kWholeRounds * warps) cut = 2 * in < C ? at - in : at + (C - in);
    if (k) {
      at_hi = cut + 1;
    } else {
      at_lo = cut;
      s_lo = s;
    }
  }
  r.lo = (int)__reduce_max_sync(0xffffffffu, (unsigned)at_lo);
  const int h = (int)__reduce_max_sync(0xffffffffu, (unsigned)at_hi);
  r.hi = h == 0 ? r.T : h - 1;   // the last range ends with the last chunk
  r.s = (int)__reduce_max_sync(0xffffffffu, (unsigned)s_lo);
  if (c >= r.G) r.lo = r.hi = 0;
  __syncwarp();
  return r;
}

// One arrival at a split stream's count: the records written before it (by
// all threads, ordered by the barrier) are seen by whoever arrives later.
__device__ __forceinline__ unsigned arrive_acq_rel(unsigned* count) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(count) : "memory");
  return old;
}

// ------------------------------------------------------------ segment results

// One stream segment's result as the CTA's threads produce it: dst is the
// output row, the record, or a partial record slot.
struct SegmentOut {
  float* o;        // element (h, d) at o[h*stride + d]
  float* m;        // or null (normalised output)
  float* l;
  size_t stride, ml_stride;
};

__device__ __forceinline__ SegmentOut segment_out(const PagedAttnParams& p, int s, int g, int hb) {
  const int h0 = g * p.group + hb * kPagedHeads;
  SegmentOut r;
  if (p.mode == 0) {
    r.o = p.out + ((size_t)s * p.n_head + h0) * p.hd;
    r.stride = p.hd;
    r.m = r.l = nullptr;
    r.ml_stride = 0;
  } else {
    const size_t at = p.mode == 1 ? (size_t)s * p.n_head + h0
                                  : ((size_t)s * p.n_kv + g) * kPagedHeads;
    r.o = p.records + at * (p.hd + 2);
    r.stride = r.ml_stride = p.hd + 2;
    r.m = r.o + p.hd;
    r.l = r.m + 1;
  }
  return r;
}

__device__ __forceinline__ SegmentOut part_out(const PagedAttnParams& p, int slot) {
  SegmentOut r;
  r.o = p.part + (size_t)slot * kPagedHeads * (p.hd + 2);
  r.stride = p.hd;
  r.m = r.o + kPagedHeads * p.hd;
  r.l = r.m + kPagedHeads;
  r.ml_stride = 1;
  return r;
}

// Four elements of a result: as they are with (m, l), or normalised.
__device__ __forceinline__ void store_segment4(const SegmentOut& dst, int h, int d, float4 O,
                                               float M, float L) {
  if (!dst.m) {
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    O.x *= inv; O.y *= inv; O.z *= inv; O.w *= inv;
  } else if (d == 0) {
    dst.m[h * dst.ml_stride] = M;
    dst.l[h * dst.ml_stride] = L;
  }
  // Output rows are 8-byte aligned, records of hd + 2 floats too.
  float2* o = reinterpret_cast<float2*>(dst.o + h * dst.stride + d);
  o[0] = make_float2(O.x, O.y);
  o[1] = make_float2(O.z, O.w);
}

// Streams without a row: zeros, or neutral records.
__device__ void write_empty(const PagedAttnParams& p, const int* prefix) {
  const int per = p.n_head * p.hd;
  for (int s = blockIdx.x; s < p.n; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    if (p.mode == 0) {
      for (int e = threadIdx.x; e < per; e += blockDim.x) p.out[(size_t)s * per + e] = 0.f;
    } else {
      for (int e = threadIdx.x; e < p.n_head * (p.hd + 2); e += blockDim.x)
        p.records[(size_t)s * p.n_head * (p.hd + 2) + e] = (e % (p.hd + 2)) == p.hd ? kNegBig : 0.f;
    }
  }
}

// The last CTA to leave its part of a split stream merges all parts.  A CTA
// has two slots: 2c for a stream it continues (its first segment), 2c + 1 for
// one that it begins and does not end (its last), so the parts of a stream
// are slot 2 c1 + 1 and the slots 2 (c1 + 1), ..., 2 c2.
__device__ __forceinline__ int part_slot(int c1, int k) { return 2 * (c1 + k) + (k == 0 ? 1 : 0); }

__device__ void merge_parts(const PagedAttnParams& p, const SegmentOut& dst, int heads,
                            int c1, int n_parts, int tid, int nthreads) {
  constexpr int B = 8;
  const int hd = p.hd;
  for (int e = tid; e < heads * hd; e += nthreads) {
    const int h = e / hd, d = e - h * hd;
    float M = kNegBig, L = 0.f, O = 0.f;
    for (int k0 = 0; k0 < n_parts; k0 += B) {
      float m[B], l[B], o[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int k = k0 + u;
        m[u] = kNegBig;
        l[u] = o[u] = 0.f;
        if (k < n_parts) {
          const SegmentOut a = part_out(p, part_slot(c1, k));
          m[u] = __ldcg(a.m + h);
          l[u] = __ldcg(a.l + h);
          o[u] = __ldcg(a.o + e);
        }
      }
      float mb = M;
#pragma unroll
      for (int u = 0; u < B; ++u) mb = fmaxf(mb, m[u]);
      const float w0 = ex2(M - mb);
      M = mb;
      L *= w0;
      O *= w0;
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const float w = ex2(m[u] - M);
        L = fmaf(l[u], w, L);
        O = fmaf(o[u], w, O);
      }
    }
    if (dst.m) {
      dst.o[h * dst.stride + d] = O;
      if (d == 0) {
        dst.m[h * dst.ml_stride] = M;
        dst.l[h * dst.ml_stride] = L;
      }
    } else {
      dst.o[h * dst.stride + d] = L > 0.f ? O / L : (L == 0.f ? 0.f : L);
    }
  }
}

// ------------------------------------------------------------ CUDA-core attention

constexpr int kCoreWarps = 8;
constexpr int kCoreThreads = 32 * kCoreWarps;

size_t paged_core_smem(int n, int hd) {
  const size_t floats = (size_t)kPagedHeads * hd                          // q
                        + (size_t)kCoreWarps * kPagedHeads * kPagedChunk    // probabilities
                        + (size_t)kCoreWarps * kPagedHeads * (hd + 2);      // warp results
  return floats * 4 + (size_t)(2 * n + 1 + 4) * 4;
}

template <typename T>
__device__ __forceinline__ float2 load_pair(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float2*>(p);
  } else {
    const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(p);
    return make_float2(__low2float(b), __high2float(b));
  }
}

// Any head_dim (even, at most 128), type and group: one warp per chunk of 32
// rows, lane r forming the scores of row r, then lane i the dimension pairs
// i, i + 32 of P.V.  All sums in binary32.
template <typename T>
__global__ void __launch_bounds__(kCoreThreads) paged_core_kernel(const PagedAttnParams p) {
  extern __shared__ float sm[];
  const int hd = p.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* q_s = sm;
  float* p_s = q_s + kPagedHeads * hd + warp * kPagedHeads * kPagedChunk;
  float* res = sm + kPagedHeads * hd + kCoreWarps * kPagedHeads * kPagedChunk;
  int* prefix = reinterpret_cast<int*>(res + kCoreWarps * kPagedHeads * (hd + 2));
  int* past_s = prefix + p.n + 1;
  int* flag = past_s + p.n;
  float* my_res = res + warp * kPagedHeads * (hd + 2);

  griddep_launch_dependents();
  griddep_wait();
  const int streams = p.n_kv * p.hblocks, cta = blockIdx.x;
  const PagedRange range = paged_schedule(p, prefix, past_s, streams, kCoreWarps);
  write_empty(p, prefix);
  const int T_all = range.T, G = range.G, t_lo = range.lo, t_hi = range.hi;
  if (t_lo >= t_hi) return;
  const T* kp = static_cast<const T*>(p.kp);
  const T* vp = static_cast<const T*>(p.vp);
  const int P = 1 << p.log2p;

  int s = range.s;
  for (int t = t_lo; t < t_hi;) {
    while (prefix[s + 1] * streams <= t) ++s;
    const int C = prefix[s + 1] - prefix[s];
    const int q_base = prefix[s] * streams, u = (t - q_base) / C;
    const int s_lo = q_base + u * C, s_hi = s_lo + C, e_hi = min(t_hi, s_hi);
    const int g = u / p.hblocks, hb = u - g * p.hblocks;
    const int heads = min(kPagedHeads, p.group - hb * kPagedHeads);
    const int past = past_s[s];
    const int nb = (past >> p.log2p) + 1;
    const int skip = query_skip(p, past);
    const int list = p.sel ? min(p.n_sel, nb) : nb - skip;
    const int* sel = p.sel ? p.sel + ((size_t)s * p.n_kv + g) * p.n_sel : nullptr;
    const int* table = p.table + (size_t)s * p.max_blocks;

    __syncthreads();
    const float* q = p.q + ((size_t)s * p.n_head + g * p.group + hb * kPagedHeads) * hd;
    for (int e = tid; e < kPagedHeads * hd; e += kCoreThreads)
      q_s[e] = e < heads * hd ? q[e] * p.scale_log2 : 0.f;
    __syncthreads();

    float m[kPagedHeads], l[kPagedHeads];
    float2 o[kPagedHeads][2];
#pragma unroll
    for (int h = 0; h < kPagedHeads; ++h) {
      m[h] = kNegBig;
      l[h] = 0.f;
      o[h][0] = o[h][1] = make_float2(0.f, 0.f);
    }
    for (int c = t + warp; c < e_hi; c += kCoreWarps) {
      const int r = (c - s_lo) * kPagedChunk + lane;
      const int i = r >> p.log2p, slot = r & (P - 1);
      bool ok = i < list;
      size_t row = 0;
      if (ok) {
        const int j = sel ? sel[i] : skip + i;
        ok = j >= 0 && j < nb && (long long)j * P + slot <= past;
        if (ok) {
          const int page = table[j];
          if (page < 0 || page >= p.n_pages) {
            record_error(p.err, kDevErrBadPage);
            ok = false;
          } else {
            row = ((((size_t)page * p.n_kv + g) << p.log2p) + slot) * hd;
          }
        }
      }
      float sc[kPagedHeads];
#pragma unroll
      for (int h = 0; h < kPagedHeads; ++h) sc[h] = 0.f;
      if (ok) {
#pragma unroll 4
        for (int d = 0; d < hd; d += 2) {
          const float2 x = load_pair(kp + row + d);
#pragma unroll
          for (int h = 0; h < kPagedHeads; ++h) {
            const float2 y = *reinterpret_cast<const float2*>(q_s + h * hd + d);
            sc[h] = fmaf(y.x, x.x, fmaf(y.y, x.y, sc[h]));
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < kPagedHeads; ++h) {
        const float x = ok ? sc[h] : -INFINITY;
        const float mn = fmaxf(m[h], warp_max(x));
        const float a = ex2(m[h] - mn), e = ex2(x - mn);
        m[h] = mn;
        l[h] = l[h] * a + e;
        o[h][0].x *= a; o[h][0].y *= a; o[h][1].x *= a; o[h][1].y *= a;
        p_s[h * kPagedChunk + lane] = e;
      }
      __syncwarp();
      const unsigned live = __ballot_sync(0xffffffffu, ok);
#pragma unroll 4
      for (int rr = 0; rr < kPagedChunk; ++rr) {
        const size_t at = __shfl_sync(0xffffffffu, (unsigned long long)row, rr);
        if (!((live >> rr) & 1)) continue;
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          const int d = 2 * lane + 64 * c2;
          if (d >= hd) continue;
          const float2 x = load_pair(vp + at + d);
#pragma unroll
          for (int h = 0; h < kPagedHeads; ++h) {
            const float w = p_s[h * kPagedChunk + rr];
            o[h][c2].x = fmaf(w, x.x, o[h][c2].x);
            o[h][c2].y = fmaf(w, x.y, o[h][c2].y);
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kPagedHeads; ++h) {
      const float lt = warp_sum(l[h]);
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        const int d = 2 * lane + 64 * c2;
        if (d < hd) *reinterpret_cast<float2*>(my_res + h * hd + d) = o[h][c2];
      }
      if (lane == 0) {
        my_res[kPagedHeads * hd + h] = m[h];
        my_res[kPagedHeads * (hd + 1) + h] = lt;
      }
    }
    __syncthreads();
    // Segment result over the warps.
    const bool complete = t == s_lo && e_hi == s_hi;
    const SegmentOut fin = segment_out(p, s, g, hb);
    const SegmentOut dst = complete ? fin : part_out(p, 2 * cta + (t == s_lo ? 1 : 0));
    for (int e = tid; e < heads * hd; e += kCoreThreads) {
      const int h = e / hd, d = e - h * hd;
      float M = kNegBig;
#pragma unroll
      for (int w = 0; w < kCoreWarps; ++w)
        M = fmaxf(M, res[w * kPagedHeads * (hd + 2) + kPagedHeads * hd + h]);
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kCoreWarps; ++w) {
        const float* rw = res + w * kPagedHeads * (hd + 2);
        const float f = ex2(rw[kPagedHeads * hd + h] - M);
        L = fmaf(rw[kPagedHeads * (hd + 1) + h], f, L);
        O = fmaf(rw[e], f, O);
      }
      if (dst.m) {
        dst.o[h * dst.stride + d] = O;
        if (d == 0) {
          dst.m[h * dst.ml_stride] = M;
          dst.l[h * dst.ml_stride] = L;
        }
      } else {
        dst.o[h * dst.stride + d] = L > 0.f ? O / L : (L == 0.f ? 0.f : L);
      }
    }
    if (!complete) {
      const int c1 = cta_of_tile(s_lo, G, T_all), c2 = cta_of_tile(s_hi - 1, G, T_all);
      unsigned* count = p.count + (size_t)s * streams + u;
      __syncthreads();
      if (tid == 0) *flag = arrive_acq_rel(count) == (unsigned)(c2 - c1);
      __syncthreads();
      if (*flag) {
        merge_parts(p, fin, heads, c1, c2 - c1 + 1, tid, kCoreThreads);
        if (tid == 0) *count = 0;
      }
    }
    t = e_hi;
  }
}

cudaError_t launch_paged_core(const PagedAttnParams& p, int dtype, int grid, cudaStream_t st) {
  static bool done_f32[64] = {}, done_bf16[64] = {};
  const size_t smem = paged_core_smem(p.n, p.hd);
  if (dtype == 1) {
    cudaError_t e = allow_max_smem(paged_core_kernel<__nv_bfloat16>, done_bf16);
    if (e != cudaSuccess) return e;
    return launch_chained(paged_core_kernel<__nv_bfloat16>, dim3(grid), dim3(kCoreThreads), smem, st, p);
  }
  cudaError_t e = allow_max_smem(paged_core_kernel<float>, done_f32);
  if (e != cudaSuccess) return e;
  return launch_chained(paged_core_kernel<float>, dim3(grid), dim3(kCoreThreads), smem, st, p);
}

// ------------------------------------------------------------ tensor-core attention

// D = A(16x8 tf32, row) * B(8x8 tf32, col) + D, fp32 accumulate.
__device__ __forceinline__ void mma_tf32_1688(float* d, const uint32_t* a, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// tma_load_2d and mbar_arrive_expect_tx by one elected lane of a converged
// warp: with warp-uniform operands the copy is issued as it is, where a
// branch of one lane moves each operand out of that lane's registers (a chunk
// of two boxes took 1000 cycles to issue).
__device__ __forceinline__ void tma_load_2d_elect(uint32_t dst, const void* tmap, uint32_t bar,
                                                  int x, int y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx_elect(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}

// A pair of floats as three pairs of bf16, each rounded from what the ones
// before leave: all 24 bits.
__device__ __forceinline__ void split3_pair(float x, float y, uint32_t& hi, uint32_t& lo,
                                            uint32_t& third) {
  float h0, r0, h1, r1, l0, l1;
  split_bf16(x, h0, r0);
  split_bf16(y, h1, r1);
  hi = pack_bf16x2(h0, h1);
  split_bf16(r0, l0, r0);
  split_bf16(r1, l1, r1);
  lo = pack_bf16x2(l0, l1);
  third = pack_bf16x2(r0, r1);
}

// mma_bf16_16816 with zeros in rows 8 to 15 of A.
__device__ __forceinline__ void mma_bf16_16816_top(float* d, const uint32_t* a, uint32_t b0,
                                                   uint32_t b1) {
  const uint32_t full[4] = {a[0], 0u, a[1], 0u};
  mma_bf16_16816(d, full, b0, b1);
}

// x = hi + lo with hi the 11 leading significant bits (a tf32 value) and lo
// exact; as an operand lo keeps its own 11 leading bits: 2^-21 of x is lost.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// Shapes of the kernel for a pool of T and head_dim HD.
template <typename T, int HD>
struct MmaPaged {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int LCH = (kHalf && HD <= 64) ? 5 : 4;   // log2 of a chunk's rows
  static constexpr int CH = 1 << LCH;
  // Warps that compute and warps that load for them.
  static constexpr int WARPS = HD <= 64 ? 8 : kHalf ? 6 : 4;
  static constexpr int PWARPS = HD <= 64 ? 4 : 2;
  static constexpr int CTHREADS = 32 * WARPS;
  // head_dim 32 and 64: four warps close segments while the others go on, and 16
  // warps share the registers of 512 threads x 128 out by role (warps of four
  // at a time: 2 x 168 + 104 + 72).  128 needs them all where it computes.
  static constexpr int CWARPS = HD <= 64 ? 4 : 0;
  static constexpr int NWARPS = WARPS + PWARPS + CWARPS;
  static constexpr int THREADS = 32 * NWARPS;
  static constexpr int RB = HD * (int)sizeof(T) < 128 ? HD * (int)sizeof(T) : 128;
  static constexpr int NX = HD * (int)sizeof(T) / RB;     // column blocks of RB bytes of a row
  static constexpr int HALF = CH * HD * (int)sizeof(T);   // K (or V) bytes of a chunk
  static constexpr int STAGE = 2 * HALF;
  static constexpr int DEPTH = HD == 32 ? 4 : 3;          // stages of a warp
  static constexpr int STAGES = DEPTH * WARPS;
  static constexpr int OT = kHalf ? HD / 16 : HD / 8;     // tiles of the output
  static constexpr int OSTRIDE = HD + (kHalf ? 4 : 8);    // floats per head in the merge area
  static constexpr int MRG = kPagedHeads * OSTRIDE + 2 * kPagedHeads;
  static constexpr int OFF_BAR = STAGES * STAGE;
  static constexpr int OFF_META = OFF_BAR + (2 * STAGES + 2) * 8;
  static constexpr int OFF_MRG = (OFF_META + STAGES * 4 + 15) & ~15;
  static constexpr int OFF_MISC = OFF_MRG + WARPS * MRG * 4;
  static constexpr int OFF_SCHED = OFF_MISC + 8 * 4;
  static constexpr size_t smem_bytes(int n) { return 1024 + (size_t)OFF_SCHED + (size_t)(2 * n + 1) * 4; }
  // Byte of 16-byte piece `piece` of row `row` in a column block, under the
  // boxes' swizzle (RB bytes: 128, or 64 with half as many pieces to turn).
  static __device__ __forceinline__ int at(int row, int piece) {
    return row * RB + ((piece ^ (RB == 128 ? row & 7 : (row >> 1) & 3)) << 4);
  }
};

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void named_sync(int bar, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(n) : "memory");
}

// Parts k0, k0 + step, ... of 16-byte item `it` (head h), merged.
struct Merged4 {
  float M, L;
  float4 O;
};

__device__ __forceinline__ Merged4 merge_item(const PagedAttnParams& p, int it, int h, int k0,
                                              int step, int n_parts, int c1) {
  constexpr int B = 4;
  Merged4 a{kNegBig, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (; k0 < n_parts; k0 += step * B) {
    float m[B], l[B];
    float4 o[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int k = k0 + u * step;
      m[u] = kNegBig;
      l[u] = 0.f;
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < n_parts) {
        const SegmentOut x = part_out(p, part_slot(c1, k));
        m[u] = __ldcg(x.m + h);
        l[u] = __ldcg(x.l + h);
        o[u] = __ldcg(reinterpret_cast<const float4*>(x.o) + it);
      }
    }
    float mb = a.M;
#pragma unroll
    for (int u = 0; u < B; ++u) mb = fmaxf(mb, m[u]);
    const float w0 = ex2(a.M - mb);
    a.M = mb;
    a.L *= w0;
    a.O.x *= w0; a.O.y *= w0; a.O.z *= w0; a.O.w *= w0;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const float w = ex2(m[u] - mb);
      a.L = fmaf(l[u], w, a.L);
      a.O.x = fmaf(o[u].x, w, a.O.x);
      a.O.y = fmaf(o[u].y, w, a.O.y);
      a.O.z = fmaf(o[u].z, w, a.O.z);
      a.O.w = fmaf(o[u].w, w, a.O.w);
    }
  }
  return a;
}

// Adds b's sums to a's.
__device__ __forceinline__ void merge_two(Merged4& a, float M, float L, float4 O) {
  const float mb = fmaxf(a.M, M), w0 = ex2(a.M - mb), w1 = ex2(M - mb);
  a.O.x = fmaf(O.x, w1, a.O.x * w0);
  a.O.y = fmaf(O.y, w1, a.O.y * w0);
  a.O.z = fmaf(O.z, w1, a.O.z * w0);
  a.O.w = fmaf(O.w, w1, a.O.w * w0);
  a.L = fmaf(L, w1, a.L * w0);
  a.M = mb;
}

// merge_parts for the tensor-core kernel: 16-byte items, the parts dealt out
// to `groups` sums per item that are then added in their order, whoever merges
// (so who arrives last does not change a bit).  This one is by threads tid,
// tid + step, ...
template <int HD, int NT>
__device__ __forceinline__ int merge_groups(int heads) {
  return max(1, min(4, NT / (heads * HD / 4)));
}
template <int HD, int NT>
__device__ void merge_parts_items(const PagedAttnParams& p, const SegmentOut& dst, int heads,
                                  int c1, int n_parts, int tid, int step) {
  const int groups = merge_groups<HD, NT>(heads);
  for (int it = tid; it < heads * HD / 4; it += step) {
    const int h = it * 4 / HD;
    Merged4 a = merge_item(p, it, h, 0, groups, n_parts, c1);
    for (int k = 1; k < groups; ++k) {
      const Merged4 b = merge_item(p, it, h, k, groups, n_parts, c1);
      merge_two(a, b.M, b.L, b.O);
    }
    store_segment4(dst, h, it * 4 - h * HD, a.O, a.M, a.L);
  }
}

// The same by all NT computing threads, a group of them for each of an item's
// sums, joined in shared memory (`sh`, 6 floats per thread).
template <int HD, int NT>
__device__ void merge_parts_vec(const PagedAttnParams& p, const SegmentOut& dst, int heads,
                                int c1, int n_parts, int tid, float* sh) {
  const int items = heads * HD / 4, groups = merge_groups<HD, NT>(heads);
  if (groups < 2) {
    merge_parts_items<HD, NT>(p, dst, heads, c1, n_parts, tid, NT);
    return;
  }
  const int grp = tid / items, it = tid - grp * items, h = it * 4 / HD;
  Merged4 a{};
  if (grp < groups) a = merge_item(p, it, h, grp, groups, n_parts, c1);
  if (grp > 0 && grp < groups) {
    float* x = sh + ((grp - 1) * items + it) * 6;
    x[0] = a.O.x; x[1] = a.O.y; x[2] = a.O.z; x[3] = a.O.w; x[4] = a.M; x[5] = a.L;
  }
  named_sync(1, NT);
  if (grp != 0) return;
  for (int k = 1; k < groups; ++k) {
    const float* x = sh + ((k - 1) * items + it) * 6;
    merge_two(a, x[4], x[5], make_float4(x[0], x[1], x[2], x[3]));
  }
  store_segment4(dst, h, it * 4 - h * HD, a.O, a.M, a.L);
}

// bf16 or fp32 pool, head_dim 32, 64 or 128; bound by HBM (a chunk's products
// take 1800 cycles of a warp, eight warps; the memory delivers a chunk in 350).
// Chunk k of the CTA's range is computing warp k % WARPS's, and each such warp
// has DEPTH stages of its own (a stage that changed hands could be two phases
// ahead of a waiting warp, which a parity cannot tell), so the warps share
// nothing until a stream's segment ends.  PWARPS warps fill the stages of
// WARPS / PWARPS computing warps each by TMA (boxes of min(page, CH) rows,
// swizzled), with the pages looked up two steps ahead.  One loading warp for
// all took 740 to 950 cycles per 8 KB chunk; computing warps that load for
// themselves spend 1000 cycles a chunk on it.  CWARPS warps join a segment's
// sums while the others are in the next one (256 x 4096 rows: 110 us without
// them, 104 with, on one machine).
//
// Products are mma.sync: a step has at most 8 query rows, far below the 64 of
// a tcgen05 tile.  For S = q K^T the 8 spare rows of the 16-row operand carry
// the low part of q.  Against exact bf16 rows x is three bf16, all its 24
// bits (two alone left results 3e-6 from those in 64 bits where binary32
// leaves 5e-7); against fp32 rows x and the rows are two tf32 each, good to
// 2^-21.
//
// In mode 2 the 8 rows are (query, head) pairs of one KV head over a prefix
// that all queries share.
//
// Measured, 14 / 2 heads of 64, bf16: 256 sequences x 4096 rows in pages of 16
// 106 us, 5.1 TB/s; 4 x 131072 in pages of 64 53 us, 5.0 TB/s.  Of a CTA's
// 207000 cycles in the first, 168000 are chunks at 6.2 TB/s, the rest the
// start (7000) and the segments' ends.
template <typename T, int HD>
__global__ void __launch_bounds__(MmaPaged<T, HD>::THREADS, 1)
    paged_mma_kernel(const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const PagedAttnParams p) {
  using Cfg = MmaPaged<T, HD>;
  constexpr int STAGES = Cfg::STAGES, NX = Cfg::NX, CH = Cfg::CH, NT = CH / 8;
  constexpr int WARPS = Cfg::WARPS, PWARPS = Cfg::PWARPS, DEPTH = Cfg::DEPTH;
  constexpr int NCT = Cfg::CTHREADS;
  constexpr bool kHalf = Cfg::kHalf;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t *left_bar = empty + STAGES, *closed_bar = left_bar + 1;
  uint32_t* meta = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_META);
  float* mrg = reinterpret_cast<float*>(smem + Cfg::OFF_MRG);
  int *flag = reinterpret_cast<int*>(smem + Cfg::OFF_MISC), *close_flag = flag + 4;
  int* prefix = reinterpret_cast<int*>(smem + Cfg::OFF_SCHED);
  int* past_s = prefix + p.n + 1;
  const int lane = threadIdx.x & 31;
  const int warp = (int)__reduce_max_sync(0xffffffffu, threadIdx.x >> 5);   // warp-uniform
  const uint32_t smem_u = smem_u32(smem), full_u = smem_u32(full);

  griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * STAGES; ++i) mbar_init(&full[i], 1);   // full and empty
    mbar_init(left_bar, WARPS);
    mbar_init(closed_bar, max(1, Cfg::CWARPS));
    fence_mbar_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  __syncthreads();
  griddep_wait();
  const int streams = p.n_kv * p.hblocks, cta = blockIdx.x;
  const PagedRange range = paged_schedule(p, prefix, past_s, streams, WARPS);
  write_empty(p, prefix);
  const int T_all = range.T, G = range.G, t_lo = range.lo, t_hi = range.hi;
  if (t_lo >= t_hi) return;
  const int P = 1 << p.log2p;
  const int box = min(P, CH), lbox = min(p.log2p, Cfg::LCH);   // rows of a TMA box
  const int nbx = CH >> lbox;                                  // boxes of a chunk, 1, 2 or 4
  const uint32_t cnt_full = (uint32_t)box * (nbx == 1 ? 1u : nbx == 2 ? 0x101u : 0x1010101u);

  // Looking a chunk's pages up takes two steps, so that neither load is waited
  // for: `entry` walks to the chunk's stream and reads the listed entry j (if
  // there is a list), `page` reads the table.  Lane b has box b.
  struct Entry {
    int s, g, j, off;    // j -1: no such box
  };
  struct Box {
    int page, rows, y0;  // rows 0: nothing to load; y0: TMA row less the page's
  };
  // The stream that `entry` stands in: query ls, stream lu of it, flat chunks
  // [l_lo, l_hi).
  int ls = range.s;
  while (prefix[ls + 1] * streams <= t_lo) ++ls;
  int s = ls;
  int l_c = prefix[ls + 1] - prefix[ls], lu = (t_lo - prefix[ls] * streams) / l_c;
  int l_lo = prefix[ls] * streams + lu * l_c, l_hi = l_lo + l_c;
  auto entry = [&](int t) -> Entry {
    Entry e{0, 0, -1, 0};
    if (t >= t_hi) return e;
    while (t >= l_hi) {
      if (++lu == streams) {
        lu = 0;
        do ++ls; while (prefix[ls + 1] == prefix[ls]);
        l_c = prefix[ls + 1] - prefix[ls];
      }
      l_lo = l_hi;
      l_hi += l_c;
    }
    if (lane >= nbx) return e;
    e.s = ls;
    e.g = p.hblocks == 1 ? lu : lu / p.hblocks;
    const int past = past_s[ls], nb = (past >> p.log2p) + 1, skip = query_skip(p, past);
    const int list = p.sel ? min(p.n_sel, nb) : nb - skip;
    const int row = ((t - l_lo) * nbx + lane) << lbox;   // row of the stream, below 2^31
    const int i = row >> p.log2p;
    e.off = row & (P - 1);
    if (i < list) e.j = p.sel ? p.sel[((size_t)ls * p.n_kv + e.g) * p.n_sel + i] : skip + i;
    return e;
  };
  auto page = [&](const Entry& e) -> Box {
    Box b{0, 0, 0};
    if (e.j < 0) return b;
    const int rows = past_s[e.s] + 1 - ((e.j << p.log2p) + e.off);
    if (e.j > past_s[e.s] >> p.log2p || rows <= 0) return b;
    b.rows = min(box, rows);
    b.page = p.table[(p.mode == 2 ? 0 : (size_t)e.s * p.max_blocks) + e.j];
    b.y0 = (int)((p.page0 * p.n_kv + e.g) << p.log2p) + e.off;
    return b;
  };
  // Fills stage st with the chunk whose boxes lanes 0..nbx-1 have.
  auto load = [&](int st, const Box& x) {
    int rows = x.rows;
    if (rows > 0 && (x.page < 0 || x.page >= p.n_pages)) {
      record_error(p.err, kDevErrBadPage);
      rows = 0;
    }
    // Reductions leave warp-uniform values: the rows of all boxes, and below
    // each box's TMA row.
    const int y = x.y0 + ((x.page * p.n_kv) << p.log2p);
    const uint32_t m = __reduce_or_sync(0xffffffffu, lane < nbx ? (uint32_t)rows << (8 * lane) : 0u);
    meta[st] = m;
    const uint32_t bar = full_u + 8 * st, to = smem_u + st * Cfg::STAGE;
    int loads = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) loads += ((m >> (8 * b)) & 255u) != 0;
    mbar_arrive_expect_tx_elect(bar, (uint32_t)(loads * box * 2 * NX * Cfg::RB));
    for (int b = 0; b < nbx; ++b) {
      const int yb = (int)__reduce_max_sync(0xffffffffu, lane == b ? (uint32_t)y : 0u);
      if ((m >> (8 * b)) & 255u) {
#pragma unroll
        for (int c = 0; c < NX; ++c) {
          const uint32_t at = to + b * box * Cfg::RB + c * (CH * Cfg::RB);
          tma_load_2d_elect(at, &tmk, bar, c * (Cfg::RB / (int)sizeof(T)), yb);
          tma_load_2d_elect(at + Cfg::HALF, &tmv, bar, c * (Cfg::RB / (int)sizeof(T)), yb);
        }
      }
    }
    __syncwarp();
  };

  if (warp >= WARPS && warp < WARPS + PWARPS) {
    // -------------------------------------------------------------- loading
    // Chunk n of this warp: chunk first + n % M of round n / M.
    constexpr int M = WARPS / PWARPS, L = M * DEPTH;
    if constexpr (Cfg::CWARPS > 0) setmaxnreg_dec<104>();
    const int first = (warp - WARPS) * M;
    Entry e[L + 3];
    Box b[L + 2];
#pragma unroll
    for (int n = 0; n < L + 3; ++n) e[n] = entry(t_lo + n / M * WARPS + first + n % M);
#pragma unroll
    for (int n = 0; n < L + 2; ++n) b[n] = page(e[n]);
    int issued = 0;
#pragma unroll
    for (int n = 0; n < L; ++n) {
      if (t_lo + n / M * WARPS + first + n % M >= t_hi) break;
      load((first + n % M) * DEPTH + n / M, b[n]);
      ++issued;
    }
    Box b0 = b[L], b1 = b[L + 1];
    Entry e2 = e[L + 2];
    int round = DEPTH, i = 0, slot = 0;   // of the next chunk
    int round3 = (L + 3) / M, i3 = (L + 3) % M;   // of the one to look up
    uint32_t ph = 0;
    while (t_lo + round * WARPS + first + i < t_hi) {
      const int st = (first + i) * DEPTH + slot;
      const bool got = mbar_wait(&empty[st], ph, p.err, kDevErrWaitEmpty);
      if (!__all_sync(0xffffffffu, got)) break;
      load(st, b0);
      ++issued;
      b0 = b1;
      b1 = page(e2);
      e2 = entry(t_lo + round3 * WARPS + first + i3);
      if (++i3 == M) {
        i3 = 0;
        ++round3;
      }
      if (++i == M) {
        i = 0;
        ++round;
        if (++slot == DEPTH) {
          slot = 0;
          ph ^= 1u;
        }
      }
    }
    // Every load lands (bounded) before the CTA exits.
    for (int n = max(0, issued - L); n < issued; ++n)
      mbar_wait(&full[(first + n % M) * DEPTH + n / M % DEPTH], (uint32_t)(n / L & 1), p.err,
                kDevErrWaitFull);
    return;
  }

  // A CTA's range falls into segments, one per stream.
  struct Segment {
    int u, g, hb, heads;
    int s_lo, s_hi, e_hi;   // the stream's chunks, the segment's end
  };
  auto segment = [&](int t) -> Segment {   // of chunk t of query s
    while (prefix[s + 1] * streams <= t) ++s;
    const int C = prefix[s + 1] - prefix[s], q_base = prefix[s] * streams;
    Segment x;
    x.u = (t - q_base) / C;
    x.s_lo = q_base + x.u * C;
    x.s_hi = x.s_lo + C;
    x.e_hi = min(t_hi, x.s_hi);
    x.g = x.u / p.hblocks;
    x.hb = x.u - x.g * p.hblocks;
    x.heads = min(kPagedHeads, p.mode == 2 ? p.n_rows - s * kPagedHeads
                                           : p.group - x.hb * kPagedHeads);
    return x;
  };
  // The computing warps' sums of a segment, joined by threads first, first +
  // step, ... and stored as the stream's result or as a part of it.
  auto join = [&](const Segment& x, int t, int first, int step) -> bool {
    const bool complete = t == x.s_lo && x.e_hi == x.s_hi;
    const SegmentOut dst = complete ? segment_out(p, s, x.g, x.hb)
                                    : part_out(p, 2 * cta + (t == x.s_lo ? 1 : 0));
    for (int e = first; e < x.heads * HD / 4; e += step) {
      const int h = e * 4 / HD, d = e * 4 - h * HD;
      float M = kNegBig;
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
        M = fmaxf(M, mrg[w * Cfg::MRG + kPagedHeads * Cfg::OSTRIDE + h]);
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* mw = mrg + w * Cfg::MRG;
        const float f = ex2(mw[kPagedHeads * Cfg::OSTRIDE + h] - M);
        const float4 v = *reinterpret_cast<const float4*>(mw + h * Cfg::OSTRIDE + d);
        L = fmaf(mw[kPagedHeads * (Cfg::OSTRIDE + 1) + h], f, L);
        O.x = fmaf(v.x, f, O.x);
        O.y = fmaf(v.y, f, O.y);
        O.z = fmaf(v.z, f, O.z);
        O.w = fmaf(v.w, f, O.w);
      }
      store_segment4(dst, h, d, O, M, L);
    }
    return complete;
  };
  // One arrival at a split stream: whether it is the last (its count is then
  // back at 0), the stream's first CTA and its number of parts.
  auto arrive_last = [&](const Segment& x, int* to) {
    const int c1 = cta_of_tile(x.s_lo, G, T_all);
    const int parts = cta_of_tile(x.s_hi - 1, G, T_all) - c1 + 1;
    unsigned* count = p.count + (size_t)s * streams + x.u;
    to[0] = arrive_acq_rel(count) == (unsigned)(parts - 1);
    to[1] = c1;
    to[2] = parts;
    if (to[0]) *count = 0;
  };

  if (Cfg::CWARPS > 0 && warp >= WARPS + PWARPS) {
    // -------------------------------------------------------------- closing
    // All segments but the last, while the others go on with the next.
    setmaxnreg_dec<72>();
    constexpr int NC = 32 * Cfg::CWARPS;
    const int ct = threadIdx.x - 32 * (WARPS + PWARPS);
    uint32_t ph = 0;
    for (int t = t_lo; t < t_hi; ph ^= 1u) {
      const Segment x = segment(t);
      if (x.e_hi >= t_hi) break;
      mbar_wait(left_bar, ph, p.err, kDevErrWaitFull);
      __syncwarp();
      const bool complete = join(x, t, ct, NC);
      __syncwarp();
      if (lane == 0) mbar_arrive(closed_bar);
      if (!complete) {
        named_sync(2, NC);
        if (ct == 0) arrive_last(x, close_flag);
        named_sync(2, NC);
        if (close_flag[0])
          merge_parts_items<HD, NCT>(p, segment_out(p, s, x.g, x.hb), x.heads, close_flag[1],
                                     close_flag[2], ct, NC);
      }
      t = x.e_hi;
    }
    return;
  }

  // ---------------------------------------------------------------- computing
  if constexpr (Cfg::CWARPS > 0) setmaxnreg_inc<168>();
  const int r = lane >> 2, qd = lane & 3;
  float* my_mrg = mrg + warp * Cfg::MRG;
  const float sl2 = p.scale_log2;
  // q of a stream, this lane's elements (row r of the operand), loaded a
  // segment ahead: behind full rings of tiles a load takes 5000 cycles.
  float q_raw[HD / 4];
  auto load_q = [&](int qs, int qu) {
    const int g = p.hblocks == 1 ? qu : qu / p.hblocks, hb = qu - g * p.hblocks;
    int h = hb * kPagedHeads + r;
    bool row_ok = h < p.group;
    if (p.mode == 2) {
      h = qs * kPagedHeads + r;
      row_ok = h < p.n_rows;
      qs = h / p.group;
      h -= qs * p.group;
    }
    const float* q = p.q + ((size_t)qs * p.n_head + g * p.group + h) * HD;
#pragma unroll
    for (int kk = 0; kk < HD / (kHalf ? 16 : 8); ++kk)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if constexpr (kHalf) {
          float2 v = make_float2(0.f, 0.f);
          if (row_ok) v = *reinterpret_cast<const float2*>(q + 16 * kk + 8 * half + 2 * qd);
          q_raw[4 * kk + 2 * half] = v.x;
          q_raw[4 * kk + 2 * half + 1] = v.y;
        } else {
          q_raw[2 * kk + half] = row_ok ? q[8 * kk + 4 * half + qd] : 0.f;
        }
      }
  };
  load_q(ls, lu);
  int ti = t_lo + warp;   // this warp's next chunk to compute
  bool failed = false;
  int slot = 0;
  uint32_t ph = 0;
  uint32_t qa[kHalf ? HD / 16 : HD / 8][4];
  uint32_t q3[HD / 16][2];   // bf16: the third parts
  float o[Cfg::OT][4];   // bf16: (16 of head_dim) x (8 heads), else (8 heads, hi and lo) x (8)
  uint32_t closed_ph = 1;   // of the segment before: none
  for (int t = t_lo; t < t_hi;) {
    const Segment x = segment(t);
    const int e_hi = x.e_hi;
    // This segment's q was loaded before; the next one's is on its way.
#pragma unroll
    for (int kk = 0; kk < HD / (kHalf ? 16 : 8); ++kk)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if constexpr (kHalf) {
          const float2 v = make_float2(q_raw[4 * kk + 2 * half], q_raw[4 * kk + 2 * half + 1]);
          split3_pair(v.x, v.y, qa[kk][2 * half], qa[kk][2 * half + 1], q3[kk][half]);
        } else {
          split_tf32(q_raw[2 * kk + half], qa[kk][2 * half], qa[kk][2 * half + 1]);
        }
      }
    if (e_hi < t_hi) {
      int sn = s, un = x.u;
      if (e_hi == x.s_hi && ++un == streams) {
        un = 0;
        do ++sn; while (prefix[sn + 1] == prefix[sn]);
      }
      load_q(sn, un);
    }
#pragma unroll
    for (int c = 0; c < Cfg::OT; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    float m_run = kNegBig, l_run = 0.f;

    for (; ti < e_hi; ti += WARPS) {
      const int st = warp * DEPTH + slot;
      if (!failed && !mbar_wait(&full[st], ph, p.err, kDevErrWaitFull)) failed = true;
      failed = __any_sync(0xffffffffu, failed);
      const uint32_t cm = meta[st];
      if (!failed && cm != 0) {
        uint8_t* kbox = smem + st * Cfg::STAGE;
        uint8_t* vbox = kbox + Cfg::HALF;
        const bool whole = cm == cnt_full;
        if (!whole) {
          // Rows that are not attended may hold anything: their V becomes
          // zero, so that weight 0 adds exactly zero.
          const int row = lane;
          if (row < CH && (row & (box - 1)) >= (int)((cm >> (8 * (row >> lbox))) & 255u)) {
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
              for (int e = 0; e < Cfg::RB / 16; ++e)
                *reinterpret_cast<uint4*>(vbox + x * (CH * Cfg::RB) + Cfg::at(row, e)) =
                    make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        const uint32_t kb = smem_u32(kbox), vb = smem_u32(vbox);
        // S = q . K^T in blocks of 8 rows.
        float sc[NT][2];
        // bf16: products in turn on four accumulators or more, so that none
        // waits for the one before it.
        constexpr int NA = kHalf ? (NT >= 4 ? 1 : 4 / NT) : 2;
        float acc_s[NT][NA][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int a = 0; a < NA; ++a)
            acc_s[nt][a][0] = acc_s[nt][a][1] = acc_s[nt][a][2] = acc_s[nt][a][3] = 0.f;
        if constexpr (kHalf) {
#pragma unroll
          for (int kq = 0; kq < HD / 32; ++kq) {
            uint32_t b[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int row = 8 * nt + (lane & 7), chunk = 4 * (kq & 1) + (lane >> 3);
              ldmatrix_x4(kb + (kq >> 1) * (CH * Cfg::RB) + Cfg::at(row, chunk), b[nt][0],
                          b[nt][1], b[nt][2], b[nt][3]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_bf16_16816(acc_s[nt][0], qa[2 * kq + x], b[nt][2 * x], b[nt][2 * x + 1]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_bf16_16816_top(acc_s[nt][NA - 1], q3[2 * kq + x], b[nt][2 * x],
                                   b[nt][2 * x + 1]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float(&acc)[NA][4] = acc_s[nt];
          if constexpr (!kHalf) {
            const int row = 8 * nt + r;
#pragma unroll
            for (int kk = 0; kk < HD / 8; ++kk) {
              const uint8_t* a = kbox + (kk >> 2) * (CH * 128) + qd * 4;
              const int chunk = 2 * (kk & 3);
              uint32_t h0, l0, h1, l1;
              split_tf32(*reinterpret_cast<const float*>(a + Cfg::at(row, chunk)), h0, l0);
              split_tf32(*reinterpret_cast<const float*>(a + Cfg::at(row, chunk + 1)), h1, l1);
              mma_tf32_1688(acc[0], qa[kk], h0, h1);
              mma_tf32_1688(acc[1], qa[kk], l0, l1);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = acc[0][e] + acc[0][e + 2];
            if constexpr (NA > 1) x += acc[1][e] + acc[1][e + 2];
            sc[nt][e] = x * sl2;
          }
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = 8 * nt + 2 * qd + e;
              if ((c & (box - 1)) >= (int)((cm >> (8 * (c >> lbox))) & 255u)) sc[nt][e] = -INFINITY;
            }
          }
        }
        // Online softmax over the chunk's rows (a query head is a quad of lanes).
        float mx = fmaxf(sc[0][0], sc[0][1]);
#pragma unroll
        for (int nt = 1; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(sc[nt][0], sc[nt][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run, mx);
        const float alpha = ex2(m_run - m_new);
        m_run = m_new;
        float lsum = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][0] = ex2(sc[nt][0] - m_new);
          sc[nt][1] = ex2(sc[nt][1] - m_new);
          lsum += sc[nt][0] + sc[nt][1];
        }
        l_run = l_run * alpha + lsum;
        float a0 = alpha, a1 = alpha;
        if constexpr (kHalf) {   // of the heads of this lane's columns
          a0 = __shfl_sync(0xffffffffu, alpha, 8 * qd);
          a1 = __shfl_sync(0xffffffffu, alpha, 8 * qd + 4);
        }
        // O = alpha O + P . V, the chunk's product formed by itself: the
        // tensor cores truncate what they add to an accumulator, and over a
        // long stream that added up to 3e-6 of the result.
        auto add_to_o = [&](float(&o)[4], const float(&d)[4]) {
          o[0] = fmaf(o[0], a0, d[0]);
          o[1] = fmaf(o[1], a1, d[1]);
          o[2] = fmaf(o[2], a0, d[2]);
          o[3] = fmaf(o[3], a1, d[3]);
        };
        if constexpr (kHalf) {
          // A lane's scores (one head, two rows of K) are the B operand of
          // O^T += V^T . P^T as they stand.
          constexpr int NK = CH / 16;
          uint32_t p1[NK][2], p2[NK][2], p3[NK][2];
#pragma unroll
          for (int kp = 0; kp < NK; ++kp)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              split3_pair(sc[2 * kp + e][0], sc[2 * kp + e][1], p1[kp][e], p2[kp][e], p3[kp][e]);
#pragma unroll
          for (int x = 0; x < NX; ++x) {
            constexpr int NC = Cfg::RB / 32;   // 16-column tiles of a block
            float d[NC][4];
#pragma unroll
            for (int c = 0; c < NC; ++c) d[c][0] = d[c][1] = d[c][2] = d[c][3] = 0.f;
#pragma unroll
            for (int kp = 0; kp < NK; ++kp) {
              const int row = 16 * kp + ((lane >> 3) & 1) * 8 + (lane & 7);
              uint32_t v[NC][4];
#pragma unroll
              for (int c = 0; c < NC; ++c)
                ldmatrix_x4_trans(vb + x * (CH * Cfg::RB) + Cfg::at(row, 2 * c + (lane >> 4)),
                                  v[c][0], v[c][2], v[c][1], v[c][3]);
#pragma unroll
              for (int c = 0; c < NC; ++c) mma_bf16_16816(d[c], v[c], p1[kp][0], p1[kp][1]);
#pragma unroll
              for (int c = 0; c < NC; ++c) mma_bf16_16816(d[c], v[c], p2[kp][0], p2[kp][1]);
#pragma unroll
              for (int c = 0; c < NC; ++c) mma_bf16_16816(d[c], v[c], p3[kp][0], p3[kp][1]);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) add_to_o(o[NC * x + c], d[c]);
          }
        } else {
          // Rows 2 qd and 2 qd + 1 of a block are the operand's k = qd and
          // k = qd + 4, so the scores are its layout already (the order of
          // the rows in a sum is free), and no two lanes share a bank.
          uint32_t pa[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            split_tf32(sc[nt][0], pa[nt][0], pa[nt][1]);
            split_tf32(sc[nt][1], pa[nt][2], pa[nt][3]);
          }
#pragma unroll
          for (int x = 0; x < NX; ++x) {
            float d[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c][0] = d[c][1] = d[c][2] = d[c][3] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int row = 8 * nt + 2 * qd, chunk = 2 * c + (r >> 2);
                const uint8_t* a = vbox + x * (CH * 128) + (r & 3) * 4;
                uint32_t h0, l0, h1, l1;
                split_tf32(*reinterpret_cast<const float*>(a + Cfg::at(row, chunk)), h0, l0);
                split_tf32(*reinterpret_cast<const float*>(a + Cfg::at(row + 1, chunk)), h1, l1);
                mma_tf32_1688(d[c], pa[nt], h0, h1);
                mma_tf32_1688(d[c], pa[nt], l0, l1);
              }
#pragma unroll
            for (int c = 0; c < 4; ++c) add_to_o(o[4 * x + c], d[c]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++slot == DEPTH) {
        slot = 0;
        ph ^= 1u;
      }
    }
    // ---------------------------------------------------------- segment end
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    const bool handed = Cfg::CWARPS > 0 && e_hi < t_hi;   // to the closing warps
    if (Cfg::CWARPS > 0 && t > t_lo) mbar_wait(closed_bar, closed_ph, p.err, kDevErrWaitEmpty);
    closed_ph ^= 1u;
#pragma unroll
    for (int c = 0; c < Cfg::OT; ++c) {
      if constexpr (kHalf) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          my_mrg[(2 * qd + (e & 1)) * Cfg::OSTRIDE + 16 * c + 8 * (e >> 1) + r] = o[c][e];
      } else {
        *reinterpret_cast<float2*>(my_mrg + r * Cfg::OSTRIDE + 8 * c + 2 * qd) =
            make_float2(o[c][0] + o[c][2], o[c][1] + o[c][3]);
      }
    }
    if (qd == 0) {
      my_mrg[kPagedHeads * Cfg::OSTRIDE + r] = m_run;
      my_mrg[kPagedHeads * (Cfg::OSTRIDE + 1) + r] = l_run;
    }
    if (handed) {
      __syncwarp();
      if (lane == 0) mbar_arrive(left_bar);
    } else {
      // The last one: nothing is left to go on with, so all warps close it.
      named_sync(1, NCT);
      if (!join(x, t, threadIdx.x, NCT)) {
        named_sync(1, NCT);
        if (threadIdx.x == 0) arrive_last(x, flag);
        named_sync(1, NCT);
        if (flag[0])
          merge_parts_vec<HD, NCT>(p, segment_out(p, s, x.g, x.hb), x.heads, flag[1], flag[2],
                                   threadIdx.x, mrg);
      }
      if constexpr (Cfg::CWARPS == 0) named_sync(1, NCT);
    }
    t = e_hi;
  }
}

template <typename T, int HD>
static cudaError_t launch_mma_cfg(const CUtensorMap& tk, const CUtensorMap& tv,
                                  const PagedAttnParams& p, int grid, cudaStream_t st) {
  static bool done[64] = {};
  cudaError_t e = allow_max_smem(paged_mma_kernel<T, HD>, done);
  if (e != cudaSuccess) return e;
  return launch_chained(paged_mma_kernel<T, HD>, dim3(grid), dim3(MmaPaged<T, HD>::THREADS),
                        MmaPaged<T, HD>::smem_bytes(p.n), st, tk, tv, p);
}

int paged_mma_lchunk(int dtype, int hd) {
  static_assert(MmaPaged<__nv_bfloat16, 32>::LCH == MmaPaged<__nv_bfloat16, 64>::LCH, "rows");
  static_assert(MmaPaged<float, 32>::LCH == MmaPaged<float, 64>::LCH &&
                    MmaPaged<float, 128>::LCH == MmaPaged<float, 64>::LCH &&
                    MmaPaged<__nv_bfloat16, 128>::LCH == MmaPaged<float, 64>::LCH, "rows");
  return dtype == 1 && hd <= 64 ? MmaPaged<__nv_bfloat16, 64>::LCH : MmaPaged<float, 64>::LCH;
}

cudaError_t launch_paged_mma(const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnParams& p,
                             int dtype, int grid, cudaStream_t st) {
  static_assert(MmaPaged<float, 128>::smem_bytes(kPagedMaxQueries) <= 227 * 1024, "shared memory");
  static_assert(MmaPaged<__nv_bfloat16, 128>::smem_bytes(kPagedMaxQueries) <= 227 * 1024, "shared memory");
  static_assert(MmaPaged<float, 64>::smem_bytes(kPagedMaxQueries) <= 227 * 1024, "shared memory");
  static_assert(MmaPaged<__nv_bfloat16, 64>::smem_bytes(kPagedMaxQueries) <= 227 * 1024, "shared memory");
  if (p.hd == 32)
    return dtype == 1 ? launch_mma_cfg<__nv_bfloat16, 32>(tk, tv, p, grid, st)
                      : launch_mma_cfg<float, 32>(tk, tv, p, grid, st);
  if (p.hd == 64)
    return dtype == 1 ? launch_mma_cfg<__nv_bfloat16, 64>(tk, tv, p, grid, st)
                      : launch_mma_cfg<float, 64>(tk, tv, p, grid, st);
  return dtype == 1 ? launch_mma_cfg<__nv_bfloat16, 128>(tk, tv, p, grid, st)
                    : launch_mma_cfg<float, 128>(tk, tv, p, grid, st);
}

// The result of a batch behind a packed prefix: a thread per pair of
// dimensions merges two records, 1 MB at 128 queries x 14 heads (latency).
__global__ void __launch_bounds__(256) paged_packed_merge_kernel(const PagedPackedParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int pairs = p.hd / 2;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  if (e >= (long long)p.n * p.n_head * pairs) return;
  const int d = 2 * (int)(e % pairs), row = (int)(e / pairs);
  const int s = row / p.n_head, head = row - s * p.n_head, g = head / p.group;
  const int x = s * p.group + head - g * p.group;   // row of the packed prefix
  const float* a = p.own + (size_t)row * (p.hd + 2);
  const float* b = p.packed + (((size_t)(x / kPagedHeads) * p.n_kv + g) * kPagedHeads +
                               x % kPagedHeads) * (p.hd + 2);
  float2 O = *reinterpret_cast<const float2*>(a + d);
  const float2 ml = *reinterpret_cast<const float2*>(a + p.hd);
  float L = ml.y;
  const int past = p.past[s];
  if (past >= p.shared - 1 && past < p.limit) {
    const float2 o2 = *reinterpret_cast<const float2*>(b + d);
    const float2 ml2 = *reinterpret_cast<const float2*>(b + p.hd);
    const float M = fmaxf(ml.x, ml2.x), w = ex2(ml.x - M), w2 = ex2(ml2.x - M);
    O.x = fmaf(o2.x, w2, O.x * w);
    O.y = fmaf(o2.y, w2, O.y * w);
    L = fmaf(ml2.y, w2, L * w);
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  *reinterpret_cast<float2*>(p.out + (size_t)row * p.hd + d) = make_float2(O.x * inv, O.y * inv);
}

cudaError_t launch_paged_packed_merge(const PagedPackedParams& p, cudaStream_t st) {
  const long long items = (long long)p.n * p.n_head * (p.hd / 2);
  return launch_chained(paged_packed_merge_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256),
                        0, st, p);
}

// ------------------------------------------------------------ page selection
//
// Score of a page for one KV head: the largest, over the head's query group,
// of sum_d max(q_d lo_d, q_d hi_d), an upper bound of q . k for every key of
// the page.  Which of two pages is taken must not hang on the order of a
// sum's roundings, so the order of the pages is that of the scores in
// binary64 (products of a 24-bit q and a bf16 or fp32 bound are exact
// there).  Computing them all there is slow, so the scores come from the
// tensor cores with a bound E on their error, and only the pages within 2 E of
// the n_sel-th score are scored again: with T the n_sel-th largest of these
// scores, a page above T + 2 E is taken (whatever may beat it is above T too,
// and fewer than n_sel pages are), one below T - 2 E is not.

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelNear = 256;       // pages near the border that are ranked by comparisons
constexpr int kSelCached = 16384;   // binary32 keys that the picking CTA holds in shared memory
constexpr uint32_t kKeyForced = ~0u;  // pages that are always taken

// Unsigned integers in the order of the floating-point numbers (-0 as +0).
__device__ __forceinline__ uint32_t ordered_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long ordered_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// Scores of 8 pages by one warp with mma.sync: max(q, 0) times the upper
// bounds plus min(q, 0) times the lower ones, rows 0-7 of the operand the high
// parts of up to 8 heads, rows 8-15 the low parts (as in paged_mma_kernel).
// The order of the dimensions in a sum is free, so a lane's part of the 8
// page columns is whole 16-byte pieces straight from memory (piece c of lane
// (page, qd) is piece 4 c + qd of the page's row); the q operands of every
// product lie in shared memory as the lanes need them.  Lane (r, qd) returns
// the scores of pages 2 qd and 2 qd + 1, the same for every r; *big is raised
// to the largest |bound| of the lane's own pieces, or to infinity when a
// score is not finite.  (Plain multiply-adds with q read from shared memory
// took 14000 cycles for 444 pages x 7 heads, bound by those reads.)
template <typename T, int HD>
struct ScoreMma {
  static constexpr int PIECES = HD * (int)sizeof(T) / 64;  // 16-byte pieces of a lane and bound
  static constexpr int PER = 2;                            // products of a piece
  static constexpr int OPERANDS = 2 * PIECES * PER;        // of a block of 8 heads
};

template <typename T, int HD>
__device__ __forceinline__ void load_bounds(const T* row,
                                            uint4 (&b)[2][ScoreMma<T, HD>::PIECES]) {
  const int qd = threadIdx.x & 3;
#pragma unroll
  for (int c = 0; c < ScoreMma<T, HD>::PIECES; ++c) {
    b[0][c] = reinterpret_cast<const uint4*>(row + HD)[4 * c + qd];   // upper
    b[1][c] = reinterpret_cast<const uint4*>(row)[4 * c + qd];        // lower
  }
}

template <typename T, int HD>
__device__ __forceinline__ float2 page_scores(const uint4 (&b)[2][ScoreMma<T, HD>::PIECES],
                                              const uint4* q_s, int hblocks, int last_heads,
                                              float* big) {
  using Cfg = ScoreMma<T, HD>;
  const int lane = threadIdx.x & 31, r = lane >> 2;
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < Cfg::PIECES; ++c) {
      const uint32_t w[4] = {b[k][c].x, b[k][c].y, b[k][c].z, b[k][c].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 2) {
          m = fmaxf(m, fmaxf(fabsf(__uint_as_float(w[e] << 16)),
                             fabsf(__uint_as_float(w[e] & 0xffff0000u))));
        } else {
          m = fmaxf(m, fabsf(__uint_as_float(w[e])));
        }
      }
    }
  float2 best = make_float2(-INFINITY, -INFINITY);
  bool odd = false;
  for (int hb = 0; hb < hblocks; ++hb) {
    float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    const uint4* q = q_s + hb * Cfg::OPERANDS * 32 + lane;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < Cfg::PIECES; ++c) {
        const uint32_t w[4] = {b[k][c].x, b[k][c].y, b[k][c].z, b[k][c].w};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 x = q[((k * Cfg::PIECES + c) * 2 + u) * 32];
          const uint32_t a[4] = {x.x, x.y, x.z, x.w};
          if constexpr (sizeof(T) == 2) {
            mma_bf16_16816(acc[k], a, w[2 * u], w[2 * u + 1]);
          } else {
            uint32_t h0, l0, h1, l1;
            split_tf32(__uint_as_float(w[2 * u]), h0, l0);
            split_tf32(__uint_as_float(w[2 * u + 1]), h1, l1);
            mma_tf32_1688(acc[k], a, h0, h1);
            mma_tf32_1688(acc[k], a, l0, l1);
          }
        }
      }
    float x0 = (acc[0][0] + acc[0][2]) + (acc[1][0] + acc[1][2]);
    float x1 = (acc[0][1] + acc[0][3]) + (acc[1][1] + acc[1][3]);
    if (r < (hb + 1 == hblocks ? last_heads : kPagedHeads)) {
      odd |= !(fabsf(x0) < INFINITY) || !(fabsf(x1) < INFINITY);
      best.x = fmaxf(best.x, x0);
      best.y = fmaxf(best.y, x1);
    }
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    best.x = fmaxf(best.x, __shfl_xor_sync(0xffffffffu, best.x, o));
    best.y = fmaxf(best.y, __shfl_xor_sync(0xffffffffu, best.y, o));
  }
  *big = __any_sync(0xffffffffu, odd) ? INFINITY : fmaxf(*big, m);
  return best;
}

// Score of one page by one thread, any even head_dim, in binary32.
template <typename T>
__device__ float page_score_any(const T* lo_p, const float* q_f, int group, int hd, float* big) {
  float best = -INFINITY, m = 0.f;
  bool odd = false;
  for (int h = 0; h < group; ++h) {
    float sum = 0.f;
    for (int d = 0; d < hd; d += 2) {
      const float2 a = load_pair(lo_p + d), b = load_pair(lo_p + hd + d);
      const float q0 = q_f[h * hd + d], q1 = q_f[h * hd + d + 1];
      sum = fmaf(q0, q0 >= 0.f ? b.x : a.x, sum);
      sum = fmaf(q1, q1 >= 0.f ? b.y : a.y, sum);
      if (h == 0)
        m = fmaxf(m, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
    }
    odd |= !(fabsf(sum) < INFINITY);
    best = fmaxf(best, sum);
  }
  *big = odd ? INFINITY : fmaxf(*big, m);
  return best;
}

// Binary64 score of a page for one head, by eight lanes (a warp has four pairs
// of page and head in hand: with one pair, 12 pages x 16 heads took 34000
// cycles, nearly all of them latency; with eight, 9000).  Both bounds are
// loaded, so that no load waits for q.
template <typename T, int HD>
__device__ __forceinline__ double exact_score(const T* lo_p, const float* q, int hd) {
  double sum = 0.0;
  if constexpr (HD > 0) {
#pragma unroll
    for (int k = 0; k < HD / 8; ++k) {
      const int d = 8 * k + (threadIdx.x & 7);
      const float x = q[d], up = to_f32(lo_p[HD + d]), low = to_f32(lo_p[d]);
      sum = fma((double)x, (double)(x >= 0.f ? up : low), sum);
    }
  } else {
    for (int d = threadIdx.x & 7; d < hd; d += 8) {
      const float x = q[d], up = to_f32(lo_p[hd + d]), low = to_f32(lo_p[d]);
      sum = fma((double)x, (double)(x >= 0.f ? up : low), sum);
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// Shared memory of the picking CTA.
struct PickShared {
  unsigned count[2][kSelWarps];
  unsigned long long wide[2][kSelWarps];
  unsigned hist[kSelThreads];
  unsigned steps[3];
  unsigned near, sure;
  float big[kSelWarps];
  int flag;
  int near_at[kSelNear], near_page[kSelNear];
  unsigned long long near_key[kSelNear];
};

// Bit by bit from the top: does taking the bit leave k keys?  For keys so
// many of which are equal that they cannot be told apart by bins.
template <typename K>
__device__ K kth_key_bits(const K* keys, int n, unsigned k, PickShared& sh, unsigned* need) {
  const int tid = threadIdx.x, lane = tid & 31;
  __syncthreads();
  if (tid < 3) sh.steps[tid] = 0;
  __syncthreads();
  K bound = 0;
  int step = 0;
  auto count = [&](K cand) -> unsigned {
    unsigned c = 0;
    for (int i = tid; i < n; i += kSelThreads) c += keys[i] >= cand;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0 && c) atomicAdd(&sh.steps[step], c);
    if (tid == 0) sh.steps[step == 2 ? 0 : step + 1] = 0;
    __syncthreads();
    c = sh.steps[step];
    step = step == 2 ? 0 : step + 1;
    return c;
  };
  for (int bit = 8 * (int)sizeof(K) - 1; bit >= 0; --bit) {
    const K cand = bound | ((K)1 << bit);
    if (count(cand) >= k) bound = cand;
  }
  *need = bound == ~(K)0 ? k : k - count(bound + 1);
  return bound;
}

// The k-th largest of n >= k keys (k >= 1) and how many of those equal to it
// are among the k largest.  The keys' range (forced pages aside) is cut into
// as many equal bins as there are threads; the keys of the one bin that holds
// the k-th are ranked by comparisons.
template <typename K>
__device__ K kth_key(const K* keys, int n, unsigned k, PickShared& sh, unsigned* need) {
  constexpr K TOP = ~(K)0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  K lo = TOP, hi = 0;
  unsigned forced = 0;
#pragma unroll 4
  for (int i = tid; i < n; i += kSelThreads) {
    const K x = keys[i];
    if (x == TOP) {
      ++forced;
    } else {
      lo = x < lo ? x : lo;
      hi = x > hi ? x : hi;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const K x = __shfl_xor_sync(0xffffffffu, lo, o), y = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = x < lo ? x : lo;
    hi = y > hi ? y : hi;
  }
  forced = __reduce_add_sync(0xffffffffu, forced);
  __syncthreads();   // what was in sh before has been read
  if (lane == 0) {
    sh.wide[0][warp] = lo;
    sh.wide[1][warp] = hi;
    sh.count[0][warp] = forced;
  }
  sh.hist[tid] = 0;
  if (tid == 0) sh.near = 0;
  __syncthreads();
  unsigned n_forced = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    const K x = (K)sh.wide[0][w], y = (K)sh.wide[1][w];
    lo = x < lo ? x : lo;
    hi = y > hi ? y : hi;
    n_forced += sh.count[0][w];
  }
  if (n_forced >= k) {
    *need = k;
    return TOP;
  }
  k -= n_forced;
  int shift = 0;
  while (((hi - lo) >> shift) >= (K)kSelThreads) ++shift;
#pragma unroll 4
  for (int i = tid; i < n; i += kSelThreads) {
    const K x = keys[i];
    if (x != TOP) atomicAdd(&sh.hist[(unsigned)((x - lo) >> shift)], 1u);
  }
  __syncthreads();
  // Thread t has the t-th bin from the top.
  const unsigned mine = sh.hist[kSelThreads - 1 - tid];
  unsigned incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.count[0][warp] = incl;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) incl += w < warp ? sh.count[0][w] : 0;
  if (incl - mine < k && incl >= k) {   // exactly one thread
    sh.steps[0] = kSelThreads - 1 - tid;
    sh.steps[1] = k - (incl - mine);
    sh.steps[2] = mine;
  }
  __syncthreads();
  const unsigned bin = sh.steps[0], left = sh.steps[1], m = sh.steps[2];
  if (m > kSelNear) {
    K t = kth_key_bits(keys, n, k + n_forced, sh, need);
    return t;
  }
#pragma unroll 4
  for (int i = tid; i < n; i += kSelThreads) {
    const K x = keys[i];
    if (x != TOP && (unsigned)((x - lo) >> shift) == bin)
      sh.near_key[atomicAdd(&sh.near, 1u)] = (unsigned long long)x;
  }
  __syncthreads();
  if (tid < (int)m) {
    const unsigned long long x = sh.near_key[tid];
    unsigned above = 0, same = 0;
    for (unsigned i = 0; i < m; ++i) {
      above += sh.near_key[i] > x;
      same += sh.near_key[i] == x;
    }
    if (above < left && left <= above + same) {   // all threads of the same key
      sh.wide[0][0] = x;
      sh.steps[0] = left - above;
    }
  }
  __syncthreads();
  *need = sh.steps[0];
  return (K)sh.wide[0][0];
}

// Lists the indices i, ascending, of the keys of at least `lo`; of those
// equal to `tie` only the first `need`.  Every warp lists its share.
template <typename K>
__device__ void list_keys(const K* keys, int n, K lo, K tie, unsigned need, int* out,
                          PickShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = ((n + kSelWarps - 1) / kSelWarps + 31) & ~31;
  const int i0 = min(n, warp * share), i1 = min(n, i0 + share);
  unsigned ties = 0, rest = 0;
#pragma unroll 4
  for (int i = i0 + lane; i < i1; i += 32) {
    const K x = keys[i];
    ties += x == tie;
    rest += x >= lo && x != tie;
  }
  ties = __reduce_add_sync(0xffffffffu, ties);
  rest = __reduce_add_sync(0xffffffffu, rest);
  __syncthreads();   // what was in sh before has been read
  if (lane == 0) {
    sh.count[0][warp] = ties;
    sh.count[1][warp] = rest;
  }
  __syncthreads();
  unsigned tie_at = 0, rest_at = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    tie_at += w < warp ? sh.count[0][w] : 0;
    rest_at += w < warp ? sh.count[1][w] : 0;
  }
#pragma unroll 4
  for (int b = i0; b < i1; b += 32) {
    const int i = b + lane;
    const K x = i < i1 ? keys[i] : (K)0;
    const bool t = i < i1 && x == tie, r = i < i1 && x >= lo && x != tie;
    const unsigned bt = __ballot_sync(0xffffffffu, t), br = __ballot_sync(0xffffffffu, r);
    const unsigned below = (1u << lane) - 1u;
    const unsigned at_t = tie_at + __popc(bt & below), at_r = rest_at + __popc(br & below);
    if (r || (t && at_t < need)) out[at_r + min(at_t, need)] = i;
    tie_at += __popc(bt);
    rest_at += __popc(br);
  }
}

// Lists the indices of the keys in [lo, hi], ascending.
__device__ void list_range(const uint32_t* keys, int n, uint32_t lo, uint32_t hi, int* out,
                           PickShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = ((n + kSelWarps - 1) / kSelWarps + 31) & ~31;
  const int i0 = min(n, warp * share), i1 = min(n, i0 + share);
  unsigned in = 0;
  for (int i = i0 + lane; i < i1; i += 32) in += keys[i] >= lo && keys[i] <= hi;
  in = __reduce_add_sync(0xffffffffu, in);
  __syncthreads();
  if (lane == 0) sh.count[0][warp] = in;
  __syncthreads();
  unsigned at = 0;
  for (int w = 0; w < warp; ++w) at += sh.count[0][w];
  for (int b = i0; b < i1; b += 32) {
    const int i = b + lane;
    const bool t = i < i1 && keys[i] >= lo && keys[i] <= hi;
    const unsigned bt = __ballot_sync(0xffffffffu, t);
    if (t) out[at + __popc(bt & ((1u << lane) - 1u))] = i;
    at += __popc(bt);
  }
}

// gridDim.y CTAs per (query, KV head) share its pages out; each writes its
// keys, and the last to arrive picks.  HD 0: any head_dim.
template <typename T, int HD>
__global__ void __launch_bounds__(kSelThreads, sizeof(T) == 4 && HD >= 64 ? 1 : 2)
    paged_select_kernel(const PagedSelectParams p) {
  extern __shared__ uint4 sel_sm[];
  PickShared& sh = *reinterpret_cast<PickShared*>(sel_sm);
  constexpr int OFF_KEYS = (sizeof(PickShared) + 15) & ~15;
  uint32_t* cache = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(sel_sm) + OFF_KEYS);
  uint4* q_s = reinterpret_cast<uint4*>(cache + kSelCached);
  float* q_f = reinterpret_cast<float*>(q_s);
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, s = row / p.n_kv, g = row - s * p.n_kv;
  const int past = p.past[s];
  const int* table = p.table + (size_t)s * p.max_blocks;
  // Warp w: pages 8 w .. 8 w + 7 of a pass; lane (r, qd) reads page r.  The
  // first one's look-up does not wait for the query's length.
  const int first = (HD ? blockIdx.y * kSelWarps * 8 + warp * 8 + (lane >> 2)
                        : blockIdx.y * kSelThreads + tid);
  const int first_page = first < p.max_blocks ? table[first] : 0;
  // Nor do the operands.
  const int hd = HD ? HD : p.hd;
  const float* q = p.q + ((size_t)s * p.n_head + g * p.group) * hd;
  const int hblocks = (p.group + kPagedHeads - 1) / kPagedHeads;
  if constexpr (HD > 0) {
    // Operand of lane l and product u of piece c: dimensions (4 c + qd) * V +
    // u * V / 2 and the following, V to a 16-byte piece.
    using Cfg = ScoreMma<T, HD>;
    constexpr int V = 16 / (int)sizeof(T);
    for (int e = tid; e < hblocks * Cfg::OPERANDS * 32; e += kSelThreads) {
      const int l = e & 31, o = (e >> 5) % Cfg::OPERANDS, hb = (e >> 5) / Cfg::OPERANDS;
      const int u = o & 1, c = (o >> 1) % Cfg::PIECES, low = (o >> 1) / Cfg::PIECES;
      const int h = hb * kPagedHeads + (l >> 2), d = (4 * c + (l & 3)) * V + u * (V / 2);
      float x[4];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        x[i] = h < p.group ? q[h * HD + d + i] : 0.f;
        // The half that this bound is for; NaN belongs to both.
        if (low ? x[i] > 0.f : x[i] < 0.f) x[i] = 0.f;
      }
      uint4 w;
      if constexpr (sizeof(T) == 2) {
        float hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_bf16(x[i], hi[i], lo[i]);
        w = make_uint4(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(lo[0], lo[1]),
                       pack_bf16x2(hi[2], hi[3]), pack_bf16x2(lo[2], lo[3]));
      } else {
        split_tf32(x[0], w.x, w.y);
        split_tf32(x[1], w.z, w.w);
      }
      q_s[e] = w;
    }
  } else {
    for (int e = tid; e < p.group * hd; e += kSelThreads) q_f[e] = q[e];
  }
  int nb = past < 0 ? 0 : (past >> p.log2p) + 1;
  if (past < -1 || nb > p.max_blocks) {
    if (blockIdx.y == 0 && tid == 0) record_error(p.err, kDevErrBadPos);
    nb = 0;
  }
  int* out = p.pages + (size_t)row * p.n_sel;
  if (nb <= p.n_sel) {
    if (blockIdx.y == 0)
      for (int i = tid; i < p.n_sel; i += kSelThreads) out[i] = i < nb ? i : -1;
    return;
  }
  constexpr int PAGES = HD ? kSelWarps * 8 : kSelThreads;   // per pass
  const int ctas = min((int)gridDim.y, (nb + PAGES - 1) / PAGES);
  if ((int)blockIdx.y >= ctas) return;
  __syncthreads();
  const bool alone = ctas == 1, cached = nb <= kSelCached;
  // Scratch of the row: binary64 keys, then three arrays of 32-bit words.
  unsigned long long* wide = p.keys + (size_t)row * 3 * p.max_blocks;
  uint32_t* keys_g = reinterpret_cast<uint32_t*>(wide + p.max_blocks);
  int* near_g = reinterpret_cast<int*>(keys_g + p.max_blocks);
  int* taken_g = near_g + p.max_blocks;
  float* big_g = reinterpret_cast<float*>(near_g);   // of the CTAs, until one picks
  uint32_t* keys = alone && cached ? cache : keys_g;
  const int stride = ctas * PAGES;
  float big = 0.f;
  if constexpr (HD > 0) {
    const int r = lane >> 2, qd = lane & 3;
    constexpr int PIECES = ScoreMma<T, HD>::PIECES;
    int j0 = blockIdx.y * PAGES + warp * 8;
    // Columns behind the last page repeat the warp's first one.  (They took
    // page 0 of the pool, whatever it held, and its bounds raised E: with NaN
    // there 4 x 8192 pages took 763 us in place of 21.)
    auto column = [&](int j, int page) -> int {
      const int first_column = __shfl_sync(0xffffffffu, page, 0);
      return j + r < nb ? page : first_column;
    };
    auto bounds_of = [&](int page) -> const T* {
      const bool bad = page < 0 || page >= p.n_pages;
      if (bad && qd == 0) record_error(p.err, kDevErrBadPage);
      return static_cast<const T*>(p.bounds) + ((size_t)(bad ? 0 : page) * p.n_kv + g) * 2 * HD;
    };
    auto entry = [&](int j) { return j + r < nb ? table[j + r] : 0; };
    uint4 b[2][PIECES];
    if (j0 < nb) load_bounds<T, HD>(bounds_of(column(j0, first_page)), b);
    int page = entry(j0 + stride);
    for (; j0 < nb; j0 += stride) {
      // The next pass's bounds and the page of the one after are on their way.
      uint4 b_n[2][PIECES];
      const bool more = j0 + stride < nb;
      if (more) load_bounds<T, HD>(bounds_of(column(j0 + stride, page)), b_n);
      page = entry(j0 + 2 * stride);
      const float2 x = page_scores<T, HD>(b, q_s, hblocks,
                                          p.group - (hblocks - 1) * kPagedHeads, &big);
      if (r < 2) {
        const int j = j0 + 2 * qd + r;
        if (j < nb)
          keys[j] = j < p.keep_first || j >= nb - p.keep_last ? kKeyForced
                                                              : ordered_key(r ? x.y : x.x);
      }
      if (more)
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
          b[0][c] = b_n[0][c];
          b[1][c] = b_n[1][c];
        }
    }
  } else {
    for (int j = first; j < nb; j += stride) {
      int page = j == first ? first_page : table[j];
      const bool bad = page < 0 || page >= p.n_pages;
      if (bad) {
        record_error(p.err, kDevErrBadPage);
        page = 0;
      }
      const T* lo = static_cast<const T*>(p.bounds) + ((size_t)page * p.n_kv + g) * 2 * hd;
      const float x = page_score_any<T>(lo, q_f, p.group, hd, &big);
      keys[j] = j < p.keep_first || j >= nb - p.keep_last ? kKeyForced : ordered_key(x);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  if (lane == 0) sh.big[warp] = big;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) big = fmaxf(big, sh.big[w]);
  if (!alone) {
    if (tid == 0) big_g[blockIdx.y] = big;
    __syncthreads();
    if (tid == 0) sh.flag = arrive_acq_rel(p.count + row) == (unsigned)(ctas - 1);
    __syncthreads();
    if (!sh.flag) return;
    if (tid == 0) p.count[row] = 0;
    for (int i = tid; i < ctas; i += kSelThreads) big = fmaxf(big, __ldcg(big_g + i));
    if (cached) {
#pragma unroll 4
      for (int i = tid; i < nb; i += kSelThreads) cache[i] = __ldcg(keys + i);
      keys = cache;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    if (lane == 0) sh.big[warp] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) big = fmaxf(big, sh.big[w]);
  }
  // E, with S = big * sum |q| >= the sum of a score's absolute terms: 2 hd
  // products and hd / 8 partial sums, each added with an error of at most
  // 2^-23 S (the tensor cores may truncate), and 2^-17 S of split operands.
  // What is below 2^-126 may count as zero, parts of q and of bounds, products
  // and sums: at most 2^-123 (big + sum |q| + 1) per dimension.
  float sum_q = 0.f;
  for (int h = warp; h < p.group; h += kSelWarps) {
    float x = 0.f;
    for (int d = lane; d < hd; d += 32) x += fabsf(q[h * hd + d]);
    sum_q = fmaxf(sum_q, warp_sum(x));
  }
  __syncthreads();
  if (lane == 0) sh.big[warp] = sum_q;
  unsigned need;
  const uint32_t t_key = kth_key<uint32_t>(keys, nb, (unsigned)p.n_sel, sh, &need);
  if (t_key == kKeyForced) {   // more forced pages than places
    list_keys<uint32_t>(keys, nb, kKeyForced, kKeyForced, need, out, sh);
    return;
  }
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) sum_q = fmaxf(sum_q, sh.big[w]);
  const float E2 = 2.02f * (2.125f * hd * 1.1920929e-7f + 7.6293945e-6f) * big * sum_q   // 2 E, and its own roundings
                   + 0x1p-122f * hd * (big + sum_q + 1.f);
  uint32_t k_lo = 0, k_hi = kKeyForced - 1;
  if (E2 < INFINITY) {
    const float t = key_value(t_key);
    k_lo = ordered_key(__fsub_rd(t, E2));
    k_hi = ordered_key(__fadd_ru(t, E2));
  }
  __syncthreads();
  if (tid == 0) sh.near = sh.sure = 0;
  __syncthreads();
  // Pages near the border, and those surely taken.
  unsigned near = 0, sure = 0;
  for (int i = tid; i < nb; i += kSelThreads) {
    const uint32_t x = keys[i];
    sure += x > k_hi;
    if (x >= k_lo && x <= k_hi) {
      const unsigned at = atomicAdd(&sh.near, 1u);
      if (at < kSelNear) {
        sh.near_at[at] = i;
        sh.near_page[at] = table[i];
      }
    }
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  if (lane == 0 && sure) atomicAdd(&sh.sure, sure);
  __syncthreads();
  near = sh.near;
  sure = sh.sure;
  if (sure + near == (unsigned)p.n_sel) {   // all of them
    list_keys<uint32_t>(keys, nb, k_lo, 0u, 0u, out, sh);
    return;
  }
  // Not all: in the order of their binary64 scores, ties to the lower index.
  const unsigned left = (unsigned)p.n_sel - sure;
  const bool few = near <= kSelNear;
  if (!few) {
    list_range(keys, nb, k_lo, k_hi, near_g, sh);
    __syncthreads();
  }
  for (unsigned i = tid; i < near; i += kSelThreads) (few ? sh.near_key : wide)[i] = 0ull;
  __syncthreads();
  // Eight lanes per (page, head); NaN is above every key while the heads meet.
  const unsigned pairs = near * p.group;
  for (unsigned e0 = 4 * warp; e0 < pairs; e0 += 4 * kSelWarps) {
    // (The lanes behind the last pair take it too.)
    const unsigned e = min(e0 + (lane >> 3), pairs - 1), i = e / p.group, h = e - i * p.group;
    const int pg = few ? sh.near_page[i] : table[near_g[i]];
    const bool bad = pg < 0 || pg >= p.n_pages;
    const T* lo = static_cast<const T*>(p.bounds) + ((size_t)(bad ? 0 : pg) * p.n_kv + g) * 2 * hd;
    const double x = exact_score<T, HD>(lo, q + (size_t)h * hd, hd);
    if ((lane & 7) == 0)
      atomicMax(&(few ? sh.near_key : wide)[i], bad || x != x ? ~0ull : ordered_key(x));
  }
  __syncthreads();
  for (unsigned i = tid; i < near; i += kSelThreads) {
    unsigned long long* x = &(few ? sh.near_key : wide)[i];
    if (*x == ~0ull) *x = 0ull;   // NaN ranks last
  }
  __syncthreads();
  if (few) {
    if (tid < (int)near) {
      const unsigned long long x = sh.near_key[tid];
      const int at = sh.near_at[tid];
      unsigned above = 0;
      for (unsigned i = 0; i < near; ++i) {
        const unsigned long long y = sh.near_key[i];
        above += y > x || (y == x && sh.near_at[i] < at);
      }
      if (above < left) keys[at] = kKeyForced;
    }
  } else {
    unsigned ties;
    const unsigned long long t64 = kth_key<unsigned long long>(wide, (int)near, left, sh, &ties);
    list_keys<unsigned long long>(wide, (int)near, t64, t64, ties, taken_g, sh);
    __syncthreads();
    for (unsigned i = tid; i < left; i += kSelThreads) keys[near_g[taken_g[i]]] = kKeyForced;
  }
  __syncthreads();
  list_keys<uint32_t>(keys, nb, k_hi + 1, 0u, 0u, out, sh);
}

template <typename T, int HD>
static cudaError_t launch_select_cfg(const PagedSelectParams& p, int num_sms, cudaStream_t st) {
  static bool done[64] = {};
  cudaError_t e = allow_max_smem(paged_select_kernel<T, HD>, done);
  if (e != cudaSuccess) return e;
  const int hblocks = (p.group + kPagedHeads - 1) / kPagedHeads;
  const size_t q_bytes = HD ? (size_t)hblocks * ScoreMma<T, HD ? HD : 64>::OPERANDS * 32 * 16
                            : (size_t)p.group * p.hd * 4;
  const size_t smem = ((sizeof(PickShared) + 15) & ~size_t(15)) + (size_t)kSelCached * 4 + q_bytes;
  // Two CTAs fit an SM; more than one per row only while there are SMs
  // without one and pages for another pass.
  const int pages = HD ? kSelWarps * 8 : kSelThreads;
  const int most = (p.max_blocks + pages - 1) / pages;
  int ctas = 2 * num_sms / (p.n * p.n_kv);
  if (ctas > most) ctas = most;
  if (ctas < 1) ctas = 1;
  return launch_chained(paged_select_kernel<T, HD>, dim3((unsigned)(p.n * p.n_kv), (unsigned)ctas),
                        dim3(kSelThreads), smem, st, p);
}

template <typename T>
static cudaError_t launch_select_type(const PagedSelectParams& p, int num_sms, cudaStream_t st) {
  switch (p.hd) {
    case 32: return launch_select_cfg<T, 32>(p, num_sms, st);
    case 64: return launch_select_cfg<T, 64>(p, num_sms, st);
    case 128: return launch_select_cfg<T, 128>(p, num_sms, st);
    default: return launch_select_cfg<T, 0>(p, num_sms, st);
  }
}

cudaError_t launch_paged_select(const PagedSelectParams& p, int num_sms, cudaStream_t st) {
  return p.dtype == 1 ? launch_select_type<__nv_bfloat16>(p, num_sms, st)
                      : launch_select_type<float>(p, num_sms, st);
}

}  // namespace tg
