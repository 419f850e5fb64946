// tg_paged_prefix.cu -- decode attention over the shared prefix of a batch on
// the 5th-generation tensor cores (tcgen05 + TMEM), and the merge of its
// softmax records with those of the queries' own rows (tg_paged.cu).  No
// counterpart in the reference, which decodes one sequence at a time.
//
// The queries of one KV head over the same keys are a matrix: row
// s * group + h of n * group rows.  For 128 rows x 64 keys the products
// S = Q K^T and O += P V run on tcgen05, and a key is read once for 256 rows
// instead of once for 8.
//
// Against the exact bf16 keys q is three bf16, all its 24 bits, since an error
// of a score grows with the score: with two (17 bits) the largest error, over
// the largest result, was 1.3e-5 at scores of 4 times the usual size and 5e-5
// at 16, where a plain binary32 form has 3e-6 and 9e-6 (with three: 3e-6 and
// 3e-6).  The third part costs 2.4 us of 67 at the size below.  The
// probabilities are two bf16: what that leaves out, 2^-18 of each, has no
// common sign over the keys.
//
// A step (64 keys for two slots of 128 rows) costs an SM 1280 cycles of tensor
// core (two slots x (12 + 8) products of 128 x 64 x 16 at 4096 multiply-adds a
// cycle) and 1024 cycles of ex2 (16 per cycle).  128 queries x 14 / 2 heads
// over 32768 rows are 28 steps per CTA, 19 us of products; the kernel takes
// 43, 2200 cycles a step: products and softmax of a slot wait for each other,
// and the two slots overlap far less than they could.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tg_device.cuh"
#include "tg_launch.cuh"
#include "tg_paged.h"
#include "tg_shared.h"
#include "tg_tc.cuh"

namespace tg {

constexpr int PX_ROWS = 128;        // query rows of a slot (TMEM lanes)
constexpr int PX_KEYS = 64;         // keys of a step
constexpr int PX_STAGES = 8;        // K/V ring
constexpr int PX_FLUSH = 16;        // steps that O gathers in TMEM
constexpr int PX_THREADS = 384;     // TMA warp, 2 MMA warps, an idle one, 2 x 4 softmax warps
constexpr int PX_TILE = PX_KEYS * 128;           // bytes of a K (or V) tile
constexpr int PX_OFF_Q = PX_STAGES * 2 * PX_TILE;   // 8 KB per softmax warp: q on its way to
                                                    // TMEM, then what O has gathered
constexpr int PX_OFF_Q3 = PX_OFF_Q + 8 * 32 * 64 * 4;   // third parts of q: a 128 x 64 operand
                                                       // per slot, 128-byte swizzle
constexpr int PX_Q3 = PX_ROWS * 128;
constexpr int PX_OFF_BAR = PX_OFF_Q3 + 2 * PX_Q3;
// kv_full[S], kv_empty[S], q_full[slot], s_full[slot][buf], p_full[slot][buf],
// pv_done[slot], drained[slot]
constexpr int PX_NBAR = 2 * PX_STAGES + 2 + 4 + 4 + 2 + 2;
constexpr int PX_OFF_MISC = PX_OFF_BAR + PX_NBAR * 8;
constexpr size_t PX_SMEM = 1024 + PX_OFF_MISC + 16;
static_assert(PX_SMEM <= 227 * 1024, "shared memory");
constexpr uint32_t PX_COLS = 512;
// TMEM columns of slot x from 256 x: two buffers of 64 (S as binary32, then P
// in its place: 32 columns hi, 32 lo, two bf16 each), O 64, Q 64 (lo, hi).
__device__ __forceinline__ uint32_t px_s(int x, int buf) { return 256u * x + 64u * buf; }
__device__ __forceinline__ uint32_t px_o(int x) { return 256u * x + 128u; }
__device__ __forceinline__ uint32_t px_q(int x) { return 256u * x + 192u; }

__device__ __forceinline__ bool px_wait(uint64_t* bar, uint32_t parity, int* err,
                                        volatile int* abort_flag) {
  if (*abort_flag) return false;
  if (mbar_wait(bar, parity, err, kDevErrWaitFull)) return true;
  *abort_flag = 1;
  return false;
}

// Every lane polls (and so acquires the phase itself), then the warp agrees.
// The usual case, a phase that is already complete, reads nothing else.
__device__ __forceinline__ bool px_wait_warp(uint64_t* bar, uint32_t parity, int* err,
                                             volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const bool got = px_wait(bar, parity, err, abort_flag);
  return __all_sync(0xffffffffu, got) != 0;
}

// Pairs of floats in 64-bit registers, added by one instruction, and the
// maximum of three: the softmax is bound by the issue of its instructions
// beside those of the ex2 unit.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two floats as two pairs of bf16, the rounded values and what they leave,
// rounded: 16 bits and a sign, off by at most 2^-18.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(a, b);
  // a - its rounded value, the latter with its sign turned.
  const uint64_t rest = add_pair(f32x2(a, b), f32x2(__uint_as_float((hi << 16) ^ 0x80000000u),
                                                    __uint_as_float((hi & 0xffff0000u) ^ 0x80000000u)));
  float ra, rb;
  unpair(rest, ra, rb);
  lo = pack_bf16x2(ra, rb);
}

// One CTA: 256 query rows of a KV head (two slots of 128) x a range of the
// prefix's keys, both slots over the same keys.  With at most 128 rows
// (p.single) both slots hold the same rows and each takes half of the keys.
//   warp 0      TMA: K and V tiles of 64 keys (boxes of min(page, 32) rows,
//               128-byte swizzle) into a ring; the pages of the next tile are
//               looked up while this one is issued.
//   warps 1, 2  issue the products of a slot each (one warp for both spent
//               900 of 2200 cycles of a step in waits and bookkeeping while
//               the tensor core stood still); warp 1 owns TMEM.  S of step
//               j + 2 goes into the buffer that P of step j has just been
//               read from (products of one thread run in their order), so S
//               is ready when a softmax warp comes for it.
//   warps 4-11  softmax, a thread per query row: S to registers, running
//               maximum (the exponent's base moves only when the maximum
//               grew by more than 2^8; then O is rescaled in TMEM), P = 2^(S
//               - m) split into hi and lo in place of S.
// Every wait is bounded; a failed one raises the abort flag, every role
// leaves its loop, issued loads and products are drained and TMEM is freed.
__global__ void __launch_bounds__(PX_THREADS, 1)
    paged_prefix_kernel(const __grid_constant__ CUtensorMap tmk,
                        const __grid_constant__ CUtensorMap tmv, const PagedPrefixParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + PX_OFF_BAR);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = kv_full + PX_STAGES;
  uint64_t* q_full = kv_empty + PX_STAGES;
  uint64_t* s_full = q_full + 2;   // [slot * 2 + buf]
  uint64_t* p_full = s_full + 4;   // [slot * 2 + buf]
  uint64_t* pv_done = p_full + 4;  // [slot]: the last two steps' O
  uint64_t* drained = pv_done + 2; // [slot]: everything issued has completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + PX_OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + PX_OFF_MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Item: KV head, pair of row tiles, range of key steps.
  const int split = blockIdx.x % p.splits, gp = blockIdx.x / p.splits;
  const int g = gp / p.pairs, pair = gp - g * p.pairs;
  const int k0 = (int)((long long)split * p.steps / p.splits);
  const int k1 = (int)((long long)(split + 1) * p.steps / p.splits);
  const int rows = p.n * p.group;
  const bool both = p.single || (2 * pair + 1) * PX_ROWS < rows;   // slot 1 has rows
  // Steps of the slots, and the tile (from k0) of ring entry i.
  const int n0 = p.single ? (k1 - k0 + 1) / 2 : k1 - k0;
  const int n1 = p.single ? (k1 - k0) / 2 : (both ? k1 - k0 : 0);
  const int entries = k1 - k0;
  auto tile_of = [&](int i) { return p.single ? ((i & 1) ? n0 + (i >> 1) : i >> 1) : i; };

  griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < PX_STAGES; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], !p.single && both ? 2 : 1);   // the slots that read an entry
    }
    mbar_init(&q_full[0], 4);
    mbar_init(&q_full[1], 4);
    mbar_init(&drained[0], 1);
    mbar_init(&drained[1], 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(PX_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  if (warp == 0) {
    // ---------------------------------------------------------- TMA
    const int box = min(1 << p.log2p, 32), lbox = min(p.log2p, 5), nbx = PX_KEYS >> lbox;
    auto look_up = [&](int i) -> int {   // lane b: TMA row of box b of entry i
      if (lane >= nbx) return 0;
      const int r = (k0 + tile_of(i)) * PX_KEYS + (lane << lbox);
      int page = p.table[r >> p.log2p];
      if (page < 0 || page >= p.n_pages) {
        record_error(p.err, kDevErrBadPage);
        page = 0;
      }
      return (int)(((p.page0 + page) * p.n_kv + g) << p.log2p) + (r & ((1 << p.log2p) - 1));
    };
    int y = entries > 0 ? look_up(0) : 0, issued = 0;
    for (int i = 0; i < entries; ++i) {
      const int y_n = i + 1 < entries ? look_up(i + 1) : 0;
      const int st = i % PX_STAGES;
      if (!px_wait_warp(&kv_empty[st], (uint32_t)(((i / PX_STAGES) & 1) ^ 1), p.err, abort_flag))
        break;
      if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], 2 * PX_TILE);
      uint8_t* to = smem + st * 2 * PX_TILE;
      for (int b = 0; b < nbx; ++b) {
        const int yb = __shfl_sync(0xffffffffu, y, b);
        if (lane == 0) {
          tma_load_2d(to + b * box * 128, &tmk, &kv_full[st], 0, yb);
          tma_load_2d(to + PX_TILE + b * box * 128, &tmv, &kv_full[st], 0, yb);
        }
      }
      y = y_n;
      ++issued;
    }
    for (int i = max(0, issued - PX_STAGES); i < issued; ++i)
      mbar_wait(&kv_full[i % PX_STAGES], (uint32_t)((i / PX_STAGES) & 1), p.err, kDevErrWaitFull);
  } else if (warp <= 2) {
    // ---------------------------------------------------------- products
    // The whole warp walks the loop, one lane issues (see umma_f16_ts_x8).
    constexpr uint32_t IDESC_QK = idesc_bf16(PX_ROWS, PX_KEYS, false);
    constexpr uint32_t IDESC_PV = idesc_bf16(PX_ROWS, 64, true);
    const uint64_t dk0 = smem_desc_sw128(smem_u32(smem), 16, 1024);
    const uint64_t dv0 = smem_desc_sw128(smem_u32(smem) + PX_TILE, PX_TILE, 1024);
    const int x = (int)__reduce_max_sync(0xffffffffu, threadIdx.x >> 5) - 1;   // warp-uniform
    const uint64_t dq3 = smem_desc_sw128(smem_u32(smem) + PX_OFF_Q3 + x * PX_Q3, 16, 1024);
    const uint32_t base = __reduce_max_sync(0xffffffffu, tmem) + 256u * x;
    const int n = x ? n1 : n0;
    // This slot's ring entries: x, x + 2, ... (single) or 0, 1, ...  qk is the
    // one of the next S, pv the one of the next O.
    const int by = p.single ? 2 : 1;
    struct Ring {
      int st;
      uint32_t ph;
      __device__ __forceinline__ void step(int by) {
        st += by;
        if (st >= PX_STAGES) {
          st -= PX_STAGES;
          ph ^= 1u;
        }
      }
    };
    Ring qk{p.single ? x : 0, 0u}, pv{p.single ? x : 0, 0u};
    auto issue_qk = [&](int j) -> bool {
      if (!px_wait_warp(&kv_full[qk.st], qk.ph, p.err, abort_flag)) return false;
      tc_fence_after();
      // 4 steps of 16 dimensions (32 bytes), the third parts, the low and the
      // high ones: what the tensor core truncates is small while the sum is.
      const uint64_t dk = dk0 + (uint64_t)(qk.st * (2 * PX_TILE >> 4));
      umma_f16_ss_x4<2, 2>(base + px_s(0, j & 1), dq3, dk, IDESC_QK, 0u);
      umma_f16_ts_x8<2>(base + px_s(0, j & 1), base + px_q(0), dk, IDESC_QK, 1u);
      umma_commit_elect(&s_full[2 * x + (j & 1)]);
      qk.step(by);
      return true;
    };
    bool ok = n > 0 && px_wait_warp(&q_full[x], 0, p.err, abort_flag);
    const bool any = ok;
    for (int j = 0; j < 2 && ok; ++j)
      if (j < n) ok = issue_qk(j);
    for (int j = 0; j < n && ok; ++j) {
      if (!px_wait_warp(&p_full[2 * x + (j & 1)], (uint32_t)((j >> 1) & 1), p.err, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // 4 steps of 16 keys (2048 bytes), the high parts and the low ones.
      umma_f16_ts_x8<128>(base + px_o(0), base + px_s(0, j & 1),
                          dv0 + (uint64_t)(pv.st * (2 * PX_TILE >> 4)), IDESC_PV,
                          j % PX_FLUSH != 0 ? 1u : 0u);
      umma_commit_elect(&kv_empty[pv.st]);
      pv.step(by);
      // Products of one thread complete in their order: s_full of step j + 2
      // covers this one.  The last two steps have no such product.
      if (j + 2 >= n)
        umma_commit_elect(&pv_done[x]);
      else
        ok = issue_qk(j + 2);
    }
    // Everything issued has completed before TMEM is freed.
    if (any) {
      umma_commit_elect(&drained[x]);
      mbar_wait(&drained[x], 0, p.err, kDevErrWaitFull);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------- softmax
    const int x = (warp - 4) >> 2, quarter = warp & 3;
    const int row = (p.single ? 0 : (2 * pair + x) * PX_ROWS) + quarter * 32 + lane;
    const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16);
    const int steps = x ? n1 : n0;
    {
      // This row of Q, scaled to log2 units, as lo and hi in TMEM and a third
      // part, for which TMEM has no room, in shared memory.  The warp reads its
      // 32 rows one by one, whole, and turns them in shared memory (a lane
      // reading a row by itself touched a line per lane and load, 8000 cycles
      // for the 8 warps).
      float2* turn = reinterpret_cast<float2*>(smem + PX_OFF_Q) + (warp - 4) * 32 * 32;
      const int row0 = row - lane, live = min(32, rows - row0);
      int hi = row0 % p.group;
      const float2* q = reinterpret_cast<const float2*>(
                            p.q + ((size_t)(row0 / p.group) * p.n_head + g * p.group + hi) * 64) +
                        lane;
      float2 v[32];   // all on their way before the first is used
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = i < live ? *q : make_float2(0.f, 0.f);
        const bool next = ++hi == p.group;   // the next query's heads of this KV head
        q += next ? (p.n_head - p.group + 1) * 32 : 32;
        hi = next ? 0 : hi;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) turn[i * 32 + (lane ^ i)] = v[i];
      __syncwarp();
      uint32_t w[64], third[4];
      const int r128 = quarter * 32 + lane;
      uint8_t* q3 = smem + PX_OFF_Q3 + x * PX_Q3 + r128 * 128;
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const float2 v = turn[lane * 32 + (c ^ lane)];
        float h0, l0, h1, l1, r0, r1;
        split_bf16(v.x * p.scale_log2, h0, r0);
        split_bf16(v.y * p.scale_log2, h1, r1);
        split_bf16(r0, l0, r0);
        split_bf16(r1, l1, r1);
        w[c] = pack_bf16x2(l0, l1);
        w[32 + c] = pack_bf16x2(h0, h1);
        third[c & 3] = pack_bf16x2(r0, r1);
        if ((c & 3) == 3)
          *reinterpret_cast<uint4*>(q3 + (((c >> 2) ^ (r128 & 7)) << 4)) =
              make_uint4(third[0], third[1], third[2], third[3]);
      }
      fence_proxy_async_smem();   // the tensor core reads them
      TG_TMEM_ST64(base + px_q(x), w);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[x]);
    }
    constexpr float kLazy = 8.f;
    float m = kNegBig, l = 0.f;
    // The tensor cores truncate what they add to an accumulator: with O in
    // TMEM for all of 28 steps the result was off by 5.5e-6.  So every
    // PX_FLUSH steps it goes to shared memory (piece c of a row at c * 32 +
    // lane), in units of 2^m_acc, and begins again; a step that does so takes
    // about 900 cycles longer.
    float4* acc = reinterpret_cast<float4*>(smem + PX_OFF_Q) + (warp - 4) * 16 * 32 + lane;
    float m_acc = kNegBig;
    bool gathered = false, ok = true;
    for (int j = 0; j < steps; ++j) {
      const int b = j & 1;
      if (!px_wait_warp(&s_full[2 * x + b], (uint32_t)((j >> 1) & 1), p.err, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[64];
      TG_TMEM_LD64(base + px_s(x, b), sv);
      float mx4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(__uint_as_float(sv[c]), __uint_as_float(sv[4 + c]));
#pragma unroll
      for (int c = 8; c < 64; c += 2)
        mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(sv[c]), __uint_as_float(sv[c + 1]));
      const float mx = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3]));
      float alpha = 1.f;
      if (j == 0) {
        m = fmaxf(mx, kNegBig);
      } else if (mx - m > kLazy) {
        alpha = ex2(m - mx);
        m = mx;
      }
      const bool flush = j > 0 && j % PX_FLUSH == 0;
      if (flush || __any_sync(0xffffffffu, alpha != 1.f)) {
        // O of the steps before this one is complete once S of the next step
        // is (or, in the last step, the product before it), and the next
        // product on O waits for this step's P.
        uint64_t* bar = j + 1 < steps ? &s_full[2 * x + (b ^ 1)] : &pv_done[x];
        const uint32_t phase = j + 1 < steps ? (uint32_t)(((j + 1) >> 1) & 1) : 0u;
        if (!px_wait_warp(bar, phase, p.err, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < 64; c0 += 32) {
          uint32_t ov[32];
          TG_TMEM_LD32(base + px_o(x) + c0, ov);
#pragma unroll
          for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
          if (!flush) {
            TG_TMEM_ST32(base + px_o(x) + c0, ov);
          } else {
            const float f = ex2(m_acc - m);
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              float4 v = make_float4(__uint_as_float(ov[c]), __uint_as_float(ov[c + 1]),
                                     __uint_as_float(ov[c + 2]), __uint_as_float(ov[c + 3]));
              float4* to = acc + ((c0 + c) >> 2) * 32;
              if (gathered) {
                const float4 a = *to;
                v = make_float4(fmaf(a.x, f, v.x), fmaf(a.y, f, v.y), fmaf(a.z, f, v.z),
                                fmaf(a.w, f, v.w));
              }
              *to = v;
            }
          }
        }
        if (flush) {
          gathered = true;
          m_acc = m;
        }
      }
      uint64_t ls[4] = {0, 0, 0, 0};   // pairs of zeros
      const uint64_t neg = f32x2(-m, -m);
      uint32_t w[64];
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        float p0, p1;
        unpair(add_pair(f32x2(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), neg), p0, p1);
        p0 = ex2(p0);
        p1 = ex2(p1);
        ls[c & 3] = add_pair(ls[c & 3], f32x2(p0, p1));
        split_pair(p0, p1, w[c], w[32 + c]);
      }
      TG_TMEM_ST64(base + px_s(x, b), w);
      float l0, l1;
      unpair(add_pair(add_pair(ls[0], ls[1]), add_pair(ls[2], ls[3])), l0, l1);
      l = l * alpha + (l0 + l1);
      // The last step first sees the product before it complete: once it has
      // handed its P on, that phase may be two behind, which a parity cannot
      // tell from the one to come.
      if (j > 0 && j + 1 == steps && !px_wait_warp(&pv_done[x], 0, p.err, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * x + b]);
    }
    uint32_t ov[64];
    if (ok && steps > 0)
      ok = px_wait_warp(&pv_done[x], steps > 1 ? 1u : 0u, p.err, abort_flag);
    if (ok && steps > 0) {
      tc_fence_after();
      TG_TMEM_LD64(base + px_o(x), ov);
      tc_fence_before();
      if (gathered) {
        const float f = ex2(m_acc - m);
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          const float4 a = acc[(c >> 2) * 32];
          ov[c] = __float_as_uint(fmaf(a.x, f, __uint_as_float(ov[c])));
          ov[c + 1] = __float_as_uint(fmaf(a.y, f, __uint_as_float(ov[c + 1])));
          ov[c + 2] = __float_as_uint(fmaf(a.z, f, __uint_as_float(ov[c + 2])));
          ov[c + 3] = __float_as_uint(fmaf(a.w, f, __uint_as_float(ov[c + 3])));
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 64; ++c) ov[c] = 0u;
      m = kNegBig;
      l = 0.f;
    }
    if (row < rows) {
      const int part = p.single ? 2 * split + x : split;
      // Column by column: a warp's 32 rows are neighbours there.
      float* rec = p.records + ((size_t)part * p.n_kv + g) * 66 * rows + row;
#pragma unroll
      for (int c = 0; c < 64; ++c) rec[(size_t)c * rows] = __uint_as_float(ov[c]);
      rec[(size_t)64 * rows] = m;
      rec[(size_t)65 * rows] = l;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PX_COLS)
                 : "memory");
  }
}

// out of every (query, head): the records of the prefix (for queries that
// attend all of it) and the record of the query's own rows.  A CTA takes 32
// rows of one KV head and 16 of the 64 dimensions: first lane = row (the
// records' columns are contiguous), 8 warps = 2 halves of the dimensions x 4
// groups of parts, joined in shared memory; then 8 threads per row, so that
// the output is written in runs.
constexpr int kPrefixMergeWarps = 8, kMergeDims = 16;

__global__ void __launch_bounds__(32 * kPrefixMergeWarps)
    paged_prefix_merge_kernel(const PagedPrefixParams p) {
  constexpr int B = 4, GRP = 4, DW = kMergeDims / (kPrefixMergeWarps / GRP);
  __shared__ float o_s[GRP][32][kMergeDims + 1];
  __shared__ float ml_s[GRP][2][32];
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.n * p.group, blocks = (rows + 31) / 32;
  const int g = blockIdx.x / blocks, row0 = (blockIdx.x - g * blocks) * 32;
  const int d0 = blockIdx.y * kMergeDims;
  {
    const int grp = warp % GRP, dw = (warp / GRP) * DW;
    const int row = row0 + lane;
    const int past = row < rows ? p.past[row / p.group] : -1;
    const bool live = past >= p.steps * PX_KEYS - 1 && past < p.limit;
    const float* rec = p.records + (size_t)g * 66 * rows + (live ? row : 0);
    const size_t part_stride = (size_t)p.n_kv * 66 * rows;
    float M = kNegBig, L = 0.f, O[DW];
#pragma unroll
    for (int c = 0; c < DW; ++c) O[c] = 0.f;
    const int parts = live ? p.parts : 0;
    for (int k0 = grp; k0 < parts; k0 += GRP * B) {
      float m[B], l[B], o[B][DW];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int k = k0 + u * GRP;
        m[u] = kNegBig;
        l[u] = 0.f;
#pragma unroll
        for (int c = 0; c < DW; ++c) o[u][c] = 0.f;
        if (k < parts) {
          const float* r = rec + (size_t)k * part_stride;
          m[u] = r[(size_t)64 * rows];
          l[u] = r[(size_t)65 * rows];
#pragma unroll
          for (int c = 0; c < DW; ++c) o[u][c] = r[(size_t)(d0 + dw + c) * rows];
        }
      }
      float mb = M;
#pragma unroll
      for (int u = 0; u < B; ++u) mb = fmaxf(mb, m[u]);
      const float w0 = ex2(M - mb);
      M = mb;
      L *= w0;
#pragma unroll
      for (int c = 0; c < DW; ++c) O[c] *= w0;
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const float w = ex2(m[u] - M);
        L = fmaf(l[u], w, L);
#pragma unroll
        for (int c = 0; c < DW; ++c) O[c] = fmaf(o[u][c], w, O[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < DW; ++c) o_s[grp][lane][dw + c] = O[c];
    if (dw == 0) {
      ml_s[grp][0][lane] = M;
      ml_s[grp][1][lane] = L;
    }
  }
  __syncthreads();
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 2;   // 8 threads per row
  if (row0 + r >= rows) return;
  const int row = row0 + r, s = row / p.group, h = g * p.group + row - s * p.group;
  const float* own = p.own + ((size_t)s * p.n_head + h) * 66;
  float2 O = *reinterpret_cast<const float2*>(own + d0 + c);
  const float2 ml = *reinterpret_cast<const float2*>(own + 64);
  float M = ml.x;
#pragma unroll
  for (int k = 0; k < GRP; ++k) M = fmaxf(M, ml_s[k][0][r]);
  const float w = ex2(ml.x - M);
  float L = ml.y * w;
  O.x *= w;
  O.y *= w;
#pragma unroll
  for (int k = 0; k < GRP; ++k) {
    const float f = ex2(ml_s[k][0][r] - M);
    L = fmaf(ml_s[k][1][r], f, L);
    O.x = fmaf(o_s[k][r][c], f, O.x);
    O.y = fmaf(o_s[k][r][c + 1], f, O.y);
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  *reinterpret_cast<float2*>(p.out + ((size_t)s * p.n_head + h) * 64 + d0 + c) =
      make_float2(O.x * inv, O.y * inv);
}

// ------------------------------------------------------------ launches

cudaError_t launch_paged_prefix(const CUtensorMap& tk, const CUtensorMap& tv,
                                const PagedPrefixParams& p, cudaStream_t st) {
  static bool done[64] = {};
  cudaError_t e = allow_max_smem(paged_prefix_kernel, done);
  if (e != cudaSuccess) return e;
  return launch_chained(paged_prefix_kernel, dim3((unsigned)(p.n_kv * p.pairs * p.splits)),
                        dim3(PX_THREADS), PX_SMEM, st, tk, tv, p);
}

cudaError_t launch_paged_prefix_merge(const PagedPrefixParams& p, cudaStream_t st) {
  return launch_chained(paged_prefix_merge_kernel,
                        dim3((unsigned)(p.n_kv * ((p.n * p.group + 31) / 32)), 64 / kMergeDims),
                        dim3(32 * kPrefixMergeWarps), 0, st, p);
}

void plan_paged_prefix(PagedPrefixParams* p, int num_sms) {
  const int tiles = (p->n * p->group + PX_ROWS - 1) / PX_ROWS;
  p->single = tiles == 1 ? 1 : 0;
  p->pairs = (tiles + 1) / 2;
  // One CTA per SM where the rows leave room for it, each with at least 2
  // steps per slot.
  const int most = p->steps / (p->single ? 4 : 2);
  p->splits = num_sms / (p->n_kv * p->pairs);
  if (p->splits > most) p->splits = most;
  if (p->splits < 1) p->splits = 1;
  p->parts = p->single ? 2 * p->splits : p->splits;
}

}  // namespace tg
