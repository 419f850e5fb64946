// tg_paged.h -- parameters and launchers of the paged-cache kernels
// (tg_paged.cu): append with rotation, decode attention through a block
// table, and page selection.
//
// Pool layout of one layer: K and V [page][kv head][row in page][head_dim],
// so that one head's rows of a page are one contiguous run (2 KB for 16 bf16
// rows of 64); bounds [page][kv head][min, max][head_dim].  Page sizes are
// powers of two.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tg_shared.h"

namespace tg {

constexpr int kPagedMinPage = 8, kPagedMaxPage = 256;
// Positions of the rotation table: beyond them binary32 has no angle of its own
// for every position.
constexpr int kPagedMaxPos = 1 << 24;
// Queries per launch: the schedule of a launch lives in shared memory.
constexpr int kPagedMaxQueries = 1024;
constexpr int kPagedHeads = 8;    // query heads of one stream (a KV head's group in blocks of 8)
constexpr int kPagedChunk = 32;   // cache rows per warp step of the CUDA-core kernel

struct PagedAppendParams {
  const float* k;        // [n_tokens][n_kv*hd] un-rotated
  const float* v;        // [n_tokens][n_kv*hd]
  const float* q;        // [n_tokens][n_head*hd] un-rotated, or null
  float* q_out;          // rotated q (may be q itself)
  const int* cu;         // [n_seqs+1] first token of each sequence, or null: token s is sequence s's
  const int* pos0;       // [n_seqs] position of each sequence's first new token
  const int* table;      // [n_seqs][max_blocks] pages
  const float* cs;       // RoPE table [table_len][hd/2][cos, sin]
  void* kp;              // layer base of the pools
  void* vp;
  void* bounds;          // or null
  int* err;
  int table_len, n_seqs, n_tokens, max_blocks, n_pages, log2p;
  int n_head, n_kv, hd, dtype;
  int vec4;              // rows and pointers are 16-byte aligned, hd a multiple of 4
};

// Decode attention.  A stream is one query's block of up to kPagedHeads query
// heads over one KV head; its rows are the rows of a list of pages: entries
// skip, skip + 1, ... of the query's table row (dense; skip 0 for a query that
// ends before entry skip), or the listed ones (sel).  The rows form chunks of 16 or 32; the chunks of all streams lie
// end to end and every CTA takes an equal contiguous range of them.
struct PagedAttnParams {
  const float* q;        // [n][n_head*hd], rotated
  float* out;            // [n][n_head*hd] (mode 0)
  float* records;        // [n][n_head][hd+2] o (un-normalised), m, l (mode 1); [n][n_kv][8] (2)
  const int* past;       // [n] last attended position, -1: none
  const int* table;      // [n][max_blocks]
  const int* sel;        // [n][n_kv][n_sel] listed table entries, or null: dense
  const void* kp;        // layer base of the pools
  const void* vp;
  float* part;           // [2*grid][kPagedHeads*(hd+2)] records of split streams
  unsigned* count;       // [n*n_kv*hblocks] arrivals at split streams, all 0 between launches
  int* err;
  long long page0;       // pages before this layer's (TMA rows)
  int n, n_head, n_kv, group, hblocks, hd;
  int max_blocks, n_pages, log2p, n_sel;
  int skip;              // leading entries left out for queries that attend all of them
  int lchunk;            // log2 of the rows of a chunk
  float scale_log2;      // log2(e) / sqrt(hd)
  int mode;              // 0 output, 1 records, 2 records of a packed prefix
  // Mode 2, a prefix that n_rows / group real queries share: "query" v is rows
  // 8 v .. 8 v + 7 of the n_rows rows query * group + head of a KV head, all
  // of them at positions 0..prefix_past of table row 0.  hblocks is 1.
  int n_rows, prefix_past;
};

// out = a batch's own records (mode 1) and those of its packed prefix, merged.
struct PagedPackedParams {
  const float* own;
  const float* packed;
  const int* past;
  float* out;
  int n, n_head, n_kv, group, hd;
  int shared;            // positions of the prefix: queries that end in it have it in `own`
  int limit;             // positions of the table: a query that ends behind them is empty
};

struct PagedSelectParams {
  const float* q;                // [n][n_head*hd], rotated
  const int* past;               // [n]
  const int* table;              // [n][max_blocks]
  const void* bounds;            // layer base
  unsigned long long* keys;      // [n][n_kv][3][max_blocks] scratch
  unsigned* count;               // [n][n_kv] arrivals, all 0 between launches
  int* pages;                    // [n][n_kv][n_sel]
  int* err;
  int n, n_head, n_kv, group, hd, dtype;
  int max_blocks, n_pages, log2p, n_sel, keep_first, keep_last;
};

// The shared prefix of a batch on the tensor cores (tg_paged_prefix.cu): bf16
// pool, head_dim 64.  steps * kPrefixKeys positions, named by table row 0.
constexpr int kPrefixKeys = 64;
struct PagedPrefixParams {
  const float* q;        // [n][n_head*64], rotated
  const int* past;       // [n]
  const int* table;      // pages of the prefix
  float* records;        // [parts][n_kv][66][n*group] o (un-normalised), m, l
  const float* own;      // [n][n_head][66] records of the queries' own rows
  float* out;            // [n][n_head*64]
  int* err;
  long long page0;
  int n, n_head, n_kv, group, n_pages, log2p, steps;
  int single, pairs, splits, parts;   // plan_paged_prefix
  float scale_log2;
  int limit;             // positions of the table: a query that ends behind them is empty
};

// Chooses single / pairs / splits / parts from n, group, n_kv and steps.
void plan_paged_prefix(PagedPrefixParams* p, int num_sms);
cudaError_t launch_paged_prefix(const CUtensorMap& tk, const CUtensorMap& tv,
                                const PagedPrefixParams& p, cudaStream_t st);
cudaError_t launch_paged_prefix_merge(const PagedPrefixParams& p, cudaStream_t st);

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t st);
cudaError_t launch_paged_core(const PagedAttnParams& p, int dtype, int grid, cudaStream_t st);
size_t paged_core_smem(int n, int hd);
// head_dim 32, 64 or 128; tk / tv are 2-D maps of the pools ({head_dim, rows},
// box {min(row, 128 bytes), min(page, 1 << paged_mma_lchunk) rows}, swizzled
// over the box's width).
int paged_mma_lchunk(int dtype, int hd);
cudaError_t launch_paged_packed_merge(const PagedPackedParams& p, cudaStream_t st);
cudaError_t launch_paged_mma(const CUtensorMap& tk, const CUtensorMap& tv, const PagedAttnParams& p,
                             int dtype, int grid, cudaStream_t st);
cudaError_t launch_paged_select(const PagedSelectParams& p, int num_sms, cudaStream_t st);

}  // namespace tg
