// The plan of a ragged serving batch, built on the GPU from request lengths: block-table entries of the
// pages that new tokens open, and for every packed new token its cache slot, position and request.
//
// Request b has old_b tokens in the cache and brings new_b.  With have_b = ceil(old_b / 16) and
// need_b = ceil((old_b + new_b) / 16), it takes the free pages base_b .. base_b + need_b - have_b, where
// base is the exclusive sum of the counts over requests from *head on; q_off is the exclusive sum of new.
// Every CTA scans the lengths of all requests itself (a few KB out of L2) and then fills its own range of
// tokens, so one launch does it all and no CTA waits for another.  Latency-bound: two dependent reads
// (lengths, then the page) and the scan.  Measured: 48 requests with one token each 2.8 us, 333 requests with
// 42 thousand new tokens 6.0 us.
#include "common.cuh"

#include <climits>
#include <stdexcept>
#include <string>

#include "../serve_ops.h"

namespace fak {
namespace {

constexpr int PAGE = 16;
constexpr int THREADS = 512;
constexpr int PER_CTA = 2048;   // tokens filled by one CTA

// Sums of tokens stay at MANY once they reach it: more than any capacity (checked below 2^30), and reported.
constexpr int MANY = 1 << 30;
FAK_DEV int add_tokens(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)MANY); }   // a <= MANY

__global__ void __launch_bounds__(THREADS) k_batch_plan(BatchPlanArgs a) {
  extern __shared__ int sm[];
  int* q_off = sm;               // [B + 1]
  int* base = sm + a.B + 1;      // [B]
  __shared__ int2 sums[THREADS / 32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.B, per = (B + THREADS - 1) / THREADS, b0 = min(B, tid * per), b1 = min(B, b0 + per);
  const int head = *a.head;
  auto lens = [&](int b, int& o, int& n) {
    o = a.old_len[b];
    n = a.new_len[b];
    if ((o < 0 || n < 0) && blockIdx.x == 0) report_error(a.err, 2);
    o = max(o, 0);
    n = max(n, 0);
  };
  auto opened = [](int o, int n) { return (int)(((int64_t)o + n + PAGE - 1) / PAGE - ((int64_t)o + PAGE - 1) / PAGE); };
  int2 mine = make_int2(0, 0);   // (new tokens, pages opened) of this thread's requests
  for (int b = b0; b < b1; b++) {
    int o, n;
    lens(b, o, n);
    mine.x = add_tokens(mine.x, n);
    mine.y += opened(o, n);
  }
  int2 inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc.x, d), y = __shfl_up_sync(0xffffffffu, inc.y, d);
    if (lane >= d) { inc.x = add_tokens(inc.x, x); inc.y += y; }
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  int2 off = make_int2(__shfl_up_sync(0xffffffffu, inc.x, 1), __shfl_up_sync(0xffffffffu, inc.y, 1));
  if (lane == 0) off = make_int2(0, 0);
  for (int w = 0; w < warp; w++) { off.x = add_tokens(off.x, sums[w].x); off.y += sums[w].y; }
  for (int b = b0; b < b1; b++) {
    int o, n;
    lens(b, o, n);
    q_off[b] = off.x;
    base[b] = head + off.y;
    off.x = add_tokens(off.x, n);
    off.y += opened(o, n);
    if (b == B - 1) {
      q_off[B] = off.x;
      if (blockIdx.x == 0) {
        a.head_out[0] = head + off.y;
        if (off.x > a.max_tokens) report_error(a.err, 2);
      }
    }
    if (blockIdx.x == 0) {
      // offsets never pass the capacity, so that what reads them stays inside the packed rows
      a.q_off[b] = min(q_off[b], a.max_tokens);
      if (b == B - 1) a.q_off[B] = min(off.x, a.max_tokens);
      a.ctx[b] = o + n;
      a.last[b] = n > 0 && off.x <= a.max_tokens ? off.x - 1 : -1;
    }
  }
  if (B == 0 && tid == 0 && blockIdx.x == 0) {
    q_off[0] = 0;
    a.q_off[0] = 0;
    a.head_out[0] = head;
  }
  if (B == 0 && tid == 0) q_off[0] = 0;
  __syncthreads();
  const int total = q_off[B];
  const int i1 = min(a.max_tokens, (int)(blockIdx.x + 1) * PER_CTA);
  for (int i = blockIdx.x * PER_CTA + tid; i < i1; i += THREADS) {
    int seq = -1, pos = 0, slot = -1;
    if (i < total) {
      int lo = 0, hi = B;   // the last request with q_off <= i (it has tokens: q_off[seq + 1] > i)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (q_off[mid] <= i) lo = mid;
        else hi = mid;
      }
      seq = lo;
      const int o = max(a.old_len[seq], 0);
      pos = o + (i - q_off[seq]);
      const int pg = pos / PAGE, have = (o + PAGE - 1) / PAGE;
      int page = -1;
      if (pos >= 0 && pg < a.width) {   // (a position that passed 32 bits is negative)
        if (pg < have) {
          page = a.table[(int64_t)seq * a.table_stride + pg];
        } else {
          const int f = base[seq] + pg - have;
          if (f >= 0 && f < a.n_free) {
            page = a.free_pages[f];
            if (pos % PAGE == 0) a.table[(int64_t)seq * a.table_stride + pg] = page;
          }
        }
      }
      if (page >= 0 && page <= INT_MAX / PAGE) slot = page * PAGE + pos % PAGE;
      else report_error(a.err, 2);   // the table is too narrow, the free pages ran out or hold no page: no slot
    }
    a.slot[i] = slot;
    a.pos[i] = pos;
    a.seq[i] = seq;
  }
  pdl_launch_dependents();
}

}  // namespace

void batch_plan_launch(const BatchPlanArgs& a, cudaStream_t stream) {
  const size_t smem = (size_t)(2 * a.B + 1) * sizeof(int);
  if (smem > 48 * 1024)
    FAK_CUDA_CHECK(cudaFuncSetAttribute(k_batch_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  const int n = a.max_tokens > 0 ? (a.max_tokens + PER_CTA - 1) / PER_CTA : 1;
  cfg.gridDim = dim3((unsigned)n);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FAK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k_batch_plan, a));
}

}  // namespace fak
