// Log probability, rank, entropy and top alternatives of given tokens, in one pass over the logit rows.
//
// Per row x[V], target t, with M = max x and S = sum e^(x - M):
//   logprob = (x_t - M) - ln S            rank = 1 + #{x_i > x_t} + #{x_i = x_t, i < t}
//   entropy = ln S - sum e^(x - M) (x - M) / S
//   the k largest x with their indices, ties to the lowest index.
// A target outside [0, V) has logprob 0 and rank 0.  A row with only -inf has entropy 0, logprobs -inf.
//
// A row is cut into n_seg segments (1 when there are enough rows to fill the machine), one CTA of 8
// warps each; the warps walk the segment in tiles of 32 lanes x 16 logits.  Each lane keeps its own
// (M, S, sum) and moves M at most once a tile.  For the top list the walk only stores the maximum of every
// lane's 32 logits of two tiles in shared memory.  Afterwards the k-th largest of the 256 lanes' maxima M
// bounds the k-th logit from below, the few groups that reach it are read again (about k of V / 32), and
// their logits that reach it are merged as 64-bit keys (ordered value, complemented index), 32 sorted ones at
// a time.  So selecting costs one store for two tiles and a few microseconds at the end of a row.
// Measured at 5 x 152064 with 5 alternatives: 11.4 us, bound by latency (some ten dependent steps).
// Measured at 2048 x 152064: f32 without alternatives 183 us (6.8 TB/s, above the copy rate it is compared
// with), with 20 226 us (5.5 TB/s); bf16 139 and 176 us, bound by instructions.  Candidates sorted out during
// the walk instead cost 293 us, groups read again one after another 256 us.
// Where the bound is -inf (a mask left fewer than k lanes a token) only larger logits and the first k indices
// can be in the list.  More candidates than the pool holds (equal logits) go to a list of each warp's own.
// Segments meet in a scratch record per segment; the CTA that takes the row's last ticket merges them in
// segment order, so results do not depend on the order of arrival.
#include "common.cuh"

#include <algorithm>
#include <climits>
#include <stdexcept>
#include <string>

#include "../serve_ops.h"

namespace fak {
namespace {

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int PER = 16;                // logits per lane and tile
constexpr int TILE = 32 * PER;         // per warp
constexpr int POOL = 512;              // candidate keys of the CTA
constexpr int MOST_TILES = 128;        // per warp and segment (their maxima take 0.5 KB of shared memory each)
constexpr int CAND = 64;               // a warp's own, when the pool is full: < 32 waiting + one per lane
constexpr int MAXK = 32;
constexpr int REC = 4 + 2 * MAXK;      // words of a segment's record: M, S, T, count, keys

typedef unsigned long long u64;

FAK_DEV u64 key_of(float v, uint32_t i) { return argmax_key(v + 0.f, i); }   // -0 counts as 0
FAK_DEV float key_value(u64 k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// Keys of a warp, one a lane: exchange towards descending order.
FAK_DEV void cx(u64& a, int lane, int d, bool down) {
  const u64 b = __shfl_xor_sync(0xffffffffu, a, d);
  const bool low = (lane & d) == 0;
  a = ((a > b) == (low == down)) ? a : b;
}
FAK_DEV u64 sort32(u64 a, int lane) {   // descending over lanes (bitonic)
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int d = n >> 1; d > 0; d >>= 1) cx(a, lane, d, n == 32 || (lane & n) == 0);
  return a;
}
FAK_DEV u64 merge32(u64 a, u64 b, int lane) {   // the 32 largest of two descending lists, descending
  b = __shfl_xor_sync(0xffffffffu, b, 31);
  a = a > b ? a : b;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) cx(a, lane, d, true);
  return a;
}

struct Stat {
  float m, s, t;   // max, sum e^(x - m), sum e^(x - m) (x - m)
};
FAK_DEV float finite_max(float m) { return m == -INFINITY ? 0.f : m; }
// Sums against a maximum m that is at least their own (the clamp keeps 0 * infinity out of t when the maxima
// are the type's extremes; empty sums stay 0).
FAK_DEV Stat against(const Stat& a, float m) {
  const float d = a.s == 0.f ? 0.f : fmaxf(a.m - finite_max(m), -1e30f), f = exp2f(d * 1.4426950408889634f);
  return {m, a.s * f, f * (a.t + a.s * d)};
}

// 16 logits a lane: 16-byte loads, neighbouring lanes side by side.
template <typename T>
constexpr int VEC = 16 / sizeof(T);
template <typename T>
struct Tile16 {
  static constexpr int E = VEC<T>;
  uint4 u[PER / E];
  // the lane's logits from i0 on; those past `end` read as -inf.  fast: the warp's tile is whole and aligned.
  FAK_DEV void load(const T* __restrict__ p, int i0, int end, bool fast) {
    if (fast) {
      const uint4* q = reinterpret_cast<const uint4*>(p + i0);
#pragma unroll
      for (int j = 0; j < PER / E; j++) u[j] = __ldcs(q + j * 32);
    } else {
      asm volatile("");   // a branch
#pragma unroll
      for (int j = 0; j < PER / E; j++) {
        const int i = i0 + j * 32 * E;
        T h[E];
#pragma unroll
        for (int e = 0; e < E; e++) h[e] = i + e < end ? p[i + e] : (T)-INFINITY;
        memcpy(&u[j], h, 16);
      }
    }
  }
  FAK_DEV void values(float (&x)[PER]) const {
#pragma unroll
    for (int j = 0; j < PER / E; j++) {
      T h[E];
      memcpy(h, &u[j], 16);
#pragma unroll
      for (int e = 0; e < E; e++) x[j * E + e] = (float)h[e];
    }
  }
};
template <typename T>
FAK_DEV int elt_at(int e) { return e % VEC<T> + e / VEC<T> * 32 * VEC<T>; }
FAK_DEV float ex2(float x) {   // 2^x, results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (out of line: the main loop shares the instruction caches with nothing larger than itself)
__device__ __noinline__ u64 merge_batch(u64 top, u64 cand, int lane) { return merge32(top, sort32(cand, lane), lane); }
FAK_DEV float ge_one(float a, float b) {   // a >= b ? 1 : 0
  float r;
  asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

FAK_DEV float gt_one(float a, float b) {   // a > b ? 1 : 0
  float r;
  asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// order-preserving integer form of a float (its own inverse on the bits)
FAK_DEV int ordered(float v) {
  const int b = __float_as_int(v);
  return b >= 0 ? b : b ^ 0x7fffffff;
}

template <typename T, bool TOP, bool CAP>
__global__ void __launch_bounds__(THREADS, 4) k_logprobs(LogprobArgs a, int seg_len) {
  __shared__ u64 s_cand[TOP ? WARPS : 1][TOP ? CAND : 1];
  __shared__ u64 s_list[WARPS][32];
  __shared__ Stat s_stat[WARPS];
  __shared__ int s_cnt[WARPS];
  __shared__ u64 s_pool[TOP ? POOL : 1];
  __shared__ int s_last, s_n, s_own;   // s_own: some warp has a list of its own
  __shared__ int s_bound;                            // (an ordered float)
  __shared__ float s_wmax[WARPS];
  __shared__ __align__(16) float s_max[TOP ? THREADS : 4];
  extern __shared__ float s_mx[];   // TOP: [two tiles of the warp][thread] maxima of 32 logits
  constexpr float LOG2E = 1.4426950408889634f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = blockIdx.x;
  const int64_t r = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (r >= a.T) return;
  if (TOP && tid == 0) {   // (a barrier comes before their use)
    s_n = s_own = 0;
    s_bound = INT_MAX;
  }
  pdl_wait();
  const T* __restrict__ x = (const T*)a.x + r * a.stride;
  auto cap = [&](float v) { return CAP ? a.softcap * tanhf(v / a.softcap) : v; };
  const int tgt = a.target[r];
  const bool given = tgt >= 0 && tgt < a.V;
  const int i_begin = seg * seg_len, i_end = min(a.V, i_begin + seg_len);

  Stat st = {-INFINITY, 0.f, 0.f};
  float above_f = 0.f;           // (a lane's count stays far below 2^24)
  const int k = a.k;

  float xt = INFINITY, xt_above = INFINITY;   // (loaded behind the first tile)
  auto whole = [&](int base) { return a.vec && base + TILE <= i_end; };
  float pair = -INFINITY;
  // one tile of the warp from logit `base` on, the round-th; i0: the lane's first logit
  auto walk = [&](const Tile16<T>& tile, int base, int round) {
    float v[PER];
    const int i0 = base + VEC<T> * lane;
    tile.values(v);
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < PER; e++) {
      if constexpr (CAP) v[e] = cap(v[e]);
      mx = fmaxf(mx, v[e]);
    }
    if (mx > st.m) {   // move the base of this lane's sums
      asm volatile("");
      const float d = st.s == 0.f ? 0.f : fmaxf(st.m - mx, -1e30f), f = ex2(d * LOG2E);
      st.t = f * (st.t + st.s * d);
      st.s *= f;
      st.m = mx;
    }
    const float mb = finite_max(st.m);
#pragma unroll
    for (int e = 0; e < PER; e++) {
      const float d = v[e] - mb, p = ex2(d * LOG2E);
      st.s += p;
      st.t = fmaf(p, fmaxf(d, -1e30f), st.t);   // p is 0 where the clamp acts; a NaN stays in p
    }
    // #{x >= x_t} in tiles before the target, #{x > x_t} = #{x >= the float above x_t} in those after it
    if (base > tgt || base + TILE <= tgt) {
      const float bar = base > tgt ? xt_above : xt;
#pragma unroll
      for (int e = 0; e < PER; e++) above_f += ge_one(v[e], bar);
    } else {
      asm volatile("");   // a branch, not predicated work in every tile
#pragma unroll
      for (int e = 0; e < PER; e++) {
        const int i = i0 + elt_at<T>(e);
        above_f += i < tgt ? ge_one(v[e], xt) : i < i_end ? ge_one(v[e], xt_above) : 0.f;
      }
    }
    if constexpr (TOP) {   // one maximum for two tiles
      pair = (round & 1) ? fmaxf(pair, mx) : mx;
      s_mx[(round >> 1) * THREADS + tid] = pair;
    }
  };
  // two tiles in registers: the loads of one are in flight while the other is worked on
  constexpr int STEP = WARPS * TILE;
  Tile16<T> even, odd;
  const int rounds = (i_end - i_begin + STEP - 1) / STEP, first = i_begin + warp * TILE, lane0 = VEC<T> * lane;
  if (first < i_end) even.load(x, first + lane0, i_end, whole(first));
  if (given) xt = cap((float)x[tgt]);
  xt_above = xt == INFINITY ? __int_as_float(0x7fffffff) : nextafterf(xt, INFINITY);   // (a NaN: nothing reaches it)
#pragma unroll 1
  for (int r2 = 0, base = first; base < i_end; r2 += 2, base += 2 * STEP) {
    const bool more = base + STEP < i_end;
    if (more) odd.load(x, base + STEP + lane0, i_end, whole(base + STEP));
    walk(even, base, r2);
    if (base + 2 * STEP < i_end) even.load(x, base + 2 * STEP + lane0, i_end, whole(base + 2 * STEP));
    if (more) walk(odd, base + STEP, r2 + 1);
  }
  int above = (int)above_f;
  // the CTA's maximum; every lane's sums against it, added in a fixed order
  {
    const float wm = warp_max(st.m);
    if (lane == 0) s_wmax[warp] = wm;
    if (TOP) s_max[tid] = st.m;
  }
  __syncthreads();
  float m_cta = s_wmax[0];
#pragma unroll
  for (int w = 1; w < WARPS; w++) m_cta = fmaxf(m_cta, s_wmax[w]);
  {
    const Stat y = against(st, m_cta);
    const float ws = warp_sum(y.s), wt = warp_sum(y.t);
    const int wc = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) {
      s_stat[warp] = {m_cta, ws, wt};
      s_cnt[warp] = wc;
    }
  }
  u64 top = 0;   // the warp's list: lane i holds the i-th largest key
  if constexpr (TOP) {
    // the k-th largest of the 256 lanes' maxima: the smallest that fewer than k others exceed
    float larger = 0.f;
#pragma unroll 8
    for (int e = 0; e < THREADS / 4; e++) {
      const float4 y = reinterpret_cast<const float4*>(s_max)[e];
      larger += (gt_one(y.x, st.m) + gt_one(y.y, st.m)) + (gt_one(y.z, st.m) + gt_one(y.w, st.m));
    }
    const int cut = __reduce_min_sync(0xffffffffu, larger < (float)k ? ordered(st.m) : INT_MAX);
    if (lane == 0) atomicMin(&s_bound, cut);
    __syncthreads();
    const int sb = s_bound;
    const float bound = __int_as_float(sb >= 0 ? sb : sb ^ 0x7fffffff);
    u64 kth = 0;
    int waiting = 0;
    // pairs of tiles whose maximum reaches the bound, a bit each; then every lane takes its next one
    u64 pairs = 0;
    for (int p = 0; p < (rounds + 1) / 2; p++) {
      const int i0 = first + 2 * p * STEP + lane0;
      const float mx = i0 < i_end ? s_mx[p * THREADS + tid] : -INFINITY;
      if (i0 < i_end && (mx > -INFINITY ? mx >= bound : bound == -INFINITY && i0 < k)) pairs |= 1ull << p;
    }
    while (__any_sync(0xffffffffu, pairs != 0)) {
      uint32_t cand = 0;   // the lane's logits that may be in the list
      int i0 = 0;
      if (pairs) {
        i0 = first + 2 * (__ffsll(pairs) - 1) * STEP + lane0;
        pairs &= pairs - 1;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          Tile16<T> g;
          const int b = i0 + h * STEP;
          g.load(x, b, i_end, a.vec && b - lane0 + TILE <= i_end);
          float v[PER];
          g.values(v);
#pragma unroll
          for (int e = 0; e < PER; e++) {
            const int i = b + elt_at<T>(e);
            const float y = cap(v[e]);
            if (i < i_end && (y > -INFINITY ? y >= bound : y == -INFINITY && bound == -INFINITY && i < k)) cand |= 1u << (16 * h + e);
          }
        }
      }
      while (__any_sync(0xffffffffu, cand != 0)) {   // one a lane at a time, read again (they are few)
        u64 key = 0;
        if (cand) {
          const int e = __ffs(cand) - 1, i = i0 + (e >> 4) * STEP + elt_at<T>(e & 15);
          cand &= cand - 1;
          key = key_of(cap((float)x[i]), (uint32_t)i);
        }
        const bool take = key > kth;
        const uint32_t votes = __ballot_sync(0xffffffffu, take);
        if (votes == 0) continue;
        const int n = __popc(votes), my = __popc(votes & ((1u << lane) - 1));
        int at = 0;
        if (lane == 0) at = atomicAdd(&s_n, n);
        at = __shfl_sync(0xffffffffu, at, 0);
        if (at + n <= POOL) {
          if (take) s_pool[at + my] = key;
        } else {   // no room: this warp's own list
          if (take && at + my < POOL) s_pool[at + my] = 0;
          if (take) s_cand[warp][waiting + my] = key;
          waiting += n;
          s_own = 1;
          __syncwarp();
          if (waiting >= 32) {
            waiting -= 32;
            top = merge_batch(top, s_cand[warp][waiting + lane], lane);
            kth = __shfl_sync(0xffffffffu, top, k - 1);
            __syncwarp();
          }
        }
      }
    }
    __syncthreads();
    const int n = min(s_n, POOL);
    if (!s_own && n <= THREADS) {   // few candidates: each finds its rank
      if (tid < n) {
        const u64 key = s_pool[tid];
        int rank = 0;
        for (int e = 0; e < n; e++) rank += s_pool[e] > key;
        if (rank < 32) s_list[0][rank] = key;
      } else if (tid < 32) {
        s_list[0][tid] = 0;
      }
    } else {
      if (warp == 0)
        for (int b = 0; b < n; b += 32) top = merge_batch(top, b + lane < n ? s_pool[b + lane] : 0ull, lane);
      if (waiting > 0) top = merge_batch(top, lane < waiting ? s_cand[warp][lane] : 0ull, lane);
      s_list[warp][lane] = top;
    }
  }
  __syncthreads();
  if (warp != 0 && a.n_seg == 1) return;
  if (warp == 0) {
    st = s_stat[0];
    above = s_cnt[0];
    if (TOP) top = s_list[0][lane];
    for (int w = 1; w < WARPS; w++) {
      st.s += s_stat[w].s;
      st.t += s_stat[w].t;
      above += s_cnt[w];
      if (TOP && (s_own || s_n > THREADS)) top = merge32(top, s_list[w][lane], lane);
    }
  }
  if (a.n_seg > 1) {
    float* rec = a.part + ((int64_t)r * a.n_seg + seg) * REC;
    if (warp == 0) {
      if (lane == 0) {
        rec[0] = st.m; rec[1] = st.s; rec[2] = st.t;
        rec[3] = __int_as_float(above);
      }
      if constexpr (TOP) reinterpret_cast<u64*>(rec + 4)[lane] = top;
      __threadfence();
      __syncwarp();
      if (lane == 0) s_last = atomicAdd(a.tickets + r, 1) == a.n_seg - 1;
    }
    __syncthreads();
    if (!s_last) {
      pdl_launch_dependents();
      return;
    }
    __threadfence();
    // lists: every warp takes the segments w, w + 8, .. (eight loads in flight), then warp 0 the warps
    const float* recs = a.part + (int64_t)r * a.n_seg * REC;
    if constexpr (TOP) {
      top = 0;
      for (int s0 = warp; s0 < a.n_seg; s0 += 8 * WARPS) {
        u64 y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int s = s0 + e * WARPS;
          y[e] = s < a.n_seg ? __ldcg(reinterpret_cast<const u64*>(recs + (int64_t)s * REC + 4) + lane) : 0ull;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (s0 + e * WARPS < a.n_seg) top = merge32(top, y[e], lane);
      }
      s_list[warp][lane] = top;
      __syncthreads();
      if (warp < 4) s_list[warp][lane] = top = merge32(top, s_list[warp + 4][lane], lane);
      __syncthreads();
    }
    if (warp != 0) return;
    if constexpr (TOP) {
      for (int w = 1; w < 4; w++) top = merge32(top, s_list[w][lane], lane);
    }
    // sums: lane l the segments l, l + 32, .., against the largest maximum
    float m = -INFINITY;
    for (int s = lane; s < a.n_seg; s += 32) m = fmaxf(m, __ldcg(recs + (int64_t)s * REC));
    m = warp_max(m);
    st = {m, 0.f, 0.f};
    above = 0;
    for (int s = lane; s < a.n_seg; s += 32) {
      const float4 q = __ldcg(reinterpret_cast<const float4*>(recs + (int64_t)s * REC));
      const Stat y = against({q.x, q.y, q.z}, m);
      st.s += y.s;
      st.t += y.t;
      above += __float_as_int(q.w);
    }
    st.s = warp_sum(st.s);
    st.t = warp_sum(st.t);
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) a.tickets[r] = 0;
  }
  const float log_s = logf(st.s);   // S >= 1 unless the row is empty
  if (lane == 0) {
    const bool none = st.m == -INFINITY && st.s == 0.f;
    a.logprob[r] = !given ? 0.f : none ? -INFINITY : (xt - st.m) - log_s;
    a.entropy[r] = none ? 0.f : log_s - st.t / st.s;
    a.rank[r] = given ? above + 1 : 0;
  }
  if constexpr (TOP) {
    if (lane < k) {
      const bool has = top != 0;
      const float tv = key_value(top);
      a.top_ids[r * k + lane] = has ? argmax_key_index(top) : -1;
      a.top_logprobs[r * k + lane] = !has || tv == -INFINITY ? (st.s != st.s ? st.s : -INFINITY) : (tv - st.m) - log_s;
    }
  }
}

}  // namespace

// Segments per row: 2 1/4 CTAs a SM where the rows are fewer, a segment at least a tile of every warp and at
// most 128.  (A CTA costs about as much as four tiles beside its tiles: 40 rows of 152064 in 8 segments took
// 20.7 us, in 16 26.5; 148 rows in 1 / 2 / 4 52.4 / 42.2 / 38.8; 300 rows in 1 58.5, in 2 73.8.)
int logprob_segments(int T, int V, int n_sm) {
  const int tiles = (V + WARPS * TILE - 1) / (WARPS * TILE);
  const int want = std::max(1, (int)std::min<int64_t>(9 * n_sm / ((int64_t)4 * T), std::min(tiles, 64)));
  return std::max(want, (tiles + MOST_TILES - 1) / MOST_TILES);
}
int64_t logprob_part_words(int T, int n_seg) { return n_seg > 1 ? (int64_t)T * n_seg * REC : 0; }

void logprob_launch(const LogprobArgs& a, cudaStream_t stream) {
  if (a.T == 0) return;
  int seg = (a.V + a.n_seg - 1) / a.n_seg;
  seg = (seg + TILE - 1) / TILE * TILE;
  const int tiles = (seg + WARPS * TILE - 1) / (WARPS * TILE);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_seg, (unsigned)(a.T < 32768 ? a.T : 32768), (unsigned)(((int64_t)a.T + 32767) / 32768));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto go = [&](auto tag) {
    using E = decltype(tag);
    const bool top = a.k > 0, cap = a.softcap > 0.f;
    auto launch = [&](auto kern, size_t smem) {
      cfg.dynamicSmemBytes = smem;
      FAK_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      FAK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, seg));
    };
    const size_t maxima = (size_t)((tiles + 1) / 2) * THREADS * sizeof(float);
    if (top && cap) launch(k_logprobs<E, true, true>, maxima);
    else if (top) launch(k_logprobs<E, true, false>, maxima);
    else if (cap) launch(k_logprobs<E, false, true>, 0);
    else launch(k_logprobs<E, false, false>, 0);
  };
  if (a.type == Elt::F32) go(float());
  else if (a.type == Elt::F16) go(__half());
  else go(__nv_bfloat16());
}

}  // namespace fak
