// Attention over the 4-bit paged KV cache (layout in kv4.cuh): single tokens, verification blocks and chunks.
//
// Sequence b has ctx_b keys, the last n_b of them its new tokens; query i of them sees the keys up to its
// own position ctx_b - n_b + i (with a window, only the last `window` of those).  The n_b * G query rows
// of a KV head (G query heads share it) are the columns of the matrix products, 8 NT of them a CTA:
//
//   S^T [16 tokens x 8 rows] = K Q^T    m16n8k16, K codes as the A operand, straight from the page words
//   O^T [D x 8 rows]        += V^T P^T  m16n8k16, V codes as the A operand, P^T from S^T by movmatrix
//
// Codes enter the tensor cores as f16 denormals: a nibble in the low bits of a half is code * 2^-24
// exactly, one in bits 4-7 is 16 times that, so one AND makes two operands and no conversion is needed
// (products with f16 and their f32 sums are exact for denormals too).  Scales and minima stay outside:
//   q.k = sum_g s_g (q_g . c_g) + sum_g m_g sum(q_g)      the group's product is scaled in f32; the second
//                                                         sum is one m16n8k8 with sum(q_g) in two f16 parts
//   o_d = sum_j (p_j s_jg) c_jd + sum_j p_j m_jg          the scale multiplies P (f16) per group; the second
//                                                         sum is one m16n8k16 whose fifth row, all ones,
//                                                         gives the softmax denominator
// Queries are rounded to f16 after a power-of-two scaling of their row (exact for f16 inputs up to 23 binades below
// the row's largest, for bf16 up to 26: every other dim is scaled down by 16 more); P is f16, raised by a power of
// two that the warp's largest scale so far allows, so that P s is neither above 65504 nor subnormal where a key of
// little weight meets a small scale (values around 1e-4, 8000 keys 7 below the largest logit, one split: error
// 5e-2 -> 7e-4 of the largest output).  Rounding P alone moves numerator and denominator alike; what P s loses
// meets codes around 8, and for outputs finer than bf16 the loss times 8 is added back over up to 1024 keys (f16,
// 3 to 12 keys: error 3.4e-4 -> 2.4e-4 of the output, 2.0e-4 being that of its rounding; over 8000 keys 2.04e-4 ->
// 2.02e-4, for 9 to 14% more time).
//
// A warp streams its own pages through a ring of shared memory filled by one bulk copy a page and walks
// them with an online softmax whose base moves only when a row outgrows it; the CTA's warps, then the
// splits of a sequence, are merged at the end: through distributed shared memory where the splits of a
// sequence form a cluster, by k_kv4_combine where there are more of them.
//
// Measured (graph of calls, us): single tokens, 32 lanes up to 32768 keys of 40 heads over 8 KV heads of 128
// 180 (834 MB, 4.6 TB/s; bound by the copies; f32 in and out in 16 splits 193), 28 heads over 4 KV heads of 128, 5 up
// to 9000 16.3 and 1 x 2048 5.9 (both bound by latency: the longest chain is lengths, table entry, page, softmax,
// merge); 16 x 5 tokens of 64 heads over 8 KV heads of 64 at 4097 keys, f16, 55 (bound by instructions: three
// column blocks unpack the same pages).  The vote on the scales of every page takes 3 to 6% of these.
#include "kv4_common.cuh"

#include <algorithm>
#include <stdexcept>
#include <string>
#include <type_traits>

namespace fak {
namespace {

using namespace kv4;

constexpr int W = kRowsGrain;   // warps per CTA
constexpr int STAGES = 4;     // pages in flight per warp
constexpr float HEADROOM = 0.875f;   // log2 growth of a row's max before its base moves
constexpr float LIFT = 2.f;          // P = 2^(z - base + LIFT + raise) <= 7.34 * 2^raise
// P s must fit f16 from its largest (P 7.34 * 2^raise, scales up to 8736 from the append) down to keys of little
// weight under small scales, whose products would be subnormal: a warp raises P by the most its scales allow,
// 2^raise with all of them below 2^(MOST_RAISE - raise).
constexpr int MOST_RAISE = 13;
template <int D, int NT>
constexpr int kResident = D == 64 && NT == 1 ? 5 : 4;   // CTAs a SM
constexpr int FEW = 1024;            // keys up to which f16 and f32 outputs take the finer sums
constexpr float LOG2E = 1.4426950408889634f;
// More query rows than this per (sequence, KV head) go to kv4_prefill.cu.  Measured over 4 KV heads (us, here /
// there): head dim 128, 48 rows 8 x 8000 50.8 / 49.6, 16 x 1000 18.3 / 25.6, 64 rows 73.8 / 49.9, 21.9 / 25.6;
// head dim 64, 64 rows 39.4 / 38.0, 18.7 / 19.5, 80 rows 51.3 / 38.5, 19.2 / 19.8.
constexpr int prefill_rows(int D) { return D == 128 ? 48 : 64; }
constexpr float kPrefillLift = 4.f;   // LIFT of that kernel

FAK_DEV void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a zero accumulator
FAK_DEV void mma_f16_16816_z(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
FAK_DEV void mma_f16_1688_z(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
FAK_DEV void mma_f16_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(b0));
}
// a b - c, exact for c = a b rounded
FAK_DEV uint32_t left_h2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), __hneg2(*reinterpret_cast<__half2*>(&c)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
FAK_DEV uint32_t add_h2(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
FAK_DEV uint32_t max_h2(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
FAK_DEV uint32_t pow2_h2(int n) { return (uint32_t)(n + 15) * 0x04000400u; }   // 2^n, -14 <= n <= 15
FAK_DEV bool reaches(uint32_t a, uint32_t b) {   // either half of a is at least b's
  return __hge2_mask(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b)) != 0;
}
FAK_DEV uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <int D, int NT>
struct Smem {
  static constexpr int COLS = 8 * NT;
  static constexpr int OSTRIDE = D + 4;   // floats per column of the merge area (keeps its stores on distinct banks)
  union {
    uint8_t ring[W][STAGES][Lay<D>::BYTES];
    float o[W][COLS][OSTRIDE];
  };
  uint64_t full[W][STAGES];
  float base[W][COLS], sum[W][COLS];
  alignas(16) float ml[COLS][2];   // (base, sum) of the CTA, for its cluster
  float qmax[COLS][Lay<D>::NG];
  alignas(16) float qsum[COLS][Lay<D>::NG];
  uint4 qf[NT][Lay<D>::NG][32];
  int fail;   // a wait gave up
  uint32_t lost[COLS];   // groups with a value that the column sees and that is no number (taken out of V)
};

// Weight of a part (base, sum) against a base m: 0 for one without keys; one whose logits were all NaN (its base
// never moved) passes its NaN on.
FAK_DEV float part_weight(float base, float sum, float m) {
  return base == -INFINITY ? (sum != sum ? 1.f : 0.f) : ex2(base - m);
}
// One split's (weight f, sum ls, N outputs z) into the running sums.
template <int N>
FAK_DEV void merge_split(float f, float ls, const float* z, float& l, float (&acc)[N]) {
  if (f == 0.f) return;   // (a split without keys: nothing of it is defined)
  l = fmaf(f, ls, l);
#pragma unroll
  for (int i = 0; i < N; i++) acc[i] = fmaf(f, z[i], acc[i]);
}

FAK_DEV float2 remote_f2(const float* p, int rank) {   // *p of the cluster's CTA `rank`
  uint32_t at;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
FAK_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CLUSTER: the splits of a block are one thread-block cluster and merge through shared memory; else they
// leave partial results for k_kv4_combine.  The sums are the same, in the same order.
// MULTI: sequences may bring several tokens, so that rows differ in the keys they see (without what that asks for
// single tokens take 3% less, 32 lanes up to 32768 187 us instead of 194).
template <int D, int NT, bool CAP, bool CLUSTER, bool FINE, bool MULTI>
__global__ void __launch_bounds__(W * 32, kResident<D, NT>)
k_kv4_attn(const __grid_constant__ Kv4Attn a, int n_split) {
  using L = Lay<D>;
  constexpr int NG = L::NG;
  constexpr int COLS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D, NT>& sm = *reinterpret_cast<Smem<D, NT>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, b = blockIdx.z, G = a.G;
  int split = blockIdx.x, rc = 0;
  if (gridDim.x > n_split) {
    rc = blockIdx.x / n_split;
    split = blockIdx.x - rc * n_split;
  }
  if (lane < STAGES) tc::mbar_init(&sm.full[warp][lane], 1);
  if (tid == 0) sm.fail = 0;
  if (MULTI && tid < COLS) sm.lost[tid] = 0;
  tc::fence_mbar_init();
  __syncthreads();
  pdl_wait();

  const int* row = a.table + (int64_t)b * a.table_stride;
  // table entries travel with ctx: those of a sequence that fills its table (others are fetched again)
  const int pps_full = a.window <= 0 ? spread(a.width, n_split, W) : -1, ahead = split * pps_full + warp + W * lane;
  const int early = lane * W < pps_full && ahead < a.width ? row[ahead] : -1;
  const int ctx = min(a.ctx[b], a.width * PAGE);
  if (tid == 0 && a.ctx[b] > ctx) report_error(a.err, 2);   // more keys than the table has pages for
  const bool few = ctx <= FEW;
  int tok0 = b, n = 1;
  if (a.q_off) {
    tok0 = max(a.q_off[b], 0);
    n = min(a.q_off[b + 1], a.n_tokens) - tok0;
    if (n > a.max_new) {
      report_error(a.err, 3);
      n = a.max_new;
    }
  }
  const int R = n * G, r0 = rc * COLS;
  if (R <= r0) return;
  const Span sp = span_of(ctx, n, a.query_of(r0), a.query_of(min(R - 1, r0 + COLS - 1)), a.window, n_split, W, a.width);
  const int p_begin = sp.p0 + split * sp.pps, p_end = min(sp.p1, p_begin + sp.pps);
  if (!CLUSTER && p_begin >= p_end && !(split == 0 && sp.live == 0)) return;

  // pages of this warp: p_begin + warp, + W, ..; 32 table entries at a time, one a lane
  const int np = max(0, (p_end - p_begin - warp + W - 1) / W);
  const int* table = row + p_begin + warp;
  const uint8_t* page = nullptr;   // lane l: address of page 32 j + l, refreshed every 32 pages
  auto issue = [&](int i) {
    if ((i & 31) == 0 && i + lane < np) {
      int pid = i == 0 && sp.pps == pps_full ? early : table[(int64_t)W * (i + lane)];
      if ((unsigned)pid >= (uint64_t)a.n_pages) {
        report_error(a.err, 2);
        pid = 0;
      }
      page = a.pages + ((int64_t)pid * a.Hkv + kvh) * L::BYTES;
    }
    if (lane == (i & 31)) {
      uint64_t* bar = &sm.full[warp][i % STAGES];
      tc::mbar_arrive_expect_tx(bar, L::BYTES);
      bulk_load(sm.ring[warp][i % STAGES], page, L::BYTES, bar);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++)
    if (i < np) issue(i);

  // Queries.  Lane (g, t) of the fragments holds column nt * 8 + g, dims group * 32 + 8 t .. + 7; the CTA's
  // warps share the (n-tile, group) pairs out, and every warp then reads all of them.
  constexpr int PAIRS = NT * NG, MINE = (PAIRS + W - 1) / W;
  float x[MINE][8];
#pragma unroll
  for (int m = 0; m < MINE; m++) {
    const int pr = warp + m * W, nt = pr / NG, gr = pr % NG;
    const int r = r0 + nt * 8 + g;
#pragma unroll
    for (int e = 0; e < 8; e++) x[m][e] = 0.f;
    if (pr < PAIRS && r < R) {
      const int qi = a.query_of(r);
      const int64_t at = (int64_t)(tok0 + qi) * a.q_tok + (int64_t)(kvh * G + r - qi * G) * a.q_head + gr * 32 + 8 * t;
      if (a.q_vec && a.q_type != Elt::F32) {
        const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 f = unpack_h2(w[e]);
          x[m][2 * e] = a.q_type == Elt::F16 ? f.x : bf16_bits_lo(w[e]);
          x[m][2 * e + 1] = a.q_type == Elt::F16 ? f.y : bf16_bits_hi(w[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[m][e] = load_elt(a.q, a.q_type, at + e);
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[m][e]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (pr < PAIRS && t == 0) sm.qmax[nt * 8 + g][gr] = amax;
  }
  __syncthreads();
  // a power of two brings the row's largest into [2^13, 2^14)
  auto factor = [&](int col) {
    float amax = 0.f;
#pragma unroll
    for (int gr = 0; gr < NG; gr++) amax = fmaxf(amax, sm.qmax[col][gr]);
    const int ex = (int)(__float_as_uint(amax) >> 23);           // biased exponent; 255: infinity
    return __uint_as_float((uint32_t)(ex == 255 ? 127 : min(127 + 126, 127 + 13 + 127 - ex)) << 23);
  };
#pragma unroll
  for (int m = 0; m < MINE; m++) {
    const int pr = warp + m * W, nt = pr / NG, gr = pr % NG;
    if (pr < PAIRS) {
      const float f = factor(nt * 8 + g);
      float y[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y[e] = __half2float(__float2half_rn(x[m][e] * f));
        sum += y[e];
      }
      // nibble pairs (e, e + 4); the odd pairs arrive 16 times too large
      sm.qf[nt][gr][lane] = make_uint4(pack_f16(y[0], y[4]), pack_f16(y[1] * 0.0625f, y[5] * 0.0625f), pack_f16(y[2], y[6]),
                                       pack_f16(y[3] * 0.0625f, y[7] * 0.0625f));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) sm.qsum[nt * 8 + g][gr] = sum * 0.015625f;   // |sum| <= 32 * 2^14: back into f16's range
    }
  }
  __syncthreads();
  uint32_t qf[NT][NG][4], qs[NT];
  float cf[NT][2];                 // logit factor (log2 units) of columns 2 t, 2 t + 1
  int lim[NT][2], low[NT][2];      // keys [low, lim) are seen by the column
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
#pragma unroll
    for (int gr = 0; gr < NG; gr++) {
      const uint4 u = sm.qf[nt][gr][lane];
      qf[nt][gr][0] = u.x; qf[nt][gr][1] = u.y; qf[nt][gr][2] = u.z; qf[nt][gr][3] = u.w;
    }
    // B of the m16n8k8: rows 2 t, 2 t + 1 = the groups' sums, their high parts then the remainders
    const float2 s = *reinterpret_cast<const float2*>(&sm.qsum[nt * 8 + g][NG == 4 ? 2 * (t & 1) : 0]);
    const float h0 = __half2float(__float2half_rn(s.x)), h1 = __half2float(__float2half_rn(s.y));
    qs[nt] = (NG == 4 ? t >= 2 : t == 1) ? pack_f16(s.x - h0, s.y - h1) : pack_f16(h0, h1);
    if (NG == 2 && t >= 2) qs[nt] = 0;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = r0 + nt * 8 + 2 * t + e;
      cf[nt][e] = 64.f / factor(nt * 8 + 2 * t + e) * a.scale * (CAP ? 1.f : LOG2E);
      lim[nt][e] = r < R ? min(ctx - n + a.query_of(r) + 1, ctx) : 0;
      low[nt][e] = a.window > 0 ? max(0, lim[nt][e] - a.window) : 0;
    }
  }
  // Keys every live row sees, [low_max, lim_min): pages inside need no mask (dead columns are dropped at
  // the end).  Keys outside [low_any, lim_any) are seen by no row: their V is not touched.
  const int i_first = a.query_of(r0), i_last = a.query_of(min(R - 1, r0 + COLS - 1));
  const int lim_any = ctx - n + i_last + 1, lim_min = ctx - n + i_first + 1;
  const int low_any = a.window > 0 ? max(0, lim_min - a.window) : 0;
  const int low_max = a.window > 0 ? max(0, lim_any - a.window) : 0;

  float o[NT][NG][2][4], mt[NT][4], base[NT][2];
  float lift[NT][2];   // LIFT + raise - base (0 while the base is -inf: then every z is -inf too)
  int raise = MOST_RAISE;
  uint32_t s_most = pow2_h2(0);   // 2^(MOST_RAISE - raise), twice; infinity once raise is 0
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    base[nt][0] = base[nt][1] = -INFINITY;
    lift[nt][0] = lift[nt][1] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      mt[nt][e] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; gr++) o[nt][gr][0][e] = o[nt][gr][1][e] = 0.f;
    }
  }
  constexpr uint32_t M0 = 0x000f000fu, M4 = 0x00f000f0u;
  const float cap_in = CAP ? 1.f / a.softcap : 0.f, cap_out = CAP ? a.softcap * LOG2E : 0.f;
#pragma unroll 1
  for (int i = 0; i < np; i++) {
    if (i + STAGES - 1 < np) issue(i + STAGES - 1);
    // (a wait that gives up is reported at the end; the loop goes on, so that every copy is waited for)
    tc::mbar_wait(&sm.full[warp][i % STAGES], (uint32_t)((i / STAGES) & 1), &sm.fail);
    const uint8_t* pg = sm.ring[warp][i % STAGES];
    const int key0 = (p_begin + warp + W * i) * PAGE;
    const bool whole = key0 >= low_max && key0 + PAGE <= lim_min;   // warp-uniform

    // S^T: rows = tokens g and g + 8, columns = query rows 2 t, 2 t + 1 of each n-tile
    float z[NT][4];
    {
      uint32_t k0[NG], k1[NG], s0[NG / 2], s1[NG / 2], m0[1], m1[1];
      lds(pg + L::KC + g * (D / 2) + t * 4 * NG, k0);
      lds(pg + L::KC + (g + 8) * (D / 2) + t * 4 * NG, k1);
      lds(pg + L::KS + g * 2 * NG, s0);
      lds(pg + L::KS + (g + 8) * 2 * NG, s1);
      lds(pg + L::KM + g * 2 * NG + (NG == 4 ? (t & 1) * 4 : 0), m0);
      lds(pg + L::KM + (g + 8) * 2 * NG + (NG == 4 ? (t & 1) * 4 : 0), m1);
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        mma_f16_1688_z(z[nt], m0[0], m1[0], qs[nt]);
      }
#pragma unroll
      for (int gr = 0; gr < NG; gr++) {
        const uint32_t w0 = k0[gr], w1 = k1[gr], u0 = w0 >> 8, u1 = w1 >> 8;
        const float2 f0 = unpack_h2(s0[gr / 2]), f1 = unpack_h2(s1[gr / 2]);
        const float sa = gr & 1 ? f0.y : f0.x, sb = gr & 1 ? f1.y : f1.x;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float d[4];
          mma_f16_16816_z(d, w0 & M0, w1 & M0, w0 & M4, w1 & M4, qf[nt][gr][0], qf[nt][gr][1]);
          mma_f16_16816(d, u0 & M0, u1 & M0, u0 & M4, u1 & M4, qf[nt][gr][2], qf[nt][gr][3]);
#pragma unroll
          for (int e = 0; e < 4; e++) acc[nt][e] = gr == 0 ? (e < 2 ? sa : sb) * d[e] : fmaf(e < 2 ? sa : sb, d[e], acc[nt][e]);
        }
      }
      // codes carry 2^-24, the sums 2^-6
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          z[nt][e] = fmaf(acc[nt][e], 262144.f, z[nt][e]) * cf[nt][e & 1];
          if constexpr (CAP) z[nt][e] = cap_out * tanhf(z[nt][e] * cap_in);
        }
    }
    if (!whole) {
      asm volatile("");   // a branch, not predicated work on every page
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int key = key0 + g + (e >> 1) * 8;
          if (key < low[nt][e & 1] || key >= lim[nt][e & 1]) z[nt][e] = -INFINITY;
        }
    }
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 4; e++) grow |= z[nt][e] > base[nt][e & 1] + HEADROOM;
    if (__any_sync(0xffffffffu, grow)) {
      asm volatile("");
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float m = fmaxf(z[nt][e], z[nt][e + 2]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          m = fmaxf(m, base[nt][e]);
          const float f = m == -INFINITY ? 1.f : ex2(base[nt][e] - m);
          base[nt][e] = m;
          lift[nt][e] = m == -INFINITY ? 0.f : LIFT + raise - m;
          mt[nt][e] *= f;
#pragma unroll
          for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
              o[nt][gr][hf][e] *= f;
              o[nt][gr][hf][e + 2] *= f;
            }
        }
    }
    uint32_t p0[NT], p1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; e++) p[e] = ex2(z[nt][e] + lift[nt][e & 1]);
      p0[nt] = movmatrix(pack_f16(p[0], p[1]));   // tokens 2 t, 2 t + 1 of column g
      p1[nt] = movmatrix(pack_f16(p[2], p[3]));   // tokens 2 t + 8, 2 t + 9
    }
    {
      uint32_t v0[NG], v1[NG], s0[NG], s1[NG];
      const int x = g ^ (2 * t);   // pairs t and t + 4 share it
      lds(pg + L::VC + ((t * 8 + x) * NG) * 4, v0);
      lds(pg + L::VC + (((t + 4) * 8 + x) * NG) * 4, v1);
      lds(pg + L::VS + t * NG * 4, s0);
      lds(pg + L::VS + (t + 4) * NG * 4, s1);
      uint32_t m0 = 0, m1 = 0;   // rows 0 .. NG - 1: minima of the groups; row 4: ones
      if (g < NG) {
        m0 = *reinterpret_cast<const uint32_t*>(pg + L::VM + (t * NG + g) * 4);
        m1 = *reinterpret_cast<const uint32_t*>(pg + L::VM + ((t + 4) * NG + g) * 4);
      } else if (g == 4) {
        m0 = m1 = 0x3c003c00u;
      }
      if (!whole) {
        asm volatile("");
        // tokens no row sees: whatever their bytes hold (memory nobody wrote) must not reach the sums
        auto keep = [&](int tok) {
          const bool lo_ok = key0 + tok >= low_any && key0 + tok < lim_any;
          const bool hi_ok = key0 + tok + 1 >= low_any && key0 + tok + 1 < lim_any;
          return (lo_ok ? 0x0000ffffu : 0u) | (hi_ok ? 0xffff0000u : 0u);
        };
        const uint32_t keep0 = keep(2 * t), keep1 = keep(2 * t + 8);
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
          s0[gr] &= keep0;
          s1[gr] &= keep1;
        }
        m0 &= keep0;
        m1 &= keep1;
        // Values that are no numbers, at keys that some rows see and others do not: 0 * NaN would reach the others.
        uint32_t bad = MULTI ? nan_halves(m0) | nan_halves(m1) : 0;
#pragma unroll
        for (int gr = 0; gr < NG; gr++) bad |= MULTI ? nan_halves(s0[gr]) | nan_halves(s1[gr]) : 0;
        if (MULTI && __any_sync(0xffffffffu, bad)) {
          asm volatile("");
#pragma unroll
          for (int gr = 0; gr < NG; gr++) {   // (a group's minima are in the lanes of row gr)
            const uint32_t b0 = nan_halves(s0[gr]) | __shfl_sync(0xffffffffu, nan_halves(m0), gr * 4 + t);
            const uint32_t b1 = nan_halves(s1[gr]) | __shfl_sync(0xffffffffu, nan_halves(m1), gr * 4 + t);
            uint32_t toks = ((b0 & 1) << (2 * t)) | ((b0 >> 31) << (2 * t + 1)) | ((b1 & 1) << (2 * t + 8)) | ((b1 >> 31) << (2 * t + 9));
            toks |= __shfl_xor_sync(0xffffffffu, toks, 1);
            toks |= __shfl_xor_sync(0xffffffffu, toks, 2);
            s0[gr] &= ~b0;
            s1[gr] &= ~b1;
            if (g == gr) {
              m0 &= ~b0;
              m1 &= ~b1;
            }
#pragma unroll
            for (int c = 0; c < 2 * NT; c++)
              if (g == 0 && (toks & key_bits(key0, low[c >> 1][c & 1], lim[c >> 1][c & 1])))
                atomicOr(&sm.lost[(c >> 1) * 8 + 2 * t + (c & 1)], 1u << gr);
          }
        }
      }
      uint32_t s_top = max_h2(s0[0], s1[0]);
#pragma unroll
      for (int gr = 1; gr < NG; gr++) s_top = max_h2(s_top, max_h2(s0[gr], s1[gr]));
      if (__any_sync(0xffffffffu, reaches(s_top, s_most))) {   // scales that do not allow this raise
        asm volatile("");
        const float2 y = unpack_h2(s_top);
        const float top = warp_max(fmaxf(y.x, y.y));
        const int drop = min(raise, (int)(__float_as_uint(top) >> 23) - 126 - (MOST_RAISE - raise));
        const float f = __uint_as_float((uint32_t)(127 - drop) << 23);
        const uint32_t f2 = pack_f16(f, f);
        raise -= drop;
        s_most = raise == 0 ? 0x7c007c00u : pow2_h2(MOST_RAISE - raise);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          p0[nt] = mul_h2(p0[nt], f2);
          p1[nt] = mul_h2(p1[nt], f2);
#pragma unroll
          for (int e = 0; e < 2; e++) lift[nt][e] -= base[nt][e] == -INFINITY ? 0 : drop;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            mt[nt][e] *= f;
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
              o[nt][gr][0][e] *= f;
              o[nt][gr][1][e] *= f;
            }
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) mma_f16_16816(mt[nt], m0, 0u, m1, 0u, p0[nt], p1[nt]);
#pragma unroll
      for (int gr = 0; gr < NG; gr++) {
        const uint32_t w0 = v0[gr], w1 = v1[gr], u0 = w0 >> 8, u1 = w1 >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const uint32_t b0 = mul_h2(p0[nt], s0[gr]), b1 = mul_h2(p1[nt], s1[gr]);
          mma_f16_16816(o[nt][gr][0], w0 & M0, w0 & M4, w1 & M0, w1 & M4, b0, b1);   // dims 4 g, 4 g + 1
          mma_f16_16816(o[nt][gr][1], u0 & M0, u0 & M4, u1 & M0, u1 & M4, b0, b1);   // dims 4 g + 2, 4 g + 3
          if (FINE && few) {   // what the products p s lost, times the middle code 8
            const uint32_t e = add_h2(left_h2(p0[nt], s0[gr], b0), left_h2(p1[nt], s1[gr], b1));
            mma_f16_1688(o[nt][gr][0], 0x00080008u, 0x00800080u, e);
            mma_f16_1688(o[nt][gr][1], 0x00080008u, 0x00800080u, e);
          }
        }
      }
    }
    __syncwarp();   // every lane is done with the stage before it is refilled
  }

  // merge the CTA's warps; the ring is free once every warp has drained its copies
  __syncthreads();
  if (tid == 0 && sm.fail) report_error(a.err, 1);
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    float ml[NG][2];
#pragma unroll
    for (int gr = 0; gr < NG; gr++)
#pragma unroll
      for (int e = 0; e < 2; e++) ml[gr][e] = __shfl_sync(0xffffffffu, mt[nt][e], gr * 4 + t);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int col = nt * 8 + 2 * t + e;
#pragma unroll
      for (int gr = 0; gr < NG; gr++)
        *reinterpret_cast<float4*>(&sm.o[warp][col][gr * 32 + 4 * g]) =
            make_float4(fmaf(o[nt][gr][0][e], 16777216.f, ml[gr][e]), fmaf(o[nt][gr][0][e + 2], 1048576.f, ml[gr][e]),
                        fmaf(o[nt][gr][1][e], 16777216.f, ml[gr][e]), fmaf(o[nt][gr][1][e + 2], 1048576.f, ml[gr][e]));
      if (g == 4) {
        sm.base[warp][col] = base[nt][e] - raise;   // what the sums are against, without raise
        sm.sum[warp][col] = mt[nt][e];
      }
    }
  }
  __syncthreads();
  pdl_launch_dependents();
  const bool alone = n_split == 1;
  const int64_t part_col = block_no(b, rc, kvh, gridDim.x / n_split, a.Hkv) * COLS;
  float* part_ml = a.part + (int64_t)gridDim.z * gridDim.y * (gridDim.x / n_split) * COLS * n_split * D;
  for (int c = warp; c < COLS; c += W) {
    const int r = r0 + c;
    if (r >= R) break;
    const int qi = a.query_of(r), h = kvh * G + r - qi * G;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, sm.base[w][c]);
    const float sink = !CLUSTER && alone && a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    const float mt_ = fmaxf(m, sink), bs = mt_ == -INFINITY ? 0.f : mt_;
    float f[W], l = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) {
      f[w] = part_weight(sm.base[w][c], sm.sum[w][c], bs);
      l += f[w] * sm.sum[w][c];
    }
    if (sink != -INFINITY) l += ex2(sink - bs + LIFT);
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += 64) {
      const int d = d0 + 2 * lane;
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float2 y = *reinterpret_cast<const float2*>(&sm.o[w][c][d]);
        v.x += f[w] * y.x;
        v.y += f[w] * y.y;
      }
      if (MULTI && (sm.lost[c] >> (d / 32) & 1)) v.x = v.y = __int_as_float(0x7fffffff);
      if constexpr (CLUSTER) {
        *reinterpret_cast<float2*>(&sm.o[0][c][d]) = v;   // (this thread read the element last)
      } else if (alone) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const int64_t at = (int64_t)(tok0 + qi) * a.o_tok + (int64_t)h * a.o_head + d;
        store_elt(a.out, a.o_type, at, v.x * inv);
        store_elt(a.out, a.o_type, at + 1, v.y * inv);
      } else {
        *reinterpret_cast<float2*>(a.part + ((part_col + c) * n_split + split) * D + d) = v;
      }
    }
    if (CLUSTER ? lane == 0 : !alone && lane == 0) {
      float* ml = CLUSTER ? sm.ml[c] : part_ml + ((part_col + c) * n_split + split) * 2;
      ml[0] = mt_;
      ml[1] = l;
    }
  }
  if constexpr (CLUSTER) {
    cluster_sync();
    // 32 pairs of dims of a column are one warp's job; the jobs go round the cluster's CTAs
    for (int job = split + n_split * warp; job < COLS * D / 64; job += n_split * W) {
      const int c = job / (D / 64), d = job % (D / 64) * 64 + 2 * lane, r = r0 + c;
      if (r >= R) continue;
      const int qi = a.query_of(r), h = kvh * G + r - qi * G;
      const float sink = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
      const float2 y = lane < n_split ? remote_f2(sm.ml[c], lane) : make_float2(-INFINITY, 0.f);
      const float m = fmaxf(sink, warp_max(y.x));
      const float f = part_weight(y.x, y.y, m);
      float l = 0.f, acc[2] = {0.f, 0.f};
#pragma unroll 8
      for (int s = 0; s < n_split; s++) {
        const float2 z = remote_f2(&sm.o[0][c][d], s);
        merge_split(__shfl_sync(0xffffffffu, f, s), __shfl_sync(0xffffffffu, y.y, s), &z.x, l, acc);
      }
      if (sink != -INFINITY) l += ex2(sink - m + LIFT);
      const float inv = l != 0.f ? 1.f / l : 0.f;
      const int64_t at = (int64_t)(tok0 + qi) * a.o_tok + (int64_t)h * a.o_head + d;
      store_elt(a.out, a.o_type, at, acc[0] * inv);
      store_elt(a.out, a.o_type, at + 1, acc[1] * inv);
    }
    cluster_sync();   // shared memory stays until every CTA has read it
  }
}

// One warp merges the live splits of one query row: D / 32 dims a lane, up to 16 splits' loads in flight.
template <int D>
__global__ void __launch_bounds__(256) k_kv4_combine(const __grid_constant__ Kv4Attn a, int n_split, int whole, int grain, int cols, int row_chunks, float lift) {
  constexpr int V = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int no = blockIdx.x / (cols / 8), c = blockIdx.x % (cols / 8) * 8 + warp;   // of the row blocks that were split
  int b, rc, kvh;
  block_at((int64_t)whole + no, row_chunks, a.Hkv, b, rc, kvh);
  const int G = a.G;
  pdl_wait();
  const int64_t part_col = (int64_t)no * cols;
  const float* part_ml = a.part + (int64_t)gridDim.x * 8 * n_split * D;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + (part_col + c) * n_split;
  const float2 first = lane < n_split ? __ldcg(&ml[lane]) : make_float2(-INFINITY, 0.f);   // (travels with ctx)
  const int ctx = min(a.ctx[b], a.width * PAGE);
  int tok0 = b, n = 1;
  if (a.q_off) {
    tok0 = max(a.q_off[b], 0);
    n = min(min(a.q_off[b + 1], a.n_tokens) - tok0, a.max_new);
  }
  const int R = n * G, r0 = rc * cols;
  if (R <= r0) return;
  const Span sp = span_of(ctx, n, a.query_of(r0), a.query_of(min(R - 1, r0 + cols - 1)), a.window, n_split, grain, a.width);
  const int live = max(1, sp.live);   // an empty block's split 0 wrote zeros
  if (r0 + c < R) {
    const int r = r0 + c, qi = a.query_of(r), h = kvh * G + r - qi * G;
    const float sink = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    const float* po = a.part + (part_col + c) * n_split * D + V * lane;
    // (base, sum) of 32 splits a lane each; the partial rows' loads do not wait for them
    float m = sink, l = 0.f, acc[V] = {};
    for (int s0 = 0; s0 < live; s0 += 32) {
      const float2 y = s0 == 0 ? first : s0 + lane < live ? __ldcg(&ml[s0 + lane]) : make_float2(-INFINITY, 0.f);
      const float yb = s0 + lane < live ? y.x : -INFINITY;
      const float mn = fmaxf(m, warp_max(yb));
      const float keep = m == -INFINITY ? 0.f : ex2(m - mn), f = s0 + lane < live ? part_weight(y.x, y.y, mn) : 0.f;
      m = mn;
      l *= keep;
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] *= keep;
      const int e = min(32, live - s0);
#pragma unroll 16
      for (int s = 0; s < e; s++) {
        const float* p = po + (int64_t)(s0 + s) * D;
        float z[V];
        if constexpr (V == 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(p));
          z[0] = x.x; z[1] = x.y; z[2] = x.z; z[3] = x.w;
        } else {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(p));
          z[0] = x.x; z[1] = x.y;
        }
        merge_split(__shfl_sync(0xffffffffu, f, s), __shfl_sync(0xffffffffu, y.y, s), z, l, acc);
      }
    }
    if (sink != -INFINITY) l += ex2(sink - m + lift);
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int64_t at = (int64_t)(tok0 + qi) * a.o_tok + (int64_t)h * a.o_head + V * lane;
#pragma unroll
    for (int i = 0; i < V; i++) store_elt(a.out, a.o_type, at + i, acc[i] * inv);
  }
  pdl_launch_dependents();
}

void pdl(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
}

}  // namespace

Kv4AttnPlan kv4_attn_plan(const Kv4Attn& a, int n_sm) {
  Kv4AttnPlan p{};
  const int64_t rows = (int64_t)a.max_new * (a.H / a.Hkv);
  p.tc = a.tiles < 0 ? rows > prefill_rows(a.D) : a.tiles > 0;
  if (p.tc) {
    // 256 rows a CTA, one CTA a SM: the blocks that would fill less than half of a last wave have their keys
    // split, eight steps a split at least (448 blocks of 64 to 96 steps: 726 us whole, 649 with the last four split)
    p.row_chunks = (int)((rows + 255) / 256);
    const int64_t ctas = (int64_t)a.B * a.Hkv * p.row_chunks, last = ctas % n_sm;
    p.n_split = a.n_split > 0 ? a.n_split : (int)std::max<int64_t>(1, std::min<int64_t>(last ? n_sm / last : 1, a.width / 64));
    p.whole = p.n_split == 1 ? ctas : a.n_split > 0 ? 0 : ctas - last;
    p.part_floats = (ctas - p.whole) * 256 * p.n_split * (a.D + 2);
    return p;
  }
  // Columns a CTA: 16 at head dim 64 where there are that many rows, else 8.  More columns save unpacking but
  // cost registers and so warps: at head dim 128 two n-tiles (16 warps a SM become 8) took 29.5 us against
  // 24.0 at 16 x 2 tokens x 7 rows over 4097, 50.2 against 40.9 at 8 x 35 rows over 8000; at head dim 64 four
  // (8 warps) took 68.4 us against 56.5 with two at 16 x 40 rows over 4097, and one 48.3 against 38.3 with two
  // at 4 x 64 rows over 8000.
  p.nt = a.D == 64 && rows > 8 ? 2 : 1;
  p.row_chunks = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
  // Splits: 2 1/4 CTAs a SM, though no more than 40, and 192 pages each at most where every sequence fills its
  // table.  (us by splits: 16 x 8000 tokens over 4 KV heads 1: 67, 4: 32, 8: 25, 16: 31; 1 x 32000 over 4 8: 37,
  // 16: 22, 32: 18, 64: 22; 64 lanes up to 4000 over 4 1: 42, 2: 35, 4: 36, 8: 39; 32 lanes up to 32768 over 8
  // 2: 195, 8: 165, 16: 170, 32: 193.)
  const int64_t ctas = (int64_t)a.B * a.Hkv * p.row_chunks, most = (a.width + W - 1) / W;
  int64_t n = a.n_split;
  if (n <= 0)
    n = std::min(std::max<int64_t>({1, (a.width + 191) / 192, std::min<int64_t>(40, 9 * (int64_t)n_sm / (4 * ctas))}),
                 std::max<int64_t>(most, 1));
  // Up to 16 splits that are resident at once merge inside a cluster, without partial results in memory and a
  // second launch (1 x 2048 9.8 -> 5.8 us); a warp may have nine pages then before more splits pay for them.
  // Clusters do not span the groups of SMs, so up to c - 1 of a group's slots stay empty: at 2000 keys 28 blocks of
  // 16 take 8.8 us, 32 take 13.1; 140 of 4 15.2, 144 21.3.  (Sizes between the powers of two lose more slots than
  // they gain: 96 blocks over 4000 keys 21.7 us in fours, 26.6 in sixes.)
  const int resident = a.D == 64 && p.nt == 1 ? kResident<64, 1> : 4;   // (36 blocks of 16 at head dim 64: 7.8 us, as 28)
  int64_t c = 1;
  while (c < 16 && 2 * c * (ctas + 9) <= resident * n_sm && c < most) c *= 2;
  if (a.n_split > 0) {
    p.cluster = n > 1 && n <= c && (n & (n - 1)) == 0;
  } else if (c > 1 && n > 1 && (n <= c || a.width <= 9 * W * c)) {
    p.cluster = true;
    n = c;
  }
  p.n_split = (int)n;
  p.part_floats = p.n_split > 1 && !p.cluster ? ctas * 8 * p.nt * p.n_split * (a.D + 2) : 0;
  return p;
}

static void split_launch(const Kv4Attn& a, const Kv4AttnPlan& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_split * p.row_chunks), (unsigned)a.Hkv, (unsigned)a.B);
  cfg.blockDim = dim3(W * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  pdl(cfg, attr);
  if (p.cluster) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)p.n_split, 1, 1};
    cfg.numAttrs = 2;
  }
  auto go = [&](auto kern, size_t smem) {
    cfg.dynamicSmemBytes = smem;
    FAK_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (p.cluster) FAK_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    FAK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, p.n_split));
  };
  auto pick = [&](auto d, auto nt, auto cap, auto fine, auto multi) {
    constexpr int DV = decltype(d)::value, NTV = decltype(nt)::value;
    constexpr bool CAP = decltype(cap)::value, FINE = decltype(fine)::value, MULTI = decltype(multi)::value;
    if (p.cluster) go(k_kv4_attn<DV, NTV, CAP, true, FINE, MULTI>, sizeof(Smem<DV, NTV>));
    else go(k_kv4_attn<DV, NTV, CAP, false, FINE, MULTI>, sizeof(Smem<DV, NTV>));
  };
  auto by_rows = [&](auto d, auto nt, auto cap, auto fine) {
    if (a.max_new > 1) pick(d, nt, cap, fine, std::true_type{});
    else pick(d, nt, cap, fine, std::false_type{});
  };
  auto by_type = [&](auto d, auto nt, auto cap) {
    if (a.o_type == Elt::BF16) by_rows(d, nt, cap, std::false_type{});
    else by_rows(d, nt, cap, std::true_type{});
  };
  auto by_cap = [&](auto d, auto nt) {
    if (a.softcap > 0.f) by_type(d, nt, std::true_type{});
    else by_type(d, nt, std::false_type{});
  };
  using std::integral_constant;
  if (a.D == 128) by_cap(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  else if (p.nt == 1) by_cap(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else by_cap(integral_constant<int, 64>{}, integral_constant<int, 2>{});
}

void kv4_attn_launch(const Kv4Attn& a, const Kv4AttnPlan& p, cudaStream_t stream) {
  if (p.tc) kv4_prefill_launch(a, p, stream);
  else split_launch(a, p, stream);
  cudaLaunchAttribute attr[1];
  if (p.n_split > 1 && !p.cluster) {
    cudaLaunchConfig_t c2 = {};
    const int cols = p.tc ? 256 : 8 * p.nt;
    c2.gridDim = dim3((unsigned)(((int64_t)a.B * a.Hkv * p.row_chunks - p.whole) * (cols / 8)));
    c2.blockDim = dim3(256);
    c2.stream = stream;
    pdl(c2, attr);
    if (a.D == 128) FAK_CUDA_CHECK(cudaLaunchKernelEx(&c2, k_kv4_combine<128>, a, p.n_split, (int)p.whole, p.tc ? kTilesGrain : kRowsGrain, cols, p.row_chunks, p.tc ? kPrefillLift : LIFT));
    else FAK_CUDA_CHECK(cudaLaunchKernelEx(&c2, k_kv4_combine<64>, a, p.n_split, (int)p.whole, p.tc ? kTilesGrain : kRowsGrain, cols, p.row_chunks, p.tc ? kPrefillLift : LIFT));
  }
}

}  // namespace fak
