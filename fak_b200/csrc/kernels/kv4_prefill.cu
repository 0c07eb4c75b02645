// Chunk attention over the 4-bit paged KV cache on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// The n * G query rows of a (sequence, KV head) -- row r is query r / G, head r % G of the group -- are
// packed into tiles of 128 rows, two tiles a CTA, so that one pass of dequantized keys and values serves
// 256 rows whatever the group size.  Warp roles:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one row a thread: S from TMEM, P = 2^(S c - base) back into
//                   TMEM as f16 over the first half of S's columns (the A operand of P V is read there);
//   warps 8-11      dequantization: codes of 128 keys, fetched a step ahead into registers, to f16 K
//                   [keys][dims] and V^T [dims][keys] in the 128-byte swizzle, two buffers each (bulk copies
//                   into rings of 12 page halves held 4.0k cycles a step on their own);
//   warps 12, 13    issue the matrix products of tile 0 / 1, S = Q K^T and O += P V, so that one tile's softmax
//                   runs under the other's products (one warp for both, polling, took 0.7k cycles to notice).
// The work of a tile goes in halves of 64 keys with two buffers of S: S of half u + 1 is multiplied while the
// softmax of half u runs, once the P in its columns (of half u - 1) is used up.  (128 x 64 products take 48
// cycles for every 16 dims, three quarters of the rate of 128 x 128 ones; whole steps with one buffer of S left
// the softmax waiting for its own products.)  A row's exponent base moves only when a half's maximum outgrows
// it by 2^8 (then O is scaled, after the product of the half before), so P <= 2^12 and S is read once.  Halves
// that need a mask or a soft-cap are rewritten in TMEM by a small loop first: the main loop then has one form,
// which matters because three roles' code shares the instruction caches (with the mask inside the unrolled
// loops, waits for instructions were the first stall and a step took 12.6k cycles).
// Orders: a K chunk of 8 dims keeps its nibble pairs (0,4) (1,5) (2,6) (3,7) and Q is stored in the same order.
// Rounding, whatever the types of q and out: Q to f16 after a power-of-two scaling of its row (exact for f16 down to
// 2^-21 of the row's largest, for bf16 to 2^-24), K and V to f16, P to f16; sums in f32.  (The 4 bits of a value are
// coarser than any of these.  rms error of f32 outputs up to 2.3e-4 of their size, with f32 queries 5.5e-4; rounding
// to f16 alone is 2.1e-4.)
// Values that are no numbers are taken out of the steps in which rows differ in the keys they see, and given at the
// end to the rows that see them.
// Every wait is bounded (tc::mbar_wait); no load uses multicast.
// Measured, 28 heads over 4 KV heads of 128 (graph of calls, us): 4096 tokens over 8192 670 (601 GFLOP, 897 TFLOP/s;
// without the split of the short last wave 744), 5 turns of up to 256 tokens over 8448 184 (845 TFLOP/s).  A step
// of 2 x 128 rows and 128 keys takes 4.2k cycles, of which products and their operands alone 3.1k (2.6k if nothing waited), with dequantization 3.7k: the
// schedulers issue in half of the cycles, 8.9k instructions a step, and the exponentials hold their unit for 2.1k.
#include "kv4_common.cuh"

#include <algorithm>
#include <cfloat>
#include <stdexcept>
#include <string>

namespace fak {
namespace {

using kv4::Lay;
using kv4::PAGE;
using kv4::Span;

constexpr int ROWS = 128;          // query rows per tile, two tiles a CTA
constexpr int KEYS = 128;          // keys per step
constexpr int PPT = KEYS / PAGE;   // pages per step
static_assert(PPT == kv4::kTilesGrain, "splits of whole steps");
constexpr int AHEAD = 4;           // steps between a page's prefetch into L2 and its use (cold pages: 197 -> 189 us)
constexpr int THREADS = 448;
constexpr float LIFT = 4.f, HEADROOM = 8.f;
constexpr float LOG2E = 1.4426950408889634f;

// Steps with keys that some rows of the block see and others do not: its 256 rows are at most 256 queries, so those
// keys lie in the first four steps (windows) and the last four.
constexpr int EDGE_STEPS = 8;
FAK_DEV int edge_slot(int j, int NJ) { return NJ <= EDGE_STEPS || j < EDGE_STEPS / 2 ? j : max(0, EDGE_STEPS - (NJ - j)); }
FAK_DEV int edge_step(int slot, int NJ) { return NJ <= EDGE_STEPS || slot < EDGE_STEPS / 2 ? slot : NJ - EDGE_STEPS + slot; }

template <int D>
struct Smem {
  alignas(1024) __half q[2][D / 64][ROWS * 64];    // [tile][64-dim half][row][64]
  alignas(1024) __half k[2][D / 64][KEYS * 64];    // [buffer][64-dim half][key][64]
  alignas(1024) __half v[2][2][D * 64];            // [buffer][64-key half][dim][64]
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];   // [tile][64-key half]
  uint32_t tmem;
  int fail;
  int lost_any;                          // values that are no numbers were taken out of V, at these tokens of
  uint32_t lost[EDGE_STEPS][D / 32][4];  // [step][group][token]; see edge_slot
};

// f16 operands, f32 accumulator, both K-major
constexpr uint32_t idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

FAK_DEV uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r;
}
// D (+)= A B by the lane with `lead` set; operands by the low words of their descriptors (high word `hi`)
FAK_DEV void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 x, y;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 x, {%1, %3};\n"
      " mov.b64 y, {%2, %3};\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
FAK_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 y;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 y, {%2, %3};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
FAK_DEV void commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(tc::smem_addr(bar)),
      "r"(lead)
      : "memory");
}
// waits for this thread's TMEM loads; the operands tie their uses to the wait
FAK_DEV void ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
FAK_DEV void ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
FAK_DEV void ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28])::"memory");
  asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
FAK_DEV uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
FAK_DEV uint32_t h2_add(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The four half2 of a code word, times s plus m.  1024 + c and 1024 + 16 c come from one AND-OR; the
// subtraction (and the product with 1/16) is exact.
FAK_DEV void dequant_word(uint32_t w, uint32_t s, uint32_t m, uint32_t (&o)[4]) {
  constexpr uint32_t BIAS = 0x64006400u;
  const uint32_t u = w >> 8;
  o[0] = h2_fma(h2_add((w & 0x000f000fu) | BIAS, 0xe400e400u), s, m);              // - 1024
  o[1] = h2_fma(h2_fma((w & 0x00f000f0u) | BIAS, 0x2c002c00u, 0xd400d400u), s, m); // / 16 - 64
  o[2] = h2_fma(h2_add((u & 0x000f000fu) | BIAS, 0xe400e400u), s, m);
  o[3] = h2_fma(h2_fma((u & 0x00f000f0u) | BIAS, 0x2c002c00u, 0xd400d400u), s, m);
}
// two f32 at a time
FAK_DEV uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
FAK_DEV float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
FAK_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
FAK_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
FAK_DEV uint32_t dup_lo(uint32_t x) {
  const __half2 r = __low2half2(*reinterpret_cast<__half2*>(&x));
  return *reinterpret_cast<const uint32_t*>(&r);
}
FAK_DEV uint32_t dup_hi(uint32_t x) {
  const __half2 r = __high2half2(*reinterpret_cast<__half2*>(&x));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int D, bool CAP>
__global__ void __launch_bounds__(THREADS, 1)
k_kv4_prefill(const __grid_constant__ Kv4Attn a, int splits, int whole, int n_blk) {
  using L = Lay<D>;
  constexpr int NG = L::NG;
  extern __shared__ uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the first `whole` row blocks have a CTA each, the others `splits`
  const int n_split = blockIdx.x < whole ? 1 : splits, past = max(0, (int)blockIdx.x - whole);
  const int split = past % n_split, no = past / n_split;   // (number among the blocks that are split)
  int b, blk, kvh;
  kv4::block_at(blockIdx.x < whole ? blockIdx.x : whole + no, n_blk, a.Hkv, b, blk, kvh);
  const int G = a.G;
  pdl_wait();
  const int ctx = min(a.ctx[b], a.width * PAGE);
  if (threadIdx.x == 0 && a.ctx[b] > ctx) report_error(a.err, 2);   // more keys than the table has pages for
  int tok0 = b, n = 1;
  if (a.q_off) {
    tok0 = max(a.q_off[b], 0);
    n = min(a.q_off[b + 1], a.n_tokens) - tok0;
    if (n > a.max_new) {
      report_error(a.err, 3);
      n = a.max_new;
    }
  }
  const int R = n * G, r0 = blk * 2 * ROWS;
  if (R <= r0) return;
  const int i_first = a.query_of(r0), i_last = a.query_of(min(R - 1, r0 + 2 * ROWS - 1));
  const Span sp = kv4::span_of(ctx, n, i_first, i_last, a.window, n_split, kv4::kTilesGrain, a.width);
  const int p_begin = sp.p0 + split * sp.pps, p_end = min(sp.p1, p_begin + sp.pps);
  if (p_begin >= p_end && !(split == 0 && sp.live == 0)) return;
  const int n_pages = max(0, p_end - p_begin);
  const int NJ = (n_pages + PPT - 1) / PPT, NU = (n_pages + PPT / 2 - 1) / (PPT / 2);   // steps; halves of 64 keys
  const int tiles = R - r0 > ROWS ? 2 : 1;
  const int lim_any = ctx - n + i_last + 1;                                            // keys some row sees: below
  const int low_any = a.window > 0 ? max(0, ctx - n + i_first + 1 - a.window) : 0;     // and from here
  const int lim_all = ctx - n + i_first + 1;                                           // keys every row sees: below
  const int low_all = a.window > 0 ? max(0, ctx - n + i_last + 1 - a.window) : 0;      // and from here

  if (threadIdx.x == 0) {
    tc::mbar_init(&sm.q_full, 4 * tiles);
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&sm.k_full[i], 4);
      tc::mbar_init(&sm.k_empty[i], tiles);
      tc::mbar_init(&sm.v_full[i], 4);
      tc::mbar_init(&sm.v_empty[i], tiles);
      for (int h = 0; h < 2; h++) {
        tc::mbar_init(&sm.s_full[i][h], 1);
        tc::mbar_init(&sm.p_full[i][h], 4);
        tc::mbar_init(&sm.pv_done[i][h], 1);
      }
    }
    sm.fail = sm.lost_any = 0;
    tc::fence_mbar_init();
  }
  if (threadIdx.x < EDGE_STEPS * NG * 4) (&sm.lost[0][0][0])[threadIdx.x] = 0;
  if (warp == 12) {
    tc::tmem_alloc(&sm.tmem, 512);   // S0 [0, 128) S1 [128, 256) O0 [256, 256 + D) O1 [256 + D, 256 + 2 D)
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem;
  int* fail = &sm.fail;

  if (warp >= 12) {
    if (const int t = warp - 12; t < tiles && NJ > 0) {
      // ---- matrix products of tile t.  The whole warp walks the loop, so that descriptors stay warp-uniform; one
      // lane's instructions take effect.
      constexpr uint32_t id_s = idesc_f16(ROWS, KEYS / 2), id_o = idesc_f16(ROWS, D);
      // 64-dim halves of Q and K, 64-key halves of K and V, in units of 16 bytes
      constexpr uint32_t HALF_Q = ROWS * 128 / 16, KEYS_K = KEYS / 2 * 128 / 16, HALF_V = D * 128 / 16;
      const uint32_t leader = elect_one();
      const uint32_t hi = (uint32_t)(tc::smem_desc_sw128(sm.q) >> 32);      // (the same for every operand)
      const uint32_t lq = (uint32_t)tc::smem_desc_sw128(sm.q) + t * (D / 64) * HALF_Q;
      const uint32_t lk = (uint32_t)tc::smem_desc_sw128(sm.k), lv = (uint32_t)tc::smem_desc_sw128(sm.v);
      const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * D;
      tc::mbar_wait(&sm.q_full, 0, fail);
#pragma unroll 1
      for (int u = 0; u <= NU; u++) {   // S of half u, then O += P V of half u - 1
        if (u < NU) {
          const int j = u >> 1, h = u & 1;
          const uint32_t buf = j & 1;
          if (h == 0) tc::mbar_wait(&sm.k_full[buf], (uint32_t)(j >> 1) & 1, fail);
          if (u > 1) tc::mbar_wait(&sm.pv_done[t][h], (uint32_t)(j - 1) & 1, fail);   // P of half u - 2 sits in these columns
          __syncwarp();
          tc::tc_fence_after();
          const uint32_t k = lk + buf * (D / 64) * HALF_Q + h * KEYS_K;
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)
            mma_ss(ts + h * 64, lq + (kk >> 2) * HALF_Q + 2 * (kk & 3), k + (kk >> 2) * HALF_Q + 2 * (kk & 3), hi, id_s, kk != 0, leader);
          commit(&sm.s_full[t][h], leader);
          if (h == 1) commit(&sm.k_empty[buf], leader);
        }
        if (u > 0) {
          const int j = (u - 1) >> 1, h = (u - 1) & 1;
          const uint32_t buf = j & 1;
          if (h == 0) tc::mbar_wait(&sm.v_full[buf], (uint32_t)(j >> 1) & 1, fail);
          tc::mbar_wait(&sm.p_full[t][h], (uint32_t)j & 1, fail);
          __syncwarp();
          tc::tc_fence_after();
          const uint32_t v = lv + (buf * 2 + h) * HALF_V;
#pragma unroll
          for (int ks = 0; ks < 4; ks++) mma_ts(to, ts + h * 64 + ks * 8, v + 2 * ks, hi, id_o, ks != 0 || u > 1, leader);
          commit(&sm.pv_done[t][h], leader);
          if (h == 1) commit(&sm.v_empty[buf], leader);
        }
      }
    }
  } else if (warp >= 8) {
    // ---- dequantization: this warp's two pages of every step, fetched a step ahead into registers
    const int w = warp - 8;
    // K lanes: (token bits 0, 1, 2; t); V lanes: (g, half of the page, page of the pair)
    const int kt = lane & 3, ktok = ((lane >> 2) & 1) * 4 + (lane >> 3);
    const int vg = (lane & 1) | (lane >> 3) << 1, vh = (lane >> 1) & 1, vp = (lane >> 2) & 1;
    const int* table = a.table + (int64_t)b * a.table_stride + p_begin;
    uint32_t kc[4][NG], ks[4][NG / 2], km[4][NG / 2], vc[4][NG], vs[4][NG], vm[4][NG];
    auto entries = [&](int j) {   // 16 steps of the table: lane 2 i + u holds page u of step j + i
      const int i = (j + (lane >> 1)) * PPT + 2 * w + (lane & 1);
      int pid = i < n_pages ? table[i] : 0;
      if ((unsigned)pid >= (uint64_t)a.n_pages) {
        report_error(a.err, 2);
        pid = 0;
      }
      return pid;
    };
    int ids = NJ > 0 ? entries(0) : 0, ids_next = 0;
    auto prefetch = [&](int pid) {   // a page, into L2
      const uint8_t* pg = a.pages + ((int64_t)pid * a.Hkv + kvh) * L::BYTES;
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(pg), "r"(L::BYTES));
    };
    if (lane < 2 * AHEAD && (lane >> 1) < NJ) prefetch(ids);
    auto fetch_k = [&](int j) {
      if (j >= NJ) return;
      if ((j & 15) == 0) {
        if (j > 0) ids = ids_next;
        ids_next = entries(j + 16);
      }
      const int jp = j + AHEAD, pid = __shfl_sync(0xffffffffu, (jp ^ j) & 16 ? ids_next : ids, 2 * (jp & 15) + (lane & 1));
      if (lane < 2 && jp < NJ) prefetch(pid);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint8_t* pg = a.pages + ((int64_t)__shfl_sync(0xffffffffu, ids, 2 * (j & 15) + u) * a.Hkv + kvh) * L::BYTES;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          const int tok = hf * 8 + ktok;
          kv4::ldg(pg + L::KC + tok * (D / 2) + kt * 4 * NG, kc[2 * u + hf]);
          kv4::ldg(pg + L::KS + tok * 2 * NG, ks[2 * u + hf]);
          kv4::ldg(pg + L::KM + tok * 2 * NG, km[2 * u + hf]);
        }
      }
    };
    auto fetch_v = [&](int j) {
      if (j >= NJ) return;
      const uint8_t* pg = a.pages + ((int64_t)__shfl_sync(0xffffffffu, ids, 2 * (j & 15) + vp) * a.Hkv + kvh) * L::BYTES;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int p = vh * 4 + e;
        kv4::ldg(pg + L::VC + ((p * 8 + (vg ^ (2 * e))) * NG) * 4, vc[e]);
        kv4::ldg(pg + L::VS + p * NG * 4, vs[e]);
        kv4::ldg(pg + L::VM + p * NG * 4, vm[e]);
      }
    };
    fetch_k(0);
    fetch_v(0);
#pragma unroll 1
    for (int j = 0; j < NJ; j++) {
      const int buf = j & 1;
      const uint32_t free_parity = (uint32_t)((j >> 1) & 1) ^ 1u;
      tc::mbar_wait(&sm.k_empty[buf], free_parity, fail);
      // (rows of pages that do not exist hold whatever page 0 does; they are masked in S)
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int row = (2 * w + (x >> 1)) * PAGE + (x & 1) * 8 + ktok;
#pragma unroll
        for (int gr = 0; gr < NG; gr++) {
          uint32_t o[4];
          dequant_word(kc[x][gr], gr & 1 ? dup_hi(ks[x][gr / 2]) : dup_lo(ks[x][gr / 2]), gr & 1 ? dup_hi(km[x][gr / 2]) : dup_lo(km[x][gr / 2]), o);
          uint8_t* dst = reinterpret_cast<uint8_t*>(sm.k[buf][gr >> 1]) + row * 128 + ((((gr & 1) * 4 + kt) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.k_full[buf]);

      const int i = j * PPT + 2 * w + vp, key0 = (p_begin + i) * PAGE, step0 = (p_begin + j * PPT) * PAGE;
      if (step0 < low_all || step0 + KEYS > min(lim_all, p_end * PAGE)) {
        // tokens no row sees (memory nobody wrote, pages that do not exist): zero
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int key = key0 + 2 * (vh * 4 + e);
          const uint32_t keep = (i < n_pages && key >= low_any && key < lim_any ? 0x0000ffffu : 0u) |
                                (i < n_pages && key + 1 >= low_any && key + 1 < lim_any ? 0xffff0000u : 0u);
#pragma unroll
          for (int gr = 0; gr < NG; gr++) {
            vs[e][gr] &= keep;
            vm[e][gr] &= keep;
          }
        }
        // values that are no numbers: 0 * NaN would reach the rows that do not see them
        uint32_t bad = 0;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int gr = 0; gr < NG; gr++) bad |= kv4::nan_halves(vs[e][gr]) | kv4::nan_halves(vm[e][gr]);
        if (__any_sync(0xffffffffu, bad)) {
          asm volatile("");
          const int slot = edge_slot(j, NJ);
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int gr = 0; gr < NG; gr++) {
              const uint32_t b = kv4::nan_halves(vs[e][gr]) | kv4::nan_halves(vm[e][gr]);
              const int tok = (2 * w + vp) * PAGE + 2 * (vh * 4 + e);
              vs[e][gr] &= ~b;
              vm[e][gr] &= ~b;
              if (b && vg == 0) {
                atomicOr(&sm.lost[slot][gr][tok >> 5], ((b & 1) | (b >> 31) << 1) << (tok & 31));
                sm.lost_any = 1;
              }
            }
        }
      }
      fetch_k(j + 1);
      tc::mbar_wait(&sm.v_empty[buf], free_parity, fail);
      const int pos = 2 * w + vp, chunk = (pos & 3) * 2 + vh;
#pragma unroll
      for (int gr = 0; gr < NG; gr++) {
        uint32_t o[4][4];
#pragma unroll
        for (int e = 0; e < 4; e++) dequant_word(vc[e][gr], vs[e][gr], vm[e][gr], o[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int d = gr * 32 + 4 * vg + e;
          uint8_t* dst = reinterpret_cast<uint8_t*>(sm.v[buf][pos >> 2]) + d * 128 + ((chunk ^ (d & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = make_uint4(o[0][e], o[1][e], o[2][e], o[3][e]);
        }
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.v_full[buf]);
      fetch_v(j + 1);
    }
  } else if ((warp >> 2) < tiles) {
    // ---- softmax of tile t, one row a thread
    const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int rr = r0 + t * ROWS + row;
    const bool live = rr < R;
    const int qi = live ? a.query_of(rr) : 0, h = kvh * G + (live ? rr - qi * G : 0);
    float cf;
    {
      // the row to f16, its largest value scaled into [2^7, 2^8)
      const int64_t at = (int64_t)(tok0 + qi) * a.q_tok + (int64_t)h * a.q_head;
      const bool packed = a.q_vec && a.q_type != Elt::F32;
      auto load8 = [&](int c, float (&x)[8]) {
        if (!live) {
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = 0.f;
        } else if (packed) {
          const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + at + 8 * c);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 y = kv4::unpack_h2(w[e]);
            x[2 * e] = a.q_type == Elt::F16 ? y.x : bf16_bits_lo(w[e]);
            x[2 * e + 1] = a.q_type == Elt::F16 ? y.y : bf16_bits_hi(w[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = kv4::load_elt(a.q, a.q_type, at + 8 * c + e);
        }
      };
      float amax = 0.f;   // (the row is read twice, the second time out of L1)
#pragma unroll 4
      for (int c = 0; c < D / 8; c++) {
        float x[8];
        load8(c, x);
#pragma unroll
        for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
      }
      const int ex = (int)(__float_as_uint(amax) >> 23);
      const float f = __uint_as_float((uint32_t)(ex == 255 ? 127 : max(1, min(127 + 126, 127 + 7 + 127 - ex))) << 23);
#pragma unroll 4
      for (int c = 0; c < D / 8; c++) {
        float x[8];
        load8(c, x);
        uint8_t* dst = reinterpret_cast<uint8_t*>(sm.q[t][c >> 3]) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = make_uint4(kv4::pack_f16(x[0] * f, x[4] * f), kv4::pack_f16(x[1] * f, x[5] * f),
                                                    kv4::pack_f16(x[2] * f, x[6] * f), kv4::pack_f16(x[3] * f, x[7] * f));
      }
      // (never 0: a masked logit, -inf, is multiplied by it; |S| is at most 2^31, so that logits stay below 2^-94 there)
      cf = fmaxf(a.scale / f * (CAP ? 1.f : LOG2E), FLT_MIN);
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.q_full);
    }
    const float cap_in = CAP ? 1.f / a.softcap : 0.f, cap_out = CAP ? a.softcap * LOG2E : 0.f;
    const int lim = live ? min(ctx - n + qi + 1, ctx) : 0;
    const int low = a.window > 0 ? max(0, lim - a.window) : 0;
    // keys every live row of the warp sees
    int lim_min = live ? lim : INT_MAX, low_max = low;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, d));
      low_max = max(low_max, __shfl_xor_sync(0xffffffffu, low_max, d));
    }
    const uint32_t ts = tmem + ((uint32_t)(quarter * 32) << 16) + t * 128;
    const uint32_t to = tmem + ((uint32_t)(quarter * 32) << 16) + 256 + t * D;
    float base = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int u = 0; u < NU; u++) {   // 64 keys
      const int key0 = p_begin * PAGE + u * (KEYS / 2);
      const uint32_t par = (uint32_t)(u >> 1) & 1, su = ts + (u & 1) * 64;
      tc::mbar_wait(&sm.s_full[t][u & 1], par, fail);
      tc::tc_fence_after();
      if (CAP || key0 < low_max || key0 + KEYS / 2 > lim_min) {
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          uint32_t x[16];
          tc::tmem_ld16(su + c * 16, x);
          ld_wait(x);
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const int key = key0 + c * 16 + e;
            float y = __uint_as_float(x[e]);
            if constexpr (CAP) y = cap_out * tanhf(y * cf * cap_in);
            x[e] = __float_as_uint(key >= low && key < lim ? y : -INFINITY);
          }
          tc::tmem_st16(su + c * 16, x);
        }
        tc::tmem_st_wait();
      }
      const float mul = CAP ? 1.f : cf;
      uint32_t x[2][32];
      ld32(su, x[0]);
      ld32(su + 32, x[1]);
      ld_wait(x[0]);
      ld_wait(x[1]);
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 64; e += 2)
        m4[(e >> 1) & 3] = fmaxf(m4[(e >> 1) & 3], fmaxf(__uint_as_float(x[e >> 5][e & 31]), __uint_as_float(x[e >> 5][(e & 31) + 1])));
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mul;
      if (__any_sync(0xffffffffu, mx > base + HEADROOM)) {
        // some row outgrew its base: every row of the warp moves to its maximum, once the half before is multiplied
        const float nw = fmaxf(base, mx), f = nw == -INFINITY ? 1.f : kv4::ex2(base - nw);
        if (u > 0) {
          tc::mbar_wait(&sm.pv_done[t][(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1, fail);
          tc::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; c++) {
            uint32_t y[16];
            tc::tmem_ld16(to + c * 16, y);
            ld_wait(y);
#pragma unroll
            for (int e = 0; e < 16; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
            tc::tmem_st16(to + c * 16, y);
          }
        }
        l *= f;
        base = nw;
      }
      const float nb = base == -INFINITY ? 0.f : LIFT - base;
      const uint64_t mul2 = pair(mul, mul), nb2 = pair(nb, nb);
      uint64_t s2[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 2; c++) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 z = unpair(fma2(pair(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), mul2, nb2));
          const float p0 = kv4::ex2(z.x), p1 = kv4::ex2(z.y);
          s2[(e >> 1) & 1] = add2(s2[(e >> 1) & 1], pair(p0, p1));
          pk[e >> 1] = kv4::pack_f16(p0, p1);
        }
        tc::tmem_st16(su + c * 16, pk);   // (columns of S that have been read)
      }
      const float2 sum = unpair(add2(s2[0], s2[1]));
      l += sum.x + sum.y;
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sm.p_full[t][u & 1]);
    }
    // ---- output
    const bool alone = n_split == 1;
    if (NU > 0) {
      tc::mbar_wait(&sm.pv_done[t][(NU - 1) & 1], (uint32_t)((NU - 1) >> 1) & 1, fail);
      tc::tc_fence_after();
      tc::mbar_wait(&sm.v_full[(NJ - 1) & 1], (uint32_t)((NJ - 1) >> 1) & 1, fail);   // (long over: for what it publishes)
    }
    uint32_t lost = 0;   // groups with a value that this row sees and that is no number
    if (sm.lost_any) {
      for (int i = 0; i < EDGE_STEPS * NG * 4; i++)
        if ((&sm.lost[0][0][0])[i] & kv4::key_bits((p_begin + edge_step(i / (NG * 4), NJ) * PPT) * PAGE + i % 4 * 32, low, lim))
          lost |= 1u << (i / 4 % NG);
    }
    const float sink = alone && a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    float f = 1.f;
    if (alone) {
      const float top = fmaxf(base, sink);
      if (sink != -INFINITY) {
        f = base == -INFINITY ? 0.f : kv4::ex2(base - top);
        l = l * f + kv4::ex2(sink - top + LIFT);
      }
      f = l != 0.f ? f / l : 0.f;
    }
    const int64_t part_row = ((int64_t)no * (2 * ROWS) + t * ROWS + row) * n_split + split;
    const int64_t at = (int64_t)(tok0 + qi) * a.o_tok + (int64_t)h * a.o_head;
#pragma unroll 1
    for (int c = 0; c < D / 16; c++) {
      uint32_t o[16];
      if (NU > 0) {
        tc::tmem_ld16(to + c * 16, o);
        ld_wait(o);
      } else {
#pragma unroll
        for (int e = 0; e < 16; e++) o[e] = 0;
      }
      if (lost >> (c >> 1) & 1) {
#pragma unroll
        for (int e = 0; e < 16; e++) o[e] = 0x7fffffffu;
      }
      if (live && alone) {
        if (a.o_vec) {
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float y0 = __uint_as_float(o[2 * e]) * f, y1 = __uint_as_float(o[2 * e + 1]) * f;
            y[e] = a.o_type == Elt::F16 ? kv4::pack_f16(y0, y1) : kv4::pack_bf16x2(y0, y1);
          }
          uint4* dst = reinterpret_cast<uint4*>((uint16_t*)a.out + at + c * 16);
          dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
          dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e++) kv4::store_elt(a.out, a.o_type, at + c * 16 + e, __uint_as_float(o[e]) * f);
        }
      } else if (live) {
        float4* dst = reinterpret_cast<float4*>(a.part + part_row * D + c * 16);
#pragma unroll
        for (int e = 0; e < 4; e++)
          dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
      }
      __syncwarp();
    }
    if (!alone && live) {
      float* ml = a.part + (int64_t)(gridDim.x - whole) * (2 * ROWS) * D + part_row * 2;
      ml[0] = base;
      ml[1] = l;
    }
    tc::tc_fence_before();
  }
  pdl_launch_dependents();
  __syncthreads();
  if (threadIdx.x == 0 && sm.fail) report_error(a.err, 1);
  if (warp == 12) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace

void kv4_prefill_launch(const Kv4Attn& a, const Kv4AttnPlan& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.whole + ((int64_t)a.B * a.Hkv * p.row_chunks - p.whole) * p.n_split));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto go = [&](auto kern, size_t smem) {
    cfg.dynamicSmemBytes = smem + 1024;
    FAK_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes));
    FAK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, p.n_split, (int)p.whole, p.row_chunks));
  };
  const bool cap = a.softcap > 0.f;
  if (a.D == 128 && cap) go(k_kv4_prefill<128, true>, sizeof(Smem<128>));
  else if (a.D == 128) go(k_kv4_prefill<128, false>, sizeof(Smem<128>));
  else if (cap) go(k_kv4_prefill<64, true>, sizeof(Smem<64>));
  else go(k_kv4_prefill<64, false>, sizeof(Smem<64>));
}

}  // namespace fak
