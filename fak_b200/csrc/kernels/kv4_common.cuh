// What the attention kernels over the 4-bit cache share.
#pragma once
#include "kv4.cuh"
#include "tc.cuh"

#include "../serve_ops.h"

#define FAK_HD __host__ __device__

namespace fak {
namespace kv4 {

constexpr int kRowsGrain = 4, kTilesGrain = 8;   // pages: a warp's one of the streaming CTA's four; a step of 128 keys

FAK_DEV uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
FAK_DEV uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
FAK_DEV uint32_t mul_h2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// halves that are no finite number, all bits set
FAK_DEV uint32_t nan_halves(uint32_t a) { return __vcmpeq2(a & 0x7c007c00u, 0x7c007c00u); }
// the bits of the 32 keys from key0 on that lie in [low, lim)
FAK_DEV uint32_t key_bits(int key0, int low, int lim) {
  const int lo = min(max(low - key0, 0), 32), hi = min(max(lim - key0, 0), 32);
  return hi > lo ? (0xffffffffu >> (32 - (hi - lo))) << lo : 0u;
}
FAK_DEV float2 unpack_h2(uint32_t a) { return __half22float2(*reinterpret_cast<__half2*>(&a)); }
FAK_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
FAK_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_addr(bar))
      : "memory");
}

template <int N>
FAK_DEV void lds(const uint8_t* p, uint32_t (&r)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x; r[1] = v.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int N>
FAK_DEV void ldg(const uint8_t* p, uint32_t (&r)[N]) {
  if constexpr (N == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = v.x; r[1] = v.y;
  } else {
    r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// The pages one CTA column block needs and how n_split splits share them, `grain` pages at least: the same
// arithmetic in the attention kernels and in the combine.  It depends on the sequence alone.
FAK_HD inline int spread(int pages, int n_split, int grain) {
  const int each = (pages + n_split - 1) / n_split;
  return each <= grain ? grain : (each + grain - 1) / grain * grain;
}
struct Span {
  int p0, p1, pps, live;   // pages [p0, p1), pages a split, splits that hold any
};
FAK_DEV Span span_of(int ctx, int n, int i_lo, int i_hi, int window, int n_split, int grain, int width) {
  Span s;
  const int last = min(ctx - n + i_hi, ctx - 1);               // the last key any row of the block sees
  const int first = window > 0 ? max(0, ctx - n + i_lo + 1 - window) : 0;
  s.p0 = first / PAGE;
  s.p1 = min(width, last / PAGE + 1);
  if (last < 0) s.p1 = s.p0;
  const int pages = max(0, s.p1 - s.p0);
  s.pps = spread(pages, n_split, grain);
  s.live = (pages + s.pps - 1) / s.pps;
  return s;
}

// Row blocks are numbered in the order of their launch: a sequence's last chunks, with the longest causal
// ranges, first.
FAK_DEV int64_t block_no(int b, int chunk, int kvh, int chunks, int Hkv) { return ((int64_t)b * chunks + chunks - 1 - chunk) * Hkv + kvh; }
FAK_DEV void block_at(int64_t no, int chunks, int Hkv, int& b, int& chunk, int& kvh) {
  const uint32_t rest = (uint32_t)no / (uint32_t)Hkv;
  kvh = (int)((uint32_t)no - rest * Hkv);
  b = (int)(rest / (uint32_t)chunks);
  chunk = chunks - 1 - (int)(rest - (uint32_t)b * chunks);
}

FAK_DEV float load_elt(const void* p, Elt t, int64_t i) {
  if (t == Elt::F32) return ((const float*)p)[i];
  if (t == Elt::F16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
FAK_DEV void store_elt(void* p, Elt t, int64_t i, float v) {
  if (t == Elt::F32) ((float*)p)[i] = v;
  else if (t == Elt::F16) ((__half*)p)[i] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}

}  // namespace kv4
}  // namespace fak
