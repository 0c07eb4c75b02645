// Append into and read from the 4-bit KV cache (layout in kv4.cuh).
//
// Quantization of a group x[32], after clamping to +-65504:  m = f16(min x),  s = f16((max x - m) / 15),
// code = rint((x - m) / s) clamped to [0, 15], all codes 0 where s = 0 (a constant group).  f16 holds the
// minimum to 11 bits, more than the bf16 values that come in; the subtraction and the division are done
// in f32.  A group that holds a not-a-number stores m = NaN and reads back as NaN.
//
// Eight lanes hold one group, four consecutive dims each: a warp takes one row at head dim 128, two at
// 64.  Bound by the bytes read (2 D each of K and V per row against 20 D / 16 written).
#include "kv4.cuh"

#include <cuda_fp16.h>
#include <stdexcept>
#include <string>

#include "../serve_ops.h"

namespace fak {
namespace {

template <typename T>
FAK_DEV void load4(const T* p, bool vec, float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
      return;
    }
  } else {
    if (vec) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      T h[4];
      memcpy(h, &u, 8);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (float)h[i];
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (float)p[i];
}

// Four values of a group held by 8 lanes -> their codes (one u16), the group's scale and minimum.
FAK_DEV uint32_t quant4(float (&x)[4], __half& s16, __half& m16) {
  constexpr float LIM = 65504.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    nan |= x[i] != x[i];
    x[i] = fminf(fmaxf(x[i], -LIM), LIM);
  }
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const uint32_t votes = __ballot_sync(0xffffffffu, nan) >> (threadIdx.x & 24);
  m16 = __float2half_rn(lo);
  const float m = __half2float(m16);
  s16 = __float2half_rn(__fdiv_rn(hi - m, 15.f));
  const float s = __half2float(s16);
  uint32_t c = 0;
  if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float q = rintf(__fdiv_rn(x[i] - m, s));
      c |= (uint32_t)(int)fminf(fmaxf(q, 0.f), 15.f) << (4 * i);
    }
  }
  if (votes & 0xffu) {   // a NaN in the group
    m16 = __ushort_as_half(0x7fff);
    s16 = __ushort_as_half(0);
    c = 0;
  }
  return c;
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
k_kv4_append(Kv4Rows r, const int* __restrict__ slot, int64_t n_rows, int Hkv, uint8_t* __restrict__ pages,
             int64_t n_pages, int* __restrict__ err) {
  using L = kv4::Lay<D>;
  constexpr int RPW = 4 / L::NG;   // rows per warp
  pdl_wait();
  const int lane = threadIdx.x & 31, u = lane >> 3, j = lane & 7;
  const int grp = u % L::NG;
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = warp * RPW + u / L::NG;
  const bool live = row < n_rows;
  const int64_t tok = live ? row / Hkv : 0;
  const int h = live ? (int)(row % Hkv) : 0;
  const int sl = live ? slot[tok] : -1;
  const bool in = sl >= 0 && sl / kv4::PAGE < n_pages;
  if (sl >= 0 && !in) report_error(err, 2);
  float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    const int d = grp * 32 + 4 * j;
    load4((const T*)r.k + (tok >> 4) * r.ks_page + (tok & 15) * r.ks_row + h * r.ks_head + d, r.vec, k);
    load4((const T*)r.v + (tok >> 4) * r.vs_page + (tok & 15) * r.vs_row + h * r.vs_head + d, r.vec, v);
  }
  __half ks, km, vs, vm;
  const uint32_t kc = quant4(k, ks, km), vc = quant4(v, vs, vm);
  if (in) {
    uint8_t* pg = pages + ((int64_t)(sl >> 4) * Hkv + h) * L::BYTES;
    const int t = sl & 15;
    *reinterpret_cast<uint16_t*>(pg + L::k_u16(t, grp, j)) = (uint16_t)kc;
    *reinterpret_cast<uint16_t*>(pg + L::v_u16(t, grp, j)) = (uint16_t)vc;
    if (j == 0) *reinterpret_cast<__half*>(pg + L::KS + L::k_meta(t, grp)) = ks;
    if (j == 1) *reinterpret_cast<__half*>(pg + L::KM + L::k_meta(t, grp)) = km;
    if (j == 2) *reinterpret_cast<__half*>(pg + L::VS + L::v_meta(t, grp)) = vs;
    if (j == 3) *reinterpret_cast<__half*>(pg + L::VM + L::v_meta(t, grp)) = vm;
  }
  pdl_launch_dependents();
}

template <typename T>
FAK_DEV void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    T h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = (T)x[i];
    uint2 u;
    memcpy(&u, h, 8);
    *reinterpret_cast<uint2*>(p) = u;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
k_kv4_read(const uint8_t* __restrict__ pages, int64_t n_pages, const int* __restrict__ slot, int64_t n_rows, int Hkv,
           T* __restrict__ ko, T* __restrict__ vo, int* __restrict__ err) {
  using L = kv4::Lay<D>;
  constexpr int RPW = 4 / L::NG;
  pdl_wait();
  const int lane = threadIdx.x & 31, u = lane >> 3, j = lane & 7;
  const int grp = u % L::NG;
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = warp * RPW + u / L::NG;
  if (row < n_rows) {
    const int64_t tok = row / Hkv;
    const int h = (int)(row % Hkv);
    const int sl = slot[tok];
    const bool in = sl >= 0 && sl / kv4::PAGE < n_pages;
    if (sl >= 0 && !in) report_error(err, 2);
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (in) {
      const uint8_t* pg = pages + ((int64_t)(sl >> 4) * Hkv + h) * L::BYTES;
      const int t = sl & 15;
      const uint32_t kc = *reinterpret_cast<const uint16_t*>(pg + L::k_u16(t, grp, j));
      const uint32_t vc = *reinterpret_cast<const uint16_t*>(pg + L::v_u16(t, grp, j));
      auto h16 = [&](int at) { return __half2float(*reinterpret_cast<const __half*>(pg + at)); };
      const float ks = h16(L::KS + L::k_meta(t, grp)), km = h16(L::KM + L::k_meta(t, grp));
      const float vs = h16(L::VS + L::v_meta(t, grp)), vm = h16(L::VM + L::v_meta(t, grp));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        // separate roundings of the product (exact: 4 x 11 bits) and the sum
        k[i] = __fadd_rn(__fmul_rn((float)((kc >> (4 * i)) & 15u), ks), km);
        v[i] = __fadd_rn(__fmul_rn((float)((vc >> (4 * i)) & 15u), vs), vm);
      }
    }
    const int64_t at = row * D + grp * 32 + 4 * j;
    store4(ko + at, k);
    store4(vo + at, v);
  }
  pdl_launch_dependents();
}

template <typename... P, typename... A>
void launch_rows(void (*kern)(P...), int64_t n_rows, int D, cudaStream_t stream, A... args) {
  const int64_t per_block = 8 * (D == 64 ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((n_rows + per_block - 1) / per_block));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FAK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
}

}  // namespace

void kv4_append_launch(const Kv4Rows& r, const int* slot, int T, int Hkv, int D, uint8_t* pages, int64_t n_pages,
                       int* err, cudaStream_t stream) {
  const int64_t n = (int64_t)T * Hkv;
  if (n == 0) return;
  auto go = [&](auto tag) {
    using E = decltype(tag);
    if (D == 128) launch_rows(k_kv4_append<E, 128>, n, D, stream, r, slot, n, Hkv, pages, n_pages, err);
    else launch_rows(k_kv4_append<E, 64>, n, D, stream, r, slot, n, Hkv, pages, n_pages, err);
  };
  if (r.type == Elt::F32) go(float());
  else if (r.type == Elt::F16) go(__half());
  else go(__nv_bfloat16());
}

void kv4_read_launch(const uint8_t* pages, int64_t n_pages, const int* slot, int T, int Hkv, int D, void* k, void* v,
                     Elt type, int* err, cudaStream_t stream) {
  const int64_t n = (int64_t)T * Hkv;
  if (n == 0) return;
  auto go = [&](auto tag) {
    using E = decltype(tag);
    if (D == 128) launch_rows(k_kv4_read<E, 128>, n, D, stream, pages, n_pages, slot, n, Hkv, (E*)k, (E*)v, err);
    else launch_rows(k_kv4_read<E, 64>, n, D, stream, pages, n_pages, slot, n, Hkv, (E*)k, (E*)v, err);
  };
  if (type == Elt::F32) go(float());
  else if (type == Elt::F16) go(__half());
  else go(__nv_bfloat16());
}

}  // namespace fak
