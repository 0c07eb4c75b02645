// Append into and read from the 4-bit KV cache (layout in kv4.cuh).
//
// Quantization of a group x[32], after clamping to +-65504:  m = f16(min x),  s = f16((max x - m) / 15), one
// f16 step less where m + 15 s would pass f16's range (its readers round values to f16),
// code = rint((x - m) / s) clamped to [0, 15], all codes 0 where s = 0 (a constant group).  f16 holds the
// minimum to 11 bits, more than the bf16 values that come in; the subtraction and the division are done
// in f32.  A group that holds a not-a-number stores m = NaN and reads back as NaN.
//
// Four lanes hold one group, eight consecutive dims each: two rows a warp at head dim 128, four at 64, K
// and V of a row in the same lanes.  The bytes (2 D each of K and V per row in, 20 D / 16 out) are few, so
// instructions decide: the extremes of 16-bit types are taken two values at a time, of K and V in one word
// across lanes; half of a group's lanes work out the scale of K, half that of V; quotients are q = d r
// corrected by one remainder step with r = 1 / s correctly rounded (Markstein 1990: the result is the
// correctly rounded quotient), two at a time; the four codes of a half word are summed as floats (c0 + 16 c1
// + 256 c2 + 4096 c3 is exact); heads are a grid dimension.
// Measured at 8191 tokens x 8 heads of 128, bf16: append 15.5 us (44 MB, 2.8 TB/s; bound by instructions; 18.5
// with every lane on both scales and one quotient at a time), read 9.6 us (4.6 TB/s).
#include "kv4.cuh"

#include <cuda_fp16.h>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../serve_ops.h"

namespace fak {
namespace {

constexpr int THREADS = 256;
static_assert(sizeof(uint4) == kKv4LoadBytes && sizeof(float4) == kKv4LoadBytes, "the vector loads of Rows8");

FAK_DEV float min_nan(float a, float b) {   // as fminf, but a NaN stays
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
FAK_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T, bool MAX>
FAK_DEV uint32_t pick2(uint32_t a, uint32_t b) {   // the same for pairs of 16-bit values
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>) {
    if constexpr (MAX) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    if constexpr (MAX) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}
template <typename T>
FAK_DEV float half_of(uint32_t u, int i) {
  const uint16_t h = (uint16_t)(i ? u >> 16 : u);
  if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half(h));
  else return __uint_as_float((uint32_t)h << 16);
}

// A lane's eight dims of K and of V: as floats, and 16-bit types also as they are.
template <typename T>
struct Rows8 {
  float k[8] = {}, v[8] = {};
  uint32_t kp[4] = {}, vp[4] = {};
  FAK_DEV static void load(const T* p, bool vec, float (&x)[8], uint32_t (&w)[4]) {
    if constexpr (sizeof(T) == 4) {
      if (vec) {
        const float4 f = *reinterpret_cast<const float4*>(p), h = *reinterpret_cast<const float4*>(p + 4);
        x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
        x[4] = h.x; x[5] = h.y; x[6] = h.z; x[7] = h.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
      }
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
      if (vec) {
        const uint4 q = *reinterpret_cast<const uint4*>(u);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = half_of<T>(w[i >> 1], i & 1);
    }
  }
  // smallest and largest of the group (four lanes), of K for mine = 0, of V for 1
  FAK_DEV void range(int mine, float& lo, float& hi) const {
    if constexpr (sizeof(T) == 4) {
      float l[2] = {k[0], v[0]}, h[2] = {k[0], v[0]};
#pragma unroll
      for (int i = 1; i < 8; i++) {
        l[0] = min_nan(l[0], k[i]);
        h[0] = max_nan(h[0], k[i]);
        l[1] = min_nan(l[1], v[i]);
        h[1] = max_nan(h[1], v[i]);
      }
#pragma unroll
      for (int o = 2; o > 0; o >>= 1)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          l[e] = min_nan(l[e], __shfl_xor_sync(0xffffffffu, l[e], o));
          h[e] = max_nan(h[e], __shfl_xor_sync(0xffffffffu, h[e], o));
        }
      lo = mine ? l[1] : l[0];
      hi = mine ? h[1] : h[0];
    } else {
      auto both = [](const uint32_t (&a)[4], const uint32_t (&b)[4], auto pick) {   // {K, V} in one word
        const uint32_t x = pick(pick(a[0], a[1]), pick(a[2], a[3])), y = pick(pick(b[0], b[1]), pick(b[2], b[3]));
        uint32_t r = pick(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
        r = pick(r, __shfl_xor_sync(0xffffffffu, r, 2));
        return pick(r, __shfl_xor_sync(0xffffffffu, r, 1));
      };
      lo = half_of<T>(both(kp, vp, pick2<T, false>), mine);
      hi = half_of<T>(both(kp, vp, pick2<T, true>), mine);
    }
  }
};

struct Scale {
  __half2 sm;   // scale, minimum
  float r;      // 1 / scale, 0 for a constant group
  bool plain;   // no clamp can act
};
// Ordinary groups: all values are within +-65504, the rounding of the minimum moves no quotient below -1/2
// (s > 2^-10 |m|) nor that of a normal scale one above 15 1/2.
FAK_DEV Scale scale_of(float lo, float hi) {
  constexpr float LIM = 65504.f;
  const bool nan = hi != hi;
  lo = fminf(fmaxf(lo, -LIM), LIM);
  hi = fminf(fmaxf(hi, -LIM), LIM);
  __half hm = __float2half_rn(lo);
  const float m = __half2float(hm), d = hi - m, r15 = 1.f / 15.f;
  const float q = d * r15;   // (below f32's normal range the corrected quotient may be off: f16 has 0 there)
  __half hs = __float2half_rn(fmaf(fmaf(-q, 15.f, d), r15, q));
  // code 15 of the largest values may round past f16's range, where the readers compute in f16
  if (m + 15.f * __half2float(hs) > LIM) hs = __ushort_as_half(__half_as_ushort(hs) - 1);
  const float s = __half2float(hs);
  Scale g;
  g.r = s > 0.f && !nan ? __frcp_rn(s) : 0.f;
  g.plain = s > fabsf(m) * 0.0009765625f && s >= 6.103515625e-5f && lo > -LIM && hi < LIM && !nan;
  if (nan) {
    hm = __ushort_as_half(0x7fff);
    hs = __ushort_as_half(0);
  }
  g.sm = __halves2half2(hs, hm);
  return g;
}

// two f32 at a time
FAK_DEV uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
FAK_DEV void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
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
FAK_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct Codes {
  uint32_t lo, hi;   // of the lane's dims 0-3 and 4-7, 16 bits each
};
FAK_DEV Codes codes_of(float (&x)[8], __half2 sm, float r, bool plain) {
  constexpr float LIM = 65504.f, MAGIC = 12582912.f;   // adding 1.5 * 2^23 rounds to whole numbers, ties to even
  const float s = __low2float(sm), m = __high2float(sm);
  float c[2] = {0.f, 0.f};
  if (plain) {
    const uint64_t r2 = pair(r, r), s2 = pair(-s, -s), m2 = pair(-m, -m), up = pair(MAGIC, MAGIC), down = pair(-MAGIC, -MAGIC);
    uint64_t c2 = 0;
#pragma unroll
    for (int i = 3; i >= 0; i--) {
      const uint64_t d = add2(pair(x[i], x[i + 4]), m2);
      uint64_t q = mul2(d, r2);
      q = add2(add2(fma2(fma2(q, s2, d), r2, q), up), down);
      c2 = fma2(c2, pair(16.f, 16.f), q);
    }
    unpair(c2, c[0], c[1]);
  } else {
#pragma unroll 1
    for (int i = 7; i >= 0; i--) {
      const float d = fminf(fmaxf(x[7], -LIM), LIM) - m;   // (rotated below: no indexed registers)
      float q = d * r;
      q = fmaf(fmaf(-q, s, d), r, q);
      q = (fminf(fmaxf(q, 0.f), 15.f) + MAGIC) - MAGIC;   // (0 in a group with a NaN)
      if (i >= 4) c[1] = fmaf(c[1], 16.f, q);
      else c[0] = fmaf(c[0], 16.f, q);
#pragma unroll
      for (int e = 7; e > 0; e--) x[e] = x[e - 1];
    }
  }
  return {(uint32_t)__float_as_int(c[0] + 8388608.f) & 0xffffu, (uint32_t)__float_as_int(c[1] + 8388608.f) & 0xffffu};
}

// The row (token, head) of a lane: heads along the grid's x, tokens along its y.
template <int D>
struct RowOf {
  static constexpr int LANES = D / 8, PER_CTA = THREADS / LANES;
  int64_t tok;
  int h, grp, j;   // head, group, the lane's eighth dims 8 j of the group
  FAK_DEV RowOf() {
    const int l = threadIdx.x % LANES;
    grp = l >> 2;
    j = l & 3;
    tok = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * PER_CTA + threadIdx.x / LANES;
    h = blockIdx.x;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(THREADS)
k_kv4_append(const __grid_constant__ Kv4Rows r, const int* __restrict__ slot, int n_tok, int Hkv, uint8_t* __restrict__ pages,
             int64_t n_pages, int* __restrict__ err) {
  using L = kv4::Lay<D>;
  pdl_wait();
  const RowOf<D> w;
  const int sl = w.tok < n_tok ? slot[w.tok] : -1;
  const bool in = sl >= 0 && (sl >> 4) < n_pages;
  if (sl >= 0 && !in) report_error(err, 2);
  Rows8<T> x;
  if (in) {
    const int d = w.grp * 32 + 8 * w.j;
    const int64_t pg = w.tok >> 4, row = w.tok & 15;
    x.load((const T*)r.k + pg * r.ks_page + row * r.ks_row + w.h * r.ks_head + d, r.vec, x.k, x.kp);
    x.load((const T*)r.v + pg * r.vs_page + row * r.vs_row + w.h * r.vs_head + d, r.vec, x.v, x.vp);
  }
  // lanes 0 and 1 of a group work out the scale of K, 2 and 3 that of V
  const bool of_v = w.j & 2;
  float lo, hi;
  x.range(of_v, lo, hi);
  const Scale mine = scale_of(lo, hi);
  const uint32_t sm = *reinterpret_cast<const uint32_t*>(&mine.sm), osm = __shfl_xor_sync(0xffffffffu, sm, 2);
  const float orr = __shfl_xor_sync(0xffffffffu, mine.r, 2);
  const uint32_t smk = of_v ? osm : sm, smv = of_v ? sm : osm;
  const bool plain = __all_sync(0xffffffffu, mine.plain);
  const Codes gk = codes_of(x.k, *reinterpret_cast<const __half2*>(&smk), of_v ? orr : mine.r, plain);
  const Codes gv = codes_of(x.v, *reinterpret_cast<const __half2*>(&smv), of_v ? mine.r : orr, plain);
  if (in) {
    uint8_t* pg = pages + ((int64_t)(sl >> 4) * Hkv + w.h) * L::BYTES;
    const int t = sl & 15;
    *reinterpret_cast<uint32_t*>(pg + L::k_u16(t, w.grp, 2 * w.j)) = gk.lo | gk.hi << 16;
    *reinterpret_cast<uint16_t*>(pg + L::v_u16(t, w.grp, 2 * w.j)) = (uint16_t)gv.lo;
    *reinterpret_cast<uint16_t*>(pg + L::v_u16(t, w.grp, 2 * w.j + 1)) = (uint16_t)gv.hi;
    // lane j of the group stores one of its four halves
    const int at = w.j < 2 ? L::KS + 32 * L::NG * w.j + L::k_meta(t, w.grp) : L::VS + 32 * L::NG * (w.j - 2) + L::v_meta(t, w.grp);
    *reinterpret_cast<uint16_t*>(pg + at) = (uint16_t)(w.j & 1 ? sm >> 16 : sm);
  }
  pdl_launch_dependents();
}

template <typename T>
FAK_DEV void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (T)x[i];
    uint4 u;
    memcpy(&u, h, 16);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS)
k_kv4_read(const uint8_t* __restrict__ pages, int64_t n_pages, const int* __restrict__ slot, int n_tok, int Hkv,
           T* __restrict__ ko, T* __restrict__ vo, int* __restrict__ err) {
  using L = kv4::Lay<D>;
  pdl_wait();
  const RowOf<D> w;
  if (w.tok < n_tok) {
    const int sl = slot[w.tok];
    const bool in = sl >= 0 && (sl >> 4) < n_pages;
    if (sl >= 0 && !in) report_error(err, 2);
    float k[8] = {}, v[8] = {};
    if (in) {
      const uint8_t* pg = pages + ((int64_t)(sl >> 4) * Hkv + w.h) * L::BYTES;
      const int t = sl & 15;
      const uint32_t kc = *reinterpret_cast<const uint32_t*>(pg + L::k_u16(t, w.grp, 2 * w.j));
      const uint32_t vc = *reinterpret_cast<const uint16_t*>(pg + L::v_u16(t, w.grp, 2 * w.j)) |
                          (uint32_t)*reinterpret_cast<const uint16_t*>(pg + L::v_u16(t, w.grp, 2 * w.j + 1)) << 16;
      auto h16 = [&](int at) { return __half2float(*reinterpret_cast<const __half*>(pg + at)); };
      const float ks = h16(L::KS + L::k_meta(t, w.grp)), km = h16(L::KM + L::k_meta(t, w.grp));
      const float vs = h16(L::VS + L::v_meta(t, w.grp)), vm = h16(L::VM + L::v_meta(t, w.grp));
      const uint64_t down = pair(-8388608.f, -8388608.f), ks2 = pair(ks, ks), km2 = pair(km, km), vs2 = pair(vs, vs), vm2 = pair(vm, vm);
      auto code = [](uint32_t c, int i) { return __int_as_float(0x4b000000 | (c >> (4 * i) & 15u)); };   // + 2^23, from its bits
#pragma unroll
      for (int i = 0; i < 8; i += 2) {   // (the product, 15 bits, is exact in the fma)
        unpair(fma2(add2(pair(code(kc, i), code(kc, i + 1)), down), ks2, km2), k[i], k[i + 1]);
        unpair(fma2(add2(pair(code(vc, i), code(vc, i + 1)), down), vs2, vm2), v[i], v[i + 1]);
      }
    }
    const int64_t at = (w.tok * Hkv + w.h) * D + w.grp * 32 + 8 * w.j;
    store8(ko + at, k);
    store8(vo + at, v);
  }
  pdl_launch_dependents();
}

template <typename... P, typename... A>
void launch_rows(void (*kern)(P...), int T, int Hkv, int D, cudaStream_t stream, A... args) {
  const int per_cta = THREADS / (D / 8);
  const int n = (int)(((int64_t)T + per_cta - 1) / per_cta), y = n < 32768 ? n : 32768;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)Hkv, (unsigned)y, (unsigned)((n + y - 1) / y));
  cfg.blockDim = dim3(THREADS);
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
  if (T == 0) return;
  auto go = [&](auto tag) {
    using E = decltype(tag);
    if (D == 128) launch_rows(k_kv4_append<E, 128>, T, Hkv, D, stream, r, slot, T, Hkv, pages, n_pages, err);
    else launch_rows(k_kv4_append<E, 64>, T, Hkv, D, stream, r, slot, T, Hkv, pages, n_pages, err);
  };
  if (r.type == Elt::F32) go(float());
  else if (r.type == Elt::F16) go(__half());
  else go(__nv_bfloat16());
}

void kv4_read_launch(const uint8_t* pages, int64_t n_pages, const int* slot, int T, int Hkv, int D, void* k, void* v,
                     Elt type, int* err, cudaStream_t stream) {
  if (T == 0) return;
  auto go = [&](auto tag) {
    using E = decltype(tag);
    if (D == 128) launch_rows(k_kv4_read<E, 128>, T, Hkv, D, stream, pages, n_pages, slot, T, Hkv, (E*)k, (E*)v, err);
    else launch_rows(k_kv4_read<E, 64>, T, Hkv, D, stream, pages, n_pages, slot, T, Hkv, (E*)k, (E*)v, err);
  };
  if (type == Elt::F32) go(float());
  else if (type == Elt::F16) go(__half());
  else go(__nv_bfloat16());
}

}  // namespace fak
