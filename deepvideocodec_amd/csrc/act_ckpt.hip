// 8-bit activation checkpoints of the training step: storing (quantise), restoring, and the element-wise adjoints that
// need nothing of an activation but its sign.  The format is described in include/dvc_hip.h.
//
// Arithmetic.  The scale of a block of 32 values is a power of two taken from the exponent and mantissa bits of the
// block's largest magnitude, so x / scale is exact and a code differs from its value only by the one rounding to 7 bits
// (int8) or 4 significant bits (e4m3).  int8: half a step, which is 1/254 to 1/127 of the block's maximum (the power of two
// costs up to one bit against a free scale; it buys exact bf16 operands in the weight gradient).  e4m3: 2^-4 of the value,
// or 2^-10 of the block's scale where that is more (values below 2^-6 scales, 2^-14 to 2^-15 of the maximum).
//
// All kernels are bound by HBM: 4 + 33/32 bytes per value to store or restore.  One lane handles a unit of 4 adjacent
// values (one 16-byte access), 8 lanes a block (maximum by three lane swaps), a workgroup 4 x 256 units (four
// requests in flight per lane).  A workgroup's first plane is found once; a lane adds its local offset to that.
// 32x64x256x256: store 138 us of 125 (at 5.4 TB/s), restore 119 of 125, signs 99 of 103; planes whose rows are no multiple of
// four take four dword accesses a lane: reading them costs nothing (store at 255x253 132 us), writing them doubles the time
// (restore 252, sign-only adjoints 331-436 of 199-318).
#include "dvc_common.h"

namespace {

struct Src { const float* p; long long bs, cs; int c; };
struct Dst { float* p; long long bs, cs; };
inline Src mk(const DvcSrc* s) { return Src{s->ptr, s->batch_stride, s->chan_stride, s->channels}; }
inline Dst mk(const DvcDst* d) { return Dst{d->ptr, d->batch_stride, d->chan_stride}; }

constexpr int UPB = 4;              // units per lane
constexpr int WG_UNITS = 256 * UPB;
// unit j of a thread inside its workgroup's: a wave's 4 x 64 units are adjacent, and so are the 32 scales of their blocks
__device__ __forceinline__ unsigned unit_of(int j) { return (threadIdx.x & ~63u) * UPB + 64 * j + (threadIdx.x & 63); }

// Where the units of this launch lie: `upp` units per plane (8 per block), `planes` planes.
struct Walk {
  long long units;
  unsigned upp;
  unsigned chans;
};

struct Unit { long long plane; unsigned n, c, u; };

__device__ __forceinline__ Unit locate(const Walk& k, long long base, unsigned local) {
  const long long p0 = base / k.upp;                     // uniform over the workgroup
  const unsigned r = (unsigned)(base - p0 * k.upp) + local;
  const unsigned dp = r / k.upp;
  Unit t;
  t.plane = p0 + dp;
  t.u = r - dp * k.upp;
  const unsigned pl = (unsigned)t.plane;                 // planes < 2^31 (checked on the host)
  t.n = pl / k.chans;
  t.c = pl - t.n * k.chans;
  return t;
}

__device__ __forceinline__ const float* plane_of(const Src& s, const Unit& t) {
  return s.p + (long long)t.n * s.bs + (long long)t.c * s.cs;
}
__device__ __forceinline__ float* plane_of(const Dst& d, const Unit& t) {
  return d.p + (long long)t.n * d.bs + (long long)t.c * d.cs;
}

// the values of a unit: zeros past the plane's end.  VEC: planes are multiples of 4 floats on 16-byte addresses
template <bool VEC>
__device__ __forceinline__ float4 load_unit(const float* plane, unsigned u, unsigned hw) {
  const unsigned p = 4 * u;
  if (VEC) return p < hw ? *reinterpret_cast<const float4*>(plane + p) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 v;
  v.x = p < hw ? plane[p] : 0.f;
  v.y = p + 1 < hw ? plane[p + 1] : 0.f;
  v.z = p + 2 < hw ? plane[p + 2] : 0.f;
  v.w = p + 3 < hw ? plane[p + 3] : 0.f;
  return v;
}
template <bool VEC>
__device__ __forceinline__ void store_unit(float* plane, unsigned u, unsigned hw, float4 v) {
  const unsigned p = 4 * u;
  if (VEC) {
    if (p < hw) *reinterpret_cast<float4*>(plane + p) = v;
    return;
  }
  if (p < hw) plane[p] = v.x;
  if (p + 1 < hw) plane[p + 1] = v.y;
  if (p + 2 < hw) plane[p + 2] = v.z;
  if (p + 3 < hw) plane[p + 3] = v.w;
}

// maximum over the 8 lanes of a block: swap neighbours, pairs, then the two halves (mirrored: all four lanes of a half
// hold the same by then)
__device__ __forceinline__ unsigned max8(unsigned v) {
  unsigned o = __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);    // quad_perm 1,0,3,2
  v = v > o ? v : o;
  o = __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);             // quad_perm 2,3,0,1
  v = v > o ? v : o;
  o = __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);            // row_half_mirror
  return v > o ? v : o;
}
__device__ __forceinline__ unsigned or8(unsigned v) {
  v |= (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);
  v |= (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);
  return v | (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);
}

template <int FMT>
__device__ __forceinline__ unsigned encode4(float4 v, unsigned amax, unsigned* scale) {
  // amax = 1.m 2^(f - 127): one binade more when 1.m is past the largest magnitude's own mantissa
  const unsigned f = amax >> 23, m = amax & 0x7fffffu;
  int s = FMT == DVC_CKPT_INT8 ? (int)f - 6 + (m > 0x7e0000u) : (int)f - 8 + (m > 0x600000u);
  s = s < 17 ? 17 : s;
  const bool poison = amax >= 0x7f800000u;
  const float inv = poison ? 0.f : __uint_as_float((unsigned)(254 - s) << 23);
  *scale = poison ? 255u : (unsigned)s;
  // the largest magnitude whose code does not restore to 2^128.  e4m3: 240 steps of the largest scale; in the next one down
  // nothing is that large.  int8: 63 steps of the largest scale, while all 127 of the next one down restore below 2^128.
  // (Everywhere else a bound that only infinities and NaN, whose codes are zeros, meet.)
  const float most = FMT != DVC_CKPT_INT8 ? 0x1.ep127f : s == 249 ? 0x1.f8p127f : 0x1.fffffep127f;
  const float a0 = fminf(fabsf(v.x), most) * inv, a1 = fminf(fabsf(v.y), most) * inv;
  const float a2 = fminf(fabsf(v.z), most) * inv, a3 = fminf(fabsf(v.w), most) * inv;
  unsigned mag;
  if (FMT == DVC_CKPT_INT8) {
    // adding 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits
    const unsigned b0 = __float_as_uint(a0 + 8388608.f), b1 = __float_as_uint(a1 + 8388608.f);
    const unsigned b2 = __float_as_uint(a2 + 8388608.f), b3 = __float_as_uint(a3 + 8388608.f);
    mag = (b0 & 0x7fu) | (b1 & 0x7fu) << 8 | (b2 & 0x7fu) << 16 | (b3 & 0x7fu) << 24;
  } else {
    int k = __builtin_amdgcn_cvt_pk_fp8_f32(a0, a1, 0, false);
    k = __builtin_amdgcn_cvt_pk_fp8_f32(a2, a3, k, true);
    mag = (unsigned)k & 0x7f7f7f7fu;
  }
  return mag | (v.x > 0.f ? 0u : 0x80u) | (v.y > 0.f ? 0u : 0x8000u) | (v.z > 0.f ? 0u : 0x800000u) |
         (v.w > 0.f ? 0u : 0x80000000u);
}

template <int FMT>
__device__ __forceinline__ float4 decode4(unsigned k, unsigned s) {
  const float sc = s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s << 23);
  float4 v;
  if (FMT == DVC_CKPT_INT8) {
    v.x = __uint_as_float(__float_as_uint((float)(k & 0x7fu) * sc) | (k & 0x80u) << 24);
    v.y = __uint_as_float(__float_as_uint((float)((k >> 8) & 0x7fu) * sc) | (k & 0x8000u) << 16);
    v.z = __uint_as_float(__float_as_uint((float)((k >> 16) & 0x7fu) * sc) | (k & 0x800000u) << 8);
    v.w = __uint_as_float(__float_as_uint((float)((k >> 24) & 0x7fu) * sc) | (k & 0x80000000u));
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)k, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)k, true);
    v = make_float4(lo[0] * sc, lo[1] * sc, hi[0] * sc, hi[1] * sc);
  }
  return v;
}

template <int FMT, bool VEC>
__global__ __launch_bounds__(256) void act_checkpoint_kernel(Src x, Walk k, unsigned hw, int act, float slope,
                                                             unsigned* codes, uint8_t* scales) {
  const long long base = (long long)blockIdx.x * WG_UNITS;
  float4 v[UPB];
  Unit t[UPB];
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned local = unit_of(j);
    t[j] = locate(k, base, local);
    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (base + local < k.units) v[j] = load_unit<VEC>(plane_of(x, t[j]), t[j].u, hw);
  }
  unsigned sj = 0;
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    float4 a = v[j];
    if (act) {
      a.x = dvc::leaky(a.x, slope); a.y = dvc::leaky(a.y, slope);
      a.z = dvc::leaky(a.z, slope); a.w = dvc::leaky(a.w, slope);
    }
    const unsigned b0 = __float_as_uint(a.x) & 0x7fffffffu, b1 = __float_as_uint(a.y) & 0x7fffffffu;
    const unsigned b2 = __float_as_uint(a.z) & 0x7fffffffu, b3 = __float_as_uint(a.w) & 0x7fffffffu;
    const unsigned m01 = b0 > b1 ? b0 : b1, m23 = b2 > b3 ? b2 : b3;
    const unsigned amax = max8(m01 > m23 ? m01 : m23);   // blocks never straddle the launch's end: units % 8 == 0
    unsigned s;
    const unsigned code = encode4<FMT>(a, amax, &s);
    const long long unit = base + unit_of(j);
    if (unit < k.units) codes[unit] = code;
    sj = (threadIdx.x & 7) == (unsigned)j ? s : sj;
  }
  // the wave's 32 scales in one store: lane 8 b + j that of the block b of its j-th 64 units
  const int j = threadIdx.x & 7;
  const long long unit = base + unit_of(j) - j;      // (first unit of that block)
  if (j < UPB && unit < k.units) scales[unit >> 3] = (uint8_t)sj;
}

template <int FMT, bool VEC>
__global__ __launch_bounds__(256) void act_restore_kernel(const unsigned* codes, const uint8_t* scales, Dst out, Walk k,
                                                          unsigned hw) {
  const long long base = (long long)blockIdx.x * WG_UNITS;
  unsigned code[UPB], s[UPB];
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const long long unit = base + unit_of(j);
    code[j] = s[j] = 0;
    if (unit < k.units) {
      code[j] = codes[unit];
      s[j] = scales[unit >> 3];
    }
  }
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned local = unit_of(j);
    if (base + local < k.units) {
      const Unit t = locate(k, base, local);
      store_unit<VEC>(plane_of(out, t), t.u, hw, decode4<FMT>(code[j], s[j]));
    }
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void act_signs_kernel(Src x, Walk k, unsigned hw, unsigned* signs) {
  const long long base = (long long)blockIdx.x * WG_UNITS;
  float4 v[UPB];
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned local = unit_of(j);
    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (base + local < k.units) {
      const Unit t = locate(k, base, local);
      v[j] = load_unit<VEC>(plane_of(x, t), t.u, hw);
    }
  }
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned nib = (v[j].x > 0.f ? 1u : 0u) | (v[j].y > 0.f ? 2u : 0u) | (v[j].z > 0.f ? 4u : 0u) | (v[j].w > 0.f ? 8u : 0u);
    const unsigned word = or8(nib << (4 * (threadIdx.x & 7)));
    const long long unit = base + unit_of(j);
    if (unit < k.units && (threadIdx.x & 7) == 0) signs[unit >> 3] = word;
  }
}

// grad * (bit ? 1 : slope), contiguous result
template <bool VEC>
__global__ __launch_bounds__(256) void act_grad_signs_kernel(Src g, const unsigned* signs, float slope, float* out, Walk k,
                                                             unsigned hw) {
  const long long base = (long long)blockIdx.x * WG_UNITS;
  float4 v[UPB];
  unsigned bits[UPB];
  Unit t[UPB];
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned local = unit_of(j);
    t[j] = locate(k, base, local);
    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    bits[j] = 0;
    if (base + local < k.units) {
      v[j] = load_unit<VEC>(plane_of(g, t[j]), t[j].u, hw);
      bits[j] = signs[(base + local) >> 3] >> (4 * (local & 7));
    }
  }
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    if (base + unit_of(j) < k.units) {
      float4 r = v[j];
      r.x = (bits[j] & 1u) ? r.x : r.x * slope; r.y = (bits[j] & 2u) ? r.y : r.y * slope;
      r.z = (bits[j] & 4u) ? r.z : r.z * slope; r.w = (bits[j] & 8u) ? r.w : r.w * slope;
      store_unit<VEC>(out + t[j].plane * hw, t[j].u, hw, r);
    }
  }
}

// The same behind PixelShuffle(2): gradient and signs are in the shuffled layout, the result is not.
__global__ __launch_bounds__(256) void act_grad_signs_shuffled_kernel(Src g, const unsigned* signs, float slope, float* out,
                                                                      int batch, int c, int ho, int wo, long long blocks) {
  const long long total = (long long)batch * c * ho * wo;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int ox = (int)(i % wo);
    long long q = i / wo;
    const int oy = (int)(q % ho); q /= ho;
    const int co = (int)(q % c), n = (int)(q / c);
    const long long pix = (long long)(2 * oy + ((co >> 1) & 1)) * (2 * wo) + 2 * ox + (co & 1);
    const long long plane = (long long)n * (c >> 2) + (co >> 2);
    const float v = g.p[n * g.bs + (co >> 2) * g.cs + pix];
    out[i] = (signs[plane * blocks + (pix >> 5)] >> (pix & 31)) & 1u ? v : v * slope;
  }
}

// grad * (code < 128 ? 1 : slope) (+ plus)
template <bool VEC>
__global__ __launch_bounds__(256) void mul_act_grad_ckpt_kernel(Src g, const unsigned* codes, Src plus, int has_plus, Dst out,
                                                                float slope, Walk k, unsigned hw) {
  const long long base = (long long)blockIdx.x * WG_UNITS;
  float4 v[UPB], e[UPB];
  unsigned code[UPB];
  Unit t[UPB];
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    const unsigned local = unit_of(j);
    t[j] = locate(k, base, local);
    v[j] = e[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    code[j] = 0;
    if (base + local < k.units) {
      v[j] = load_unit<VEC>(plane_of(g, t[j]), t[j].u, hw);
      if (has_plus) e[j] = load_unit<VEC>(plane_of(plus, t[j]), t[j].u, hw);
      code[j] = codes[base + local];
    }
  }
#pragma unroll
  for (int j = 0; j < UPB; ++j) {
    if (base + unit_of(j) < k.units) {
      float4 r = v[j];
      r.x = (code[j] & 0x80u) ? r.x * slope : r.x; r.y = (code[j] & 0x8000u) ? r.y * slope : r.y;
      r.z = (code[j] & 0x800000u) ? r.z * slope : r.z; r.w = (code[j] & 0x80000000u) ? r.w * slope : r.w;
      if (has_plus) { r.x += e[j].x; r.y += e[j].y; r.z += e[j].z; r.w += e[j].w; }
      store_unit<VEC>(plane_of(out, t[j]), t[j].u, hw, r);
    }
  }
}

// ------------------------------------------------------------------ host side
inline bool al16(const void* p, long long bs, long long cs) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bs % 4 == 0 && cs % 4 == 0;
}
inline bool al16(const DvcSrc* s) { return s == nullptr || al16(s->ptr, s->batch_stride, s->chan_stride); }
inline bool al16(const DvcDst* d) { return al16(d->ptr, d->batch_stride, d->chan_stride); }

int make_walk(int batch, int channels, int h, int w, Walk* k, unsigned* hw, const char* who) {
  DVC_REQUIRE(batch >= 1 && channels >= 1 && h >= 1 && w >= 1, "%s: bad dims (%d, %d, %d, %d)", who, batch, channels, h, w);
  DVC_REQUIRE((long long)h * w < (1LL << 28), "%s: plane too large", who);
  DVC_REQUIRE((long long)batch * channels < (1LL << 31), "%s: too many planes", who);
  *hw = (unsigned)((long long)h * w);
  k->upp = (*hw + 31) / 32 * 8;
  k->chans = (unsigned)channels;
  k->units = (long long)batch * channels * k->upp;
  DVC_REQUIRE((k->units + WG_UNITS - 1) / WG_UNITS < (1LL << 31), "%s: tensor too large", who);
  return DVC_OK;
}
inline dim3 walk_grid(const Walk& k) { return dim3((unsigned)((k.units + WG_UNITS - 1) / WG_UNITS)); }

int check_src(const DvcSrc* s, long long plane, const char* who) {
  DVC_REQUIRE(s != nullptr && s->ptr != nullptr && s->channels >= 1, "%s: null/empty source", who);
  DVC_REQUIRE(s->chan_stride >= plane, "%s: channel stride < H*W", who);
  return DVC_OK;
}
#define CHECK(expr) do { int rc_ = (expr); if (rc_) return rc_; } while (0)

int check_ckpt(const DvcCkpt* c, const char* who) {
  DVC_REQUIRE(c != nullptr && c->codes != nullptr && c->scales != nullptr && c->channels >= 1, "%s: null/empty checkpoint", who);
  DVC_REQUIRE(c->format == DVC_CKPT_INT8 || c->format == DVC_CKPT_E4M3, "%s: format %d unknown", who, c->format);
  DVC_REQUIRE(reinterpret_cast<uintptr_t>(c->codes) % 16 == 0, "%s: codes must start on 16 bytes", who);
  return DVC_OK;
}

}  // namespace

#define LAUNCH_VEC(kernel, vec, ...)                                                                             \
  do {                                                                                                           \
    if (vec) hipLaunchKernelGGL((kernel<true>), walk_grid(k), dim3(256), 0, static_cast<hipStream_t>(stream), __VA_ARGS__);  \
    else hipLaunchKernelGGL((kernel<false>), walk_grid(k), dim3(256), 0, static_cast<hipStream_t>(stream), __VA_ARGS__);     \
  } while (0)

namespace {
template <bool VEC> constexpr auto ckpt_i8 = act_checkpoint_kernel<DVC_CKPT_INT8, VEC>;
template <bool VEC> constexpr auto ckpt_f8 = act_checkpoint_kernel<DVC_CKPT_E4M3, VEC>;
template <bool VEC> constexpr auto restore_i8 = act_restore_kernel<DVC_CKPT_INT8, VEC>;
template <bool VEC> constexpr auto restore_f8 = act_restore_kernel<DVC_CKPT_E4M3, VEC>;
}  // namespace

extern "C" int dvc_act_checkpoint(const DvcSrc* x, int32_t act, float slope, int32_t format, uint8_t* codes,
                                  uint8_t* scales, int32_t batch, int32_t h, int32_t w, void* stream) {
  CHECK(check_src(x, (long long)h * w, "dvc_act_checkpoint"));
  DVC_REQUIRE(codes != nullptr && scales != nullptr, "dvc_act_checkpoint: null pointer");
  DVC_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "dvc_act_checkpoint: codes must start on 16 bytes");
  DVC_REQUIRE(format == DVC_CKPT_INT8 || format == DVC_CKPT_E4M3, "dvc_act_checkpoint: format %d unknown", format);
  DVC_REQUIRE(!act || (slope >= 0.f && slope <= 1.f), "dvc_act_checkpoint: slope %g outside [0, 1]", (double)slope);
  Walk k;
  unsigned hw;
  CHECK(make_walk(batch, x->channels, h, w, &k, &hw, "dvc_act_checkpoint"));
  const bool vec = al16(x) && hw % 4 == 0;
  if (format == DVC_CKPT_INT8) LAUNCH_VEC(ckpt_i8, vec, mk(x), k, hw, act, slope, reinterpret_cast<unsigned*>(codes), scales);
  else LAUNCH_VEC(ckpt_f8, vec, mk(x), k, hw, act, slope, reinterpret_cast<unsigned*>(codes), scales);
  return dvc::check_launch("act_checkpoint_kernel");
}

extern "C" int dvc_act_restore(const DvcCkpt* ckpt, const DvcDst* out, int32_t batch, int32_t h, int32_t w, void* stream) {
  CHECK(check_ckpt(ckpt, "dvc_act_restore"));
  DVC_REQUIRE(out != nullptr && out->ptr != nullptr && out->chan_stride >= (int64_t)h * w, "dvc_act_restore: bad destination");
  Walk k;
  unsigned hw;
  CHECK(make_walk(batch, ckpt->channels, h, w, &k, &hw, "dvc_act_restore"));
  const bool vec = al16(out) && hw % 4 == 0;
  const unsigned* codes = reinterpret_cast<const unsigned*>(ckpt->codes);
  if (ckpt->format == DVC_CKPT_INT8) LAUNCH_VEC(restore_i8, vec, codes, ckpt->scales, mk(out), k, hw);
  else LAUNCH_VEC(restore_f8, vec, codes, ckpt->scales, mk(out), k, hw);
  return dvc::check_launch("act_restore_kernel");
}

extern "C" int dvc_act_signs(const DvcSrc* x, uint32_t* signs, int32_t batch, int32_t h, int32_t w, void* stream) {
  CHECK(check_src(x, (long long)h * w, "dvc_act_signs"));
  DVC_REQUIRE(signs != nullptr, "dvc_act_signs: null pointer");
  Walk k;
  unsigned hw;
  CHECK(make_walk(batch, x->channels, h, w, &k, &hw, "dvc_act_signs"));
  LAUNCH_VEC(act_signs_kernel, al16(x) && hw % 4 == 0, mk(x), k, hw, signs);
  return dvc::check_launch("act_signs_kernel");
}

extern "C" int dvc_act_grad_signs(const DvcSrc* grad, const uint32_t* signs, float slope, int32_t pixel_shuffle,
                                  float* grad_pre, int32_t batch, int32_t channels, int32_t ho, int32_t wo, void* stream) {
  const long long plane = (long long)ho * wo * (pixel_shuffle ? 4 : 1);
  CHECK(check_src(grad, plane, "dvc_act_grad_signs"));
  DVC_REQUIRE(signs != nullptr && grad_pre != nullptr, "dvc_act_grad_signs: null pointer");
  DVC_REQUIRE(!pixel_shuffle || channels % 4 == 0, "dvc_act_grad_signs: %d channels cannot be shuffled", channels);
  DVC_REQUIRE(grad->channels == (pixel_shuffle ? channels / 4 : channels), "dvc_act_grad_signs: grad has %d channels, %d expected",
              grad->channels, pixel_shuffle ? channels / 4 : channels);
  Walk k;
  unsigned hw;
  CHECK(make_walk(batch, channels, ho, wo, &k, &hw, "dvc_act_grad_signs"));
  if (pixel_shuffle) {
    DVC_REQUIRE(plane < (1LL << 28), "dvc_act_grad_signs: plane too large");
    hipLaunchKernelGGL(act_grad_signs_shuffled_kernel, dim3(dvc::stream_grid((long long)batch * channels * hw, 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), mk(grad), signs, slope, grad_pre, batch, channels, ho, wo, (plane + 31) / 32);
  } else {
    const bool vec = al16(grad) && hw % 4 == 0 && reinterpret_cast<uintptr_t>(grad_pre) % 16 == 0;
    LAUNCH_VEC(act_grad_signs_kernel, vec, mk(grad), signs, slope, grad_pre, k, hw);
  }
  return dvc::check_launch("act_grad_signs_kernel");
}

extern "C" int dvc_mul_act_grad_ckpt(const DvcSrc* grad, const DvcCkpt* x, float slope, const DvcSrc* plus, const DvcDst* out,
                                     int32_t batch, int32_t h, int32_t w, void* stream) {
  CHECK(check_src(grad, (long long)h * w, "dvc_mul_act_grad_ckpt"));
  CHECK(check_ckpt(x, "dvc_mul_act_grad_ckpt"));
  DVC_REQUIRE(x->channels == grad->channels, "dvc_mul_act_grad_ckpt: the checkpoint has %d channels, grad %d", x->channels, grad->channels);
  if (plus != nullptr) {
    CHECK(check_src(plus, (long long)h * w, "dvc_mul_act_grad_ckpt"));
    DVC_REQUIRE(plus->channels == grad->channels, "dvc_mul_act_grad_ckpt: plus has %d channels, grad %d", plus->channels, grad->channels);
  }
  DVC_REQUIRE(out != nullptr && out->ptr != nullptr && out->chan_stride >= (int64_t)h * w, "dvc_mul_act_grad_ckpt: bad destination");
  Walk k;
  unsigned hw;
  CHECK(make_walk(batch, grad->channels, h, w, &k, &hw, "dvc_mul_act_grad_ckpt"));
  const bool vec = al16(grad) && al16(plus) && al16(out) && hw % 4 == 0;
  const Src p = plus != nullptr ? mk(plus) : Src{nullptr, 0, 0, 0};
  LAUNCH_VEC(mul_act_grad_ckpt_kernel, vec, mk(grad), reinterpret_cast<const unsigned*>(x->codes), p, plus != nullptr ? 1 : 0, mk(out),
             slope, k, hw);
  return dvc::check_launch("mul_act_grad_ckpt_kernel");
}
