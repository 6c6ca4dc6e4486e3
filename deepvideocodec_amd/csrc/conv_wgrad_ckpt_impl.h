// Weight gradient of the 2-D convolutions from 8-bit activation checkpoints (include/dvc_hip.h): the kernels.
//
//   gW[co][ci][ky][kx] = sum over (n, oy, ox) of  g[n][co][oy][ox] * X[n][ci][oy*s + ky - p][ox*s + kx - p]
//
// Mathematics.  A checkpoint's value is (at most seven bits) * 2^e: exactly a bf16 number.  An fp32 gradient is exactly
// the sum of three bf16 numbers of eight bits each (cut off, subtract, cut off, subtract).  So gW is three bf16
// matrix products with exact products and fp32 sums -- the accuracy of the fp32 kernel at 2.5 PFLOP/s / 3 instead of 157
// TFLOP/s: it is the 8-bit storage that buys the rate.
//
// Shape.  [Cout x pixels] * [pixels x Cin taps], a small result and a very long reduction, on
// v_mfma_f32_32x32x16_bf16: rows = 32 output channels, columns = 32 input channels at one tap, k = 16 adjacent
// pixels of a row (a half-wave holds 8 of them: one 16-byte LDS read).  The taps of a row read the same 16-byte windows,
// shifted by whole elements in registers (v_alignbit): nine products of a 3x3 layer need three window reads.
// A workgroup (8 waves) owns (32 MT) x (32 CT) of the result for all taps.  Four waves (one per SIMD) multiply: a wave keeps a
// 32 x 32 corner for every tap in registers; the 4 / (MT CT) waves of one corner take the row pieces of a tile in turn.  The
// other four stage (7x7: wave ky < 7 multiplies tap row ky of a 32 x 32 block, and all eight stage).  With every wave doing
// both, staging and multiplying took turns: 457 us for 64->64 3x3 at 32x256x256, of 233 us staging alone and 275 us
// multiplying alone.  The pixel axis is cut into slabs -- over workgroups, over the waves of a corner and, so that
// no running sum gets too long for fp32, in time -- whose partial results a second kernel adds in a fixed order
// (deterministic, no atomics).
//
// Staging per tile of TH x TW output pixels, two LDS buffers and one barrier per tile: the codes, scales and gradients of the
// next tile (loaded a tile ago) are decoded to bf16 / stored as fp32 while a tile is multiplied, and the loads of the one
// after are issued.  A lane decodes four codes of a row (one dword).  The gradient stays fp32 in LDS (4 instead of 6
// bytes) and is split when it is read, in the shadow of the matrix instructions; the bias gradient is summed by the lanes that
// stage it.
#pragma once
#include <atomic>
#include <type_traits>

#include "dvc_common.h"

namespace dvc_wgrad_ckpt {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Args {
  const uint8_t* codes[DVC_MAX_SRC];
  const uint8_t* scales[DVC_MAX_SRC];
  int first[DVC_MAX_SRC];       // first channel of each source; sources that are not there start at cin
  int chans[DVC_MAX_SRC];
  int e4m3;
  int cin, h, w, blocks;        // blocks of 32 per plane
  int cout, ho, wo;
  const float* g;               // [N][cout][ho][wo], contiguous
  float* partial;               // [slabs][taps][cout_pad][cin_pad], slab = (segment * splits + split) * KG + wave of the corner
  float* bias_partial;          // [splits][cout_pad], or null
  int cout_pad, cin_pad, n_cib;
  int tiles_x, tiles_y;
  int tile0, n_tiles;           // this launch's tiles: from tile0 up to n_tiles
  int seg_tiles, segments;      // tiles of a workgroup per slab, slabs of a workgroup and wave (segments * seg_tiles tiles or fewer)
  int seg0;                     // slabs in time before this launch
};

__device__ __forceinline__ unsigned long long uniform64(unsigned long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return ((unsigned long long)hi << 32) | lo;
}

// Where input channel `ci` (uniform) of the concatenated checkpoints lives.
struct Plane {
  unsigned long long codes, scales;      // addresses of sample 0's plane
  unsigned step;                         // blocks between samples (< 2^31: checked on the host)
};
__device__ __forceinline__ Plane plane_of(const Args& a, int ci) {
  // (mask arithmetic instead of indexing by a run-time source number, which would become a private lookup table)
  const unsigned long long m1 = 0ull - (unsigned long long)(ci >= a.first[1]);
  const unsigned long long m2 = 0ull - (unsigned long long)(ci >= a.first[2]);
  const unsigned long long m3 = 0ull - (unsigned long long)(ci >= a.first[3]);
  auto pick = [&](unsigned long long v0, unsigned long long v1, unsigned long long v2, unsigned long long v3) {
    return v0 + ((v1 - v0) & m1) + ((v2 - v1) & m2) + ((v3 - v2) & m3);
  };
  const unsigned long long c = pick((unsigned long long)a.codes[0], (unsigned long long)a.codes[1], (unsigned long long)a.codes[2],
                                    (unsigned long long)a.codes[3]);
  const unsigned long long s = pick((unsigned long long)a.scales[0], (unsigned long long)a.scales[1],
                                    (unsigned long long)a.scales[2], (unsigned long long)a.scales[3]);
  const unsigned long long first = pick(a.first[0], a.first[1], a.first[2], a.first[3]);
  const unsigned long long chans = pick(a.chans[0], a.chans[1], a.chans[2], a.chans[3]);
  const bool have = ci < a.cin;         // (channels past the last: any plane; their loads are switched off)
  const unsigned long long at = have ? ((unsigned long long)ci - first) * (unsigned)a.blocks : 0ull;
  Plane p;
  p.codes = uniform64((have ? c : (unsigned long long)a.codes[0]) + 32ull * at);
  p.scales = uniform64((have ? s : (unsigned long long)a.scales[0]) + at);
  p.step = __builtin_amdgcn_readfirstlane(have ? (unsigned)(chans * (unsigned)a.blocks) : 0u);
  return p;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(unsigned long long at, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(at), 0, bytes, 0x00020000);
}

struct __attribute__((packed)) Dword { unsigned v; };      // a dword at any byte address

__device__ __forceinline__ float scale_of(unsigned s, unsigned flip) { return __uint_as_float((s == 255u ? 0x7fc00000u : s << 23) ^ flip); }

// four codes -> two dwords of bf16 (exact); s01 / s23 ... one scale per code
template <bool E4M3>
__device__ __forceinline__ uint2 decode(unsigned k, float s0, float s1, float s2, float s3) {
  uint2 r;
  if constexpr (E4M3) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)k, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)k, true);
    r.x = __builtin_amdgcn_perm(__float_as_uint(lo[1] * s1), __float_as_uint(lo[0] * s0), 0x07060302u);
    r.y = __builtin_amdgcn_perm(__float_as_uint(hi[1] * s3), __float_as_uint(hi[0] * s2), 0x07060302u);
  } else {
    const unsigned m = k & 0x7f7f7f7fu, sg = k & 0x80808080u;
    const float f0 = (float)(m & 0xffu) * s0, f1 = (float)((m >> 8) & 0xffu) * s1;
    const float f2 = (float)((m >> 16) & 0xffu) * s2, f3 = (float)(m >> 24) * s3;
    r.x = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u) ^ __builtin_amdgcn_perm(0u, sg, 0x010c000cu);
    r.y = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u) ^ __builtin_amdgcn_perm(0u, sg, 0x030c020cu);
  }
  return r;
}

// eight gradients -> three fragments of bf16 that add up to them
struct Split { bf16x8 a1, a2, a3; };
__device__ __forceinline__ Split split(const float4 lo, const float4 hi) {
  const float g[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  u32x4 p1, p2, p3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned b1[2], b2[2], b3[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = g[2 * i + j];
      b1[j] = __float_as_uint(v);
      const float r = v - __uint_as_float(b1[j] & 0xffff0000u);
      b2[j] = __float_as_uint(r);
      b3[j] = __float_as_uint(r - __uint_as_float(b2[j] & 0xffff0000u));
    }
    p1[i] = __builtin_amdgcn_perm(b1[1], b1[0], 0x07060302u);
    p2[i] = __builtin_amdgcn_perm(b2[1], b2[0], 0x07060302u);
    p3[i] = __builtin_amdgcn_perm(b3[1], b3[0], 0x07060302u);
  }
  return Split{__builtin_bit_cast(bf16x8, p1), __builtin_bit_cast(bf16x8, p2), __builtin_bit_cast(bf16x8, p3)};
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// eight elements from element `e` on of the dwords d[] (two elements each)
template <int E, int D>
__device__ __forceinline__ bf16x8 window(const unsigned (&d)[D]) {
  static_assert(E / 2 + (E % 2 ? 5 : 4) <= D, "window past the dwords read");
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = E % 2 ? __builtin_amdgcn_alignbit(d[E / 2 + i + 1], d[E / 2 + i], 16) : d[E / 2 + i];
  return __builtin_bit_cast(bf16x8, r);
}

// Geometry.  KS x KS taps, stride S, tiles of TH x TW output pixels; a staged input row is XD dwords of codes from column
// gx0 = ox0 * S - LEFT on (a multiple of 4), kept in LDS as XROW bf16: as it is (stride 1), or its even columns, then
// (3x3) its odd ones, so that the eight pixels of a half-wave are adjacent at stride 2 as well.
template <int KS_, int S_, int MT, int CT, int TW_>
struct Geo {
  static constexpr int KS = KS_, S = S_;
  static constexpr int NM = KS == 7 ? 7 : 4, NS = KS == 7 ? 8 : 4;      // multiplying and staging waves
  static constexpr int KG = KS == 7 ? 1 : NM / (MT * CT);        // waves sharing one corner (7x7: one tap row per wave)
  static constexpr int XCH = 32 * CT, GCH = 32 * MT;
  static constexpr int TAPS = KS * KS, ACC = KS == 7 ? 7 : TAPS; // accumulator tiles per wave
  static_assert(KS != 7 || (S == 1 && MT == 1 && CT == 1), "7x7: 32 x 32 blocks, stride 1");
  static constexpr int TW = TW_, TH = (KS == 3 && S == 2 ? 2 : 4) * (32 / TW_), PAD = KS / 2;
  static constexpr int LEFT = KS == 1 ? 0 : 4;
  static constexpr int YS = KS == 1 ? S : 1;                     // input rows between staged rows
  static constexpr int IH = KS == 1 ? TH : (TH - 1) * S + KS;
  static constexpr int XD = (TW * S + (KS == 1 ? 0 : 8)) / 4;    // dwords (4 codes) per staged row
  static constexpr int ODD = TW + 8;                             // odd columns of a stride-2 row
  static constexpr int XROW = S == 1 ? 4 * XD : KS == 1 ? TW : TW + ODD;
  static_assert(XROW % 8 == 0, "rows on 16 bytes");
  // bytes per channel: an odd multiple of what a lane reads at once (8 bytes for 3x3 stride 1, else 16), so that the lanes
  // of a read -- channels -- fall on different banks
  static constexpr int XREAD = KS == 3 && S == 1 ? 8 : 16, XSTR = ((IH * XROW * 2 / XREAD) | 1) * XREAD;
  static constexpr int GUNITS = (TH * TW / 4) | 1;
  static constexpr int XE = IH * XD, XSLOTS = (XE + 63) / 64;
  static constexpr int XPW = XCH / NS;                           // channels of x per staging wave
  static constexpr int GE = TH * TW / 4, GLOADS = GCH * GE / (64 * NS);      // 16-byte units of g per channel, per staging lane
  static_assert(GCH * GE % (64 * NS) == 0 && 64 % GE == 0, "gradient units deal out evenly, a channel's on adjacent lanes");
  static constexpr int XBYTES = XCH * XSTR, BUF = XBYTES + GCH * GUNITS * 16;
  static constexpr int LDS_BYTES = 2 * BUF;
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
  static constexpr int STEPS = TH * TW / 16;                     // row pieces of 16 pixels per tile
  static_assert(STEPS % KG == 0, "row pieces deal out evenly");
};

// The staging side of a kernel: NS waves deal out the channels of x and the 16-byte units of g of a tile.
// AL: rows of codes start on dwords and rows of gradients on 16 bytes (w % 4 == 0, wo % 4 == 0).
template <class G, bool AL>
struct Stager {
  static constexpr int KS = G::KS, S = G::S, TW = G::TW, XPW = G::XPW, XSLOTS = G::XSLOTS, GLOADS = G::GLOADS;
  const Args& a;
  const int lane, sw, stid;
  unsigned flip;                // changes sign with every slab
  int left;                     // tiles of the slab that are still to be stored
  int per_n, xlive;             // tiles per sample, this wave's channels that exist
  bool together;                // this wave's channels all exist and lie in one source: adjacent planes
  unsigned plane_bytes, gplane;
  Plane xp[XPW];
  // Gradients.  AL: 16-byte units, unit u = stid + 64 NS i is unit u % GE of channel u / GE: a load is CPL whole channels.  Else
  // dwords, so that a load reads whole row pieces wherever they start (16-byte units in four dwords each met four times the
  // cache lines: 64->64 3x3 at 32x255x253 540 us, now 471): a load is 64 pixels of one of this wave's GPW channels, LPC loads a channel.  Either way what
  // differs from load to load is uniform, in the descriptor, and the lanes' offsets are found once a tile.
  static constexpr int CPL = 64 / G::GE, GPW = G::GCH / G::NS, LPC = AL ? 1 : G::TH * TW / 64;
  static constexpr int GREGS = AL ? GLOADS : GPW * LPC, GSUMS = AL ? GLOADS : GPW;
  static_assert(AL || (G::TH * TW % 64 == 0 && 64 % TW == 0), "a channel's pixels are whole loads of whole rows");
  typedef typename std::conditional<AL, float4, float>::type GReg;
  int co0;
  float gsum[GSUMS], gbefore[GSUMS];      // the bias gradient's sums since the last slab's end and until then
  unsigned xk[XPW][XSLOTS], xs[XPW][XSLOTS], xs2[AL ? 1 : XPW][AL ? 1 : XSLOTS];
  int mask[XSLOTS];             // codes of a dword inside the row (not AL; none: it lies outside the plane)
  int cut[XSLOTS];              // codes of a dword before a block's end (not AL)
  unsigned shift[XSLOTS];       // bits by which a dword was read early (not AL)
  GReg gr[GREGS];

  __device__ __forceinline__ Stager(const Args& args, int lane_, int sw_, int co0_, int ci0, unsigned flip_)
      : a(args), lane(lane_), sw(sw_), stid(64 * sw_ + lane_), flip(flip_), left(args.seg_tiles), co0(co0_) {
    per_n = a.tiles_x * a.tiles_y;
    plane_bytes = 32u * (unsigned)a.blocks;
    gplane = (unsigned)(a.ho * a.wo);
    xlive = a.cin - (ci0 + XPW * sw);
    // (finding a channel's plane is some 80 scalar instructions: 16 times that was a fifth of a one-tile workgroup's time)
    const int c0 = ci0 + XPW * sw, c1 = c0 + XPW;
    together = c1 <= a.cin && (unsigned long long)XPW * plane_bytes < (1ull << 31);
#pragma unroll
    for (int k = 1; k < DVC_MAX_SRC; ++k) together = together && !(c0 < a.first[k] && a.first[k] < c1);
    xp[0] = plane_of(a, c0);
    if (!together) {
#pragma unroll
      for (int c = 1; c < XPW; ++c) xp[c] = plane_of(a, c0 + c);
    } else {
#pragma unroll
      for (int c = 1; c < XPW; ++c) xp[c] = xp[0];
    }
#pragma unroll
    for (int i = 0; i < GSUMS; ++i) gsum[i] = gbefore[i] = 0.f;
  }

  // request tile t (past the last: zeros)
  __device__ __forceinline__ void load(int t) {
    const bool there = t < a.n_tiles;
    const int tt = there ? t : 0;
    const int n = tt / per_n, r = tt - n * per_n;
    const int ty = r / a.tiles_x, tx = r - ty * a.tiles_x;
    const int oy0 = ty * G::TH, ox0 = tx * TW;
    const int gy0 = KS == 1 ? oy0 * S : oy0 * S - G::PAD, gx0 = ox0 * S - G::LEFT;
    unsigned off[XSLOTS], from[XSLOTS], second[XSLOTS];
#pragma unroll
    for (int j = 0; j < XSLOTS; ++j) {
      const int e = lane + 64 * j, iy = e / G::XD, q = e - iy * G::XD;
      const int gy = gy0 + iy * G::YS, gx = gx0 + 4 * q;
      const bool ok = e < G::XE && gy >= 0 && gy < a.h && gx >= 0 && gx < a.w;
      off[j] = ok ? (unsigned)(gy * a.w + gx) : 0x80000000u;
      if constexpr (!AL) {
        // a dword may start on any byte, span two blocks and reach past the plane's last byte: then the last four bytes are
        // read and shifted.  Lanes without a place read the plane's first bytes, which the mask clears.
        mask[j] = ok && there ? (a.w - gx < 4 ? a.w - gx : 4) : 0;
        off[j] = ok ? off[j] : 0u;
        cut[j] = 32 - (int)(off[j] & 31u);
        from[j] = off[j] < plane_bytes - 4u ? off[j] : plane_bytes - 4u;
        shift[j] = 8u * (off[j] - from[j]);
        second[j] = (off[j] + 3u) >> 5 < (unsigned)a.blocks - 1u ? (off[j] + 3u) >> 5 : (unsigned)a.blocks - 1u;
      }
    }
    // A wave whose channels all lie in one source needs one descriptor per tile and a scalar offset per channel; otherwise
    // every channel's address is put together (as many scalar instructions as a slot has vector ones).
    if (AL && together) {
      const unsigned long long b = (unsigned long long)(unsigned)n * xp[0].step;
      const __amdgpu_buffer_rsrc_t rc = rsrc(xp[0].codes + 32ull * b, there ? (unsigned)XPW * plane_bytes : 0u);
      const __amdgpu_buffer_rsrc_t rs = rsrc(xp[0].scales + b, there ? (unsigned)(XPW * a.blocks) : 0u);
#pragma unroll
      for (int c = 0; c < XPW; ++c)
#pragma unroll
        for (int j = 0; j < XSLOTS; ++j) {
          xk[c][j] = __builtin_amdgcn_raw_buffer_load_b32(rc, off[j], c * plane_bytes, 0);
          xs[c][j] = __builtin_amdgcn_raw_buffer_load_b8(rs, (int)off[j] >> 5, c * a.blocks, 0);      // (no place: still past the end)
        }
    } else
#pragma unroll
    for (int c = 0; c < XPW; ++c) {
      const unsigned long long b = (unsigned long long)(unsigned)n * xp[c].step;
      const unsigned live = there && c < xlive ? 0xffffffffu : 0u;
#pragma unroll
      for (int j = 0; j < XSLOTS; ++j) {
        if constexpr (AL) {
          xk[c][j] = __builtin_amdgcn_raw_buffer_load_b32(rsrc(xp[c].codes + 32ull * b, plane_bytes & live), off[j], 0, 0);
          xs[c][j] = __builtin_amdgcn_raw_buffer_load_b8(rsrc(xp[c].scales + b, (unsigned)a.blocks & live), (int)off[j] >> 5, 0, 0);
        } else {
          // (channels past the last: some plane; their sums are never looked at)
          const unsigned long long cp = together ? xp[0].codes + 32ull * b + (unsigned long long)c * plane_bytes : xp[c].codes + 32ull * b;
          const unsigned long long sp = together ? xp[0].scales + b + (unsigned long long)(c * a.blocks) : xp[c].scales + b;
          xk[c][j] = reinterpret_cast<const Dword*>(cp + from[j])->v;
          xs[c][j] = reinterpret_cast<const uint8_t*>(sp)[off[j] >> 5];
          xs2[c][j] = reinterpret_cast<const uint8_t*>(sp)[second[j]];
        }
      }
    }
    if constexpr (AL) {
      // four adjacent pixels of a row
      const int e = lane % G::GE, oy = oy0 + 4 * e / TW, ox = ox0 + 4 * e % TW;
      const unsigned at = oy < a.ho && ox < a.wo ? 4u * ((unsigned)(lane / G::GE) * gplane + (unsigned)(oy * a.wo + ox)) : 0x80000000u;
#pragma unroll
      for (int i = 0; i < GLOADS; ++i) {
        const int ch = co0 + (sw + G::NS * i) * CPL, live = there ? (a.cout - ch < CPL ? a.cout - ch : CPL) : 0;
        gr[i] = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(
            rsrc((unsigned long long)a.g + 4ull * ((unsigned long long)(unsigned)n * a.cout + (live > 0 ? ch : 0)) * gplane,
                 live > 0 ? 4u * (unsigned)live * gplane : 0u), at, 0, 0));      // (CPL planes below 2^31 bytes: checked on the host)
      }
    } else {
      unsigned at[LPC];
#pragma unroll
      for (int p = 0; p < LPC; ++p) {
        const int oy = oy0 + (64 * p + lane) / TW, ox = ox0 + lane % TW;
        at[p] = oy < a.ho && ox < a.wo ? 4u * (unsigned)(oy * a.wo + ox) : 0x80000000u;
      }
#pragma unroll
      for (int c = 0; c < GPW; ++c) {
        const int ch = co0 + GPW * sw + c;
        const bool live = there && ch < a.cout;
        const __amdgpu_buffer_rsrc_t rg = rsrc((unsigned long long)a.g + 4ull * ((unsigned long long)(unsigned)n * a.cout + (live ? ch : 0)) * gplane,
                                               live ? 4u * gplane : 0u);
#pragma unroll
        for (int p = 0; p < LPC; ++p) gr[c * LPC + p] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rg, at[p], 0, 0));
      }
    }
  }

  // decode what load() requested into an LDS buffer
  template <bool E4M3>
  __device__ __forceinline__ void store_as(char* buf) {
#pragma unroll
    for (int j = 0; j < XSLOTS; ++j) {
      const int e = lane + 64 * j, iy = e / G::XD, q = e - iy * G::XD;
#pragma unroll
      for (int c = 0; c < XPW; ++c) {
        const float s0 = scale_of(xs[c][j], flip);
        uint2 v;
        if constexpr (AL) {
          v = decode<E4M3>(xk[c][j], s0, s0, s0, s0);
        } else {
          const float s4 = scale_of(xs2[c][j], flip);
          v = decode<E4M3>(xk[c][j] >> shift[j], s0, cut[j] > 1 ? s0 : s4, cut[j] > 2 ? s0 : s4, cut[j] > 3 ? s0 : s4);
          // codes past the row's end are padding: zeros (also where the scale is that of a poisoned block)
          v.x = mask[j] > 1 ? v.x : mask[j] > 0 ? v.x & 0xffffu : 0u;
          v.y = mask[j] > 3 ? v.y : mask[j] > 2 ? v.y & 0xffffu : 0u;
        }
        if (64 * (j + 1) <= G::XE || e < G::XE) {
          char* const row = buf + (XPW * sw + c) * G::XSTR + iy * G::XROW * 2;
          if constexpr (S == 1) {
            *reinterpret_cast<uint2*>(row + 8 * q) = v;
          } else {
            const unsigned even = __builtin_amdgcn_perm(v.y, v.x, 0x05040100u), odd = __builtin_amdgcn_perm(v.y, v.x, 0x07060302u);
            if constexpr (KS == 1) {
              *reinterpret_cast<unsigned*>(row + 4 * q) = even;
            } else {
              // even columns from column 4 on (the middle tap's), odd ones from column 1 on
              if (q >= 1 && q <= TW / 2) *reinterpret_cast<unsigned*>(row + 4 * (q - 1)) = even;
              *reinterpret_cast<unsigned*>(row + 2 * TW + 4 * q) = odd;
            }
          }
        }
      }
    }
    if constexpr (AL) {
      char* const to = buf + G::XBYTES + (sw * CPL + lane / G::GE) * G::GUNITS * 16 + lane % G::GE * 16;
#pragma unroll
      for (int i = 0; i < GLOADS; ++i) {
        *reinterpret_cast<float4*>(to + i * G::NS * CPL * G::GUNITS * 16) = gr[i];
        gsum[i] += (gr[i].x + gr[i].y) + (gr[i].z + gr[i].w);
      }
    } else {
      char* const to = buf + G::XBYTES + GPW * sw * G::GUNITS * 16 + 4 * lane;
#pragma unroll
      for (int c = 0; c < GPW; ++c) {
#pragma unroll
        for (int p = 0; p < LPC; ++p) {
          *reinterpret_cast<float*>(to + c * G::GUNITS * 16 + 256 * p) = gr[c * LPC + p];
          gsum[c] += gr[c * LPC + p];
        }
      }
    }
  }

  // (called once for each of the workgroup's tiles, in order)
  __device__ __forceinline__ void store(char* buf) {
    if (a.e4m3) store_as<true>(buf);
    else store_as<false>(buf);
    --left;
    flip ^= left == 0 ? 0x80000000u : 0u;
    // (one sum over all tiles of a workgroup: 1024 equal gradients per channel over 2048 tiles off by 3e-5)
    if (left == 0) {
#pragma unroll
      for (int i = 0; i < GSUMS; ++i) {
        gbefore[i] += gsum[i];
        gsum[i] = 0.f;
      }
    }
    left = left == 0 ? a.seg_tiles : left;
  }

  // the bias gradient of what was staged: a channel's sums are those of GE adjacent lanes (not AL: of all)
  __device__ __forceinline__ void bias(float* out) {
    constexpr int LANES = AL ? G::GE : 64;
#pragma unroll
    for (int i = 0; i < GSUMS; ++i) {
      float v = gbefore[i] + gsum[i];
#pragma unroll
      for (int m = LANES / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
      if (lane % LANES == 0) out[AL ? (stid + 64 * G::NS * i) / G::GE : GPW * sw + i] = v;
    }
  }
};

template <int KS, int S, int MT, int CT, int TW, bool AL>
__global__ __launch_bounds__(512) void wgrad_ckpt_kernel(const Args a) {
  using G = Geo<KS, S, MT, CT, TW>;
  constexpr int KG = G::KG, TAPS = G::TAPS, ACC = G::ACC;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cob = blockIdx.y / a.n_cib, cib = blockIdx.y - cob * a.n_cib;
  const int co0 = cob * G::GCH, ci0 = cib * G::XCH;
  const int nsplit = gridDim.x;
  // Workgroups go to the eight XCDs in turn, each with an L2 of its own, and neighbouring tiles share the cache lines of the
  // codes (a staged row is 40 bytes): tiles that follow each other go to one XCD.
  const int part = nsplit % 8 == 0 ? ((int)blockIdx.x & 7) * (nsplit >> 3) + ((int)blockIdx.x >> 3) : (int)blockIdx.x;

  // Every second slab, over workgroups and in time, is computed with its inputs' signs changed and changed back when it is
  // stored: the matrix instruction cuts what lies far below its running sum downwards, and over an even number of slabs
  // that drift cancels (64->64 3x3 at 32x256x256: relative error 2.0e-6 without, of which 93 % is drift; 1024->1024 1x1 at
  // 4x128x128, one workgroup per block and 16 slabs: mean error of the results 2.3e-7 of their size with all slabs alike).
  // An odd number leaves one slab's.  It costs nothing: the sign rides on the scale.
  unsigned flip = ((unsigned)(part + a.seg0) & 1u) << 31;

  if (KS != 7 && wave >= G::NM) {
    // ------------------------------------------------------------ staging
    Stager<G, AL> st(a, lane, wave - G::NM, co0, ci0, flip);
    // (one copy of the code from the first load on: a one-tile workgroup spends much of its time fetching instructions, 64->64
    // stride 2 33 -> 26 us)
    int buf = G::BUF;
#pragma unroll 1
    for (int t = a.tile0 + part - 2 * nsplit; t < a.n_tiles; t += nsplit) {
      const bool begun = t > a.tile0 + part - 2 * nsplit;
      if (begun && t + nsplit < a.n_tiles) st.store(lds + (G::BUF - buf));      // tile t + nsplit
      // AL: past the last tile the descriptors are empty, and a branch here would have the loads waited for at its end
      if (AL || t + 2 * nsplit < a.n_tiles) st.load(t + 2 * nsplit);
      if (begun) {
        __syncthreads();
        buf = G::BUF - buf;
      }
    }
    if (a.bias_partial != nullptr && cib == 0) st.bias(a.bias_partial + (long long)part * a.cout_pad + co0);
    return;
  }

  // -------------------------------------------------------------- multiplying
  const int half = lane >> 5, l32 = lane & 31;
  const int corner = KS == 7 ? 0 : wave % (MT * CT), grp = KS == 7 ? 0 : wave / (MT * CT);
  const int mt = corner / CT, ct = corner % CT;
  f32x16 acc[ACC];
#pragma unroll
  for (int t = 0; t < ACC; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

  const int ga = G::XBYTES + (mt * 32 + l32) * G::GUNITS * 16 + half * 32;
  const int xa = (ct * 32 + l32) * G::XSTR + half * 16;
  constexpr int ROWS = KS == 7 ? 1 : KS;            // staged rows a row piece meets in this wave
  constexpr int STEPS = G::STEPS / KG;              // row pieces per tile in this wave

  // one tile: the operands of a row piece are read and split while the piece before is multiplied
  auto multiply = [&](const char* buf) __attribute__((always_inline)) {
    auto gradient = [&](int i) __attribute__((always_inline)) {
      const int step = i * KG + grp, row = step / (TW / 16), px = step % (TW / 16) * 16;
      const float4* const gp = reinterpret_cast<const float4*>(buf + ga + (row * TW + px) * 4);
      return split(gp[0], gp[1]);
    };
    // (7x7: two waves of a SIMD multiply, and the operands of two row pieces would not leave registers for the staging)
    constexpr bool AHEAD = KS != 7;
    Split s = gradient(0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int step = i * KG + grp, row = step / (TW / 16), px = step % (TW / 16) * 16;
      Split next = s;
      if (AHEAD && i + 1 < STEPS) next = gradient(i + 1);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int ky = KS == 7 ? wave : r;
        const char* const xr = buf + xa + ((KS == 1 ? row : row * S + ky) * G::XROW + px) * 2;
        bf16x8 b[KS];
        if constexpr (KS == 1) {
          b[0] = *reinterpret_cast<const bf16x8*>(xr);
        } else if constexpr (KS == 3 && S == 1) {
          // staged column 4 is pixel 0: the middle tap is elements 4..11, its neighbours one element either way
          const unsigned lo = *reinterpret_cast<const unsigned*>(xr + 4), hi = *reinterpret_cast<const unsigned*>(xr + 24);
          const uint2 m0 = *reinterpret_cast<const uint2*>(xr + 8), m1 = *reinterpret_cast<const uint2*>(xr + 16);
          const unsigned d[6] = {lo, m0.x, m0.y, m1.x, m1.y, hi};
          b[0] = window<1>(d); b[1] = window<2>(d); b[2] = window<3>(d);
        } else if constexpr (S == 1) {
          const u32x4 lo = *reinterpret_cast<const u32x4*>(xr), hi = *reinterpret_cast<const u32x4*>(xr + 16);
          const unsigned d[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          b[0] = window<1>(d); b[1] = window<2>(d); b[2] = window<3>(d); b[3] = window<4>(d);
          b[4] = window<5>(d); b[5] = window<6>(d); b[6] = window<7>(d);
        } else {
          const u32x4 lo = *reinterpret_cast<const u32x4*>(xr + 2 * TW);
          const unsigned d[5] = {lo[0], lo[1], lo[2], lo[3], *reinterpret_cast<const unsigned*>(xr + 2 * TW + 16)};
          b[0] = window<1>(d); b[2] = window<2>(d);
          b[1] = *reinterpret_cast<const bf16x8*>(xr);
        }
#pragma unroll
        for (int kx = 0; kx < KS; ++kx) acc[r * KS + kx] = mfma(s.a3, b[kx], acc[r * KS + kx]);
#pragma unroll
        for (int kx = 0; kx < KS; ++kx) acc[r * KS + kx] = mfma(s.a2, b[kx], acc[r * KS + kx]);
#pragma unroll
        for (int kx = 0; kx < KS; ++kx) acc[r * KS + kx] = mfma(s.a1, b[kx], acc[r * KS + kx]);
      }
      if (!AHEAD && i + 1 < STEPS) next = gradient(i + 1);
      s = next;
    }
  };

  // slab after slab (a workgroup that runs out of tiles early still writes its slabs); register r of an accumulator is row
  // (r & 3) + 8 (r >> 2) + 4 half, column l32
  const long long slab_floats = (long long)TAPS * a.cout_pad * a.cin_pad;
  float* out = a.partial + ((long long)part * KG + grp) * slab_floats + (long long)(co0 + mt * 32 + 4 * half) * a.cin_pad +
               ci0 + ct * 32 + l32;
  // 7x7: the multiplying waves stage as well (one wave cannot hold a tile's loads); of the two waves of a SIMD one does so
  // before it multiplies and one after, so that the decoding of the one runs beside the matrix instructions of the other
  auto st = [&]() __attribute__((always_inline)) {
    if constexpr (KS == 7) return Stager<G, AL>(a, lane, wave, co0, ci0, flip);
    else return 0;
  }();
  const bool late = wave >= 4;
  int t = a.tile0 + part, buf = 0;
  if constexpr (KS == 7) {
    st.load(t);
    st.store(lds);
    st.load(t + nsplit);
  }
  __syncthreads();
#pragma unroll 1
  for (int seg = 0; seg < a.segments; ++seg) {
#pragma unroll 1
    for (int k = 0; k < a.seg_tiles && t < a.n_tiles; ++k, t += nsplit) {
      if constexpr (KS == 7) {
        if (!late) {
          st.store(lds + (G::BUF - buf));
          st.load(t + 2 * nsplit);
        }
      }
      if (KS != 7 || wave < 7) multiply(lds + buf);
      if constexpr (KS == 7) {
        if (late) {
          st.store(lds + (G::BUF - buf));
          st.load(t + 2 * nsplit);
        }
      }
      __syncthreads();
      buf = G::BUF - buf;
    }
    if (KS == 7 && wave == 7) continue;
#pragma unroll
    for (int tp = 0; tp < ACC; ++tp) {
      float* const pt = out + (long long)(KS == 7 ? wave * 7 + tp : tp) * a.cout_pad * a.cin_pad;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pt[((r & 3) + 8 * (r >> 2)) * a.cin_pad] = __uint_as_float(__float_as_uint(acc[tp][r]) ^ flip);
        acc[tp][r] = 0.f;
      }
    }
    out += (long long)nsplit * KG * slab_floats;
    flip ^= 0x80000000u;
  }
  if constexpr (KS == 7) {
    if (a.bias_partial != nullptr && cib == 0) st.bias(a.bias_partial + (long long)part * a.cout_pad + co0);
  }
}

struct Plan {
  int ho, wo, tw, th, tiles_x, tiles_y, n_tiles, cout_pad, cin_pad, n_cib, blocks, nsplit, taps, mt, ct;
  int kg, seg_tiles, segments, all_segments;      // waves per corner, tiles of a workgroup per slab, slabs in time of a launch and in all
};

template <class K>
int allow_lds(K kernel, int bytes, std::atomic<unsigned long long>* done, const char* what) {
  // LDS above the default needs an opt-in per kernel and device (twice is harmless)
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device > 63) device = 0;
  const unsigned long long bit = 1ull << device;
  if (done->load(std::memory_order_acquire) & bit) return DVC_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    dvc::set_error("hipFuncSetAttribute(%s): %s", what, hipGetErrorString(e));
    return DVC_EHIP;
  }
  done->fetch_or(bit, std::memory_order_release);
  return DVC_OK;
}

template <int KS, int S, int MT, int CT, int TW, bool AL>
int launch(const Args& a, const Plan& p, hipStream_t st) {
  using G = Geo<KS, S, MT, CT, TW>;
  static std::atomic<unsigned long long> done{0};
  if (int rc = allow_lds(&wgrad_ckpt_kernel<KS, S, MT, CT, TW, AL>, G::LDS_BYTES, &done, "wgrad_ckpt_kernel")) return rc;
  hipLaunchKernelGGL((wgrad_ckpt_kernel<KS, S, MT, CT, TW, AL>), dim3(p.nsplit, p.blocks), dim3(512), G::LDS_BYTES, st, a);
  return dvc::check_launch("wgrad_ckpt_kernel");
}

template <int KS, int S, int TW, bool AL>
int launch_block(const Args& a, const Plan& p, hipStream_t st) {
  if (p.mt == 2) return p.ct == 2 ? launch<KS, S, 2, 2, TW, AL>(a, p, st) : launch<KS, S, 2, 1, TW, AL>(a, p, st);
  return p.ct == 2 ? launch<KS, S, 1, 2, TW, AL>(a, p, st) : launch<KS, S, 1, 1, TW, AL>(a, p, st);
}

template <bool AL>
int launch_shape(int ks, int stride, const Args& a, const Plan& p, hipStream_t st) {
  if (ks == 3 && stride == 1) return p.tw == 16 ? launch_block<3, 1, 16, AL>(a, p, st) : launch_block<3, 1, 32, AL>(a, p, st);
  if (ks == 3) return launch_block<3, 2, 32, AL>(a, p, st);
  if (ks == 7) return launch<7, 1, 1, 1, 32, AL>(a, p, st);
  return stride == 1 ? launch_block<1, 1, 32, AL>(a, p, st) : launch_block<1, 2, 32, AL>(a, p, st);
}

int launch_aligned(int ks, int stride, const Args& a, const Plan& p, hipStream_t st);
int launch_any(int ks, int stride, const Args& a, const Plan& p, hipStream_t st);

}  // namespace dvc_wgrad_ckpt
