// Weight gradient of the 2-D convolutions from 8-bit activation checkpoints: entry points, plan and the reduction of the
// partial results (the kernels are in conv_wgrad_ckpt_impl.h).
#include "conv_wgrad_ckpt_impl.h"

namespace dvc_wgrad_ckpt {

int launch_aligned(int ks, int stride, const Args& a, const Plan& p, hipStream_t st) { return launch_shape<true>(ks, stride, a, p, st); }

namespace {

// gW[co][ci][tap] = sum over slabs of partial[slab][tap][co][ci], gB[co] likewise over splits (units past the weight's); `more`: added
// to what they hold.  A lane takes four adjacent input channels (rows of a slab are padded to 32), a block UNITS such units; each
// of its GROUPS groups of lanes adds every GROUPS-th slab, with the loads of four slabs in flight, and the sums are added in a
// fixed order.
__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

template <int UNITS, int GROUPS>
__global__ __launch_bounds__(UNITS * GROUPS) void wgrad_ckpt_reduce_kernel(const float* partial, float* gw, int slabs, int nsplit, int taps,
                                                                       int cout, int cin, int cout_pad, int cin_pad,
                                                                       const float* bias_partial, float* gb, int more) {
  __shared__ float4 part[GROUPS][UNITS];
  const unsigned cin4 = (unsigned)(cin + 3) / 4, units = (unsigned)cout * (unsigned)taps * cin4;
  const unsigned all = units + (gb != nullptr ? (unsigned)(cout + 3) / 4 : 0u);
  const int lane = threadIdx.x % UNITS, kg = threadIdx.x / UNITS;
  for (unsigned i0 = blockIdx.x * (unsigned)UNITS; i0 < all; i0 += gridDim.x * (unsigned)UNITS) {
    const unsigned i = i0 + lane;
    const unsigned ci = i % cin4 * 4, q = i / cin4, tap = q % (unsigned)taps, co = q / (unsigned)taps;
    const bool weight = i < units;
    const float* const p = weight ? partial + ((long long)tap * cout_pad + co) * cin_pad + ci : bias_partial + 4ll * (i - units);
    const long long step = weight ? (long long)taps * cout_pad * cin_pad : cout_pad;
    const int count = i < all ? (weight ? slabs : nsplit) : 0;
    auto at = [&](int k) { return *reinterpret_cast<const float4*>(p + k * step); };
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    int k = kg;
    for (; k + 3 * GROUPS < count; k += 4 * GROUPS) {
      const float4 v0 = at(k), v1 = at(k + GROUPS), v2 = at(k + 2 * GROUPS), v3 = at(k + 3 * GROUPS);
      s = add4(s, add4(add4(v0, v1), add4(v2, v3)));
    }
    for (; k < count; k += GROUPS) s = add4(s, at(k));
    part[kg][lane] = s;
    __syncthreads();
    if (kg == 0 && i < all) {
      float4 v = part[0][lane];
#pragma unroll 5      // (all 63 of the widest form would not fit the registers of 16 waves)
      for (int w = 1; w < GROUPS; ++w) v = add4(v, part[w][lane]);
      const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (weight) {
          float* const to = gw + ((long long)co * cin + ci + j) * taps + tap;
          if ((int)ci + j < cin) *to = more ? *to + r[j] : r[j];
        } else {
          const int c = (int)(4 * (i - units)) + j;
          if (c < cout) gb[c] = more ? gb[c] + r[j] : r[j];
        }
      }
    }
    __syncthreads();
  }
}

constexpr long long kSlabBytes = 128ll << 20;

int make_plan(int cout, int cin, int ks, int stride, int batch, int h, int w, Plan* p, const char* who) {
  DVC_REQUIRE(ks == 1 || ks == 3 || ks == 7, "%s: ksize=%d unsupported", who, ks);
  DVC_REQUIRE(stride == 1 || stride == 2, "%s: stride=%d unsupported", who, stride);
  DVC_REQUIRE(!(ks == 7 && stride != 1), "%s: 7x7 stride 2 unsupported", who);
  DVC_REQUIRE(cout >= 1 && cin >= 1 && batch >= 1 && h >= 1 && w >= 1, "%s: bad dims", who);
  DVC_REQUIRE((long long)h * w < (1LL << 28), "%s: plane too large", who);
  DVC_REQUIRE(((long long)h * w + 31) / 32 * cin < (1LL << 31) && (long long)cout * cin * ks * ks < (1LL << 31), "%s: too many channels", who);
  const int pad = ks / 2;
  p->ho = (h + 2 * pad - ks) / stride + 1;
  p->wo = (w + 2 * pad - ks) / stride + 1;
  p->tw = ks == 3 && stride == 1 && p->wo <= 16 ? 16 : 32;
  p->mt = (cout > 32 && ks != 7) ? 2 : 1;
  p->ct = (cin > 32 && ks != 7) ? 2 : 1;
  p->th = (ks == 3 && stride == 2 ? 2 : 4) * (32 / p->tw);
  p->tiles_x = (p->wo + p->tw - 1) / p->tw;
  p->tiles_y = (p->ho + p->th - 1) / p->th;
  const long long nt = (long long)batch * p->tiles_x * p->tiles_y;
  DVC_REQUIRE(nt < (1LL << 29), "%s: too many tiles", who);
  p->n_tiles = (int)nt;
  const int cob = 32 * p->mt, cib = 32 * p->ct;
  p->cout_pad = (cout + cob - 1) / cob * cob;
  p->cin_pad = (cin + cib - 1) / cib * cib;
  p->n_cib = p->cin_pad / cib;
  p->blocks = (p->cout_pad / cob) * p->n_cib;
  p->taps = ks * ks;
  // one 8-wave workgroup fits a CU: about one round of them
  int s = (256 + p->blocks - 1) / p->blocks;
  p->nsplit = s > p->n_tiles ? p->n_tiles : s;
  // A running sum is rounded twice per matrix instruction, so a slab ends after 256 row pieces of a wave (768 instructions;
  // 64->64 3x3 at 32x256x256, 512 pieces per wave: relative error 7e-7 in two slabs, 1.0e-6 in one); 7x7, whose slabs are
  // five times as large, after 512
  p->kg = ks == 7 ? 1 : 4 / (p->mt * p->ct);
  p->seg_tiles = (ks == 7 ? 512 : 256) / (p->th * p->tw / 16 / p->kg);
  const int most = (p->n_tiles + p->nsplit - 1) / p->nsplit;      // tiles of a workgroup
  p->all_segments = (most + p->seg_tiles - 1) / p->seg_tiles;
  // Slabs in time do not add up in memory: beyond 128 MiB of them the tiles are dealt out over several launches, each with a
  // reduction that adds to the result (192->192 3x3 at 32x256x256: 693 MB in one launch).  Adding to the slabs
  // inside the kernel instead needs less, but is slower by the latency of reading them (64->64 3x3 at 32x256x256 460 -> 485 us,
  // 192->192 at 4x256x256 647 -> 728).
  const long long one = 4ll * p->nsplit * p->kg * p->taps * p->cout_pad * p->cin_pad, most_at_once = one < kSlabBytes ? kSlabBytes / one : 1;
  const long long launches = (p->all_segments + most_at_once - 1) / most_at_once;
  p->segments = (int)((p->all_segments + launches - 1) / launches);
  return DVC_OK;
}
inline long long slab_floats(const Plan& p) { return (long long)p.segments * p.nsplit * p.kg * p.taps * p.cout_pad * p.cin_pad; }

int check_srcs(const DvcCkpt* srcs, int n_src, int* cin, const char* who) {
  DVC_REQUIRE(srcs != nullptr && n_src >= 1 && n_src <= DVC_MAX_SRC, "%s: n_src=%d not in 1..%d", who, n_src, DVC_MAX_SRC);
  *cin = 0;
  for (int s = 0; s < n_src; ++s) {
    DVC_REQUIRE(srcs[s].codes != nullptr && srcs[s].scales != nullptr && srcs[s].channels >= 1, "%s: bad source %d", who, s);
    DVC_REQUIRE(reinterpret_cast<uintptr_t>(srcs[s].codes) % 16 == 0, "%s: source %d: codes must start on 16 bytes", who, s);
    DVC_REQUIRE(srcs[s].format == srcs[0].format && (srcs[s].format == DVC_CKPT_INT8 || srcs[s].format == DVC_CKPT_E4M3),
                "%s: source %d: format %d", who, s, srcs[s].format);
    *cin += srcs[s].channels;
  }
  return DVC_OK;
}

}  // namespace
}  // namespace dvc_wgrad_ckpt

using namespace dvc_wgrad_ckpt;

extern "C" int64_t dvc_conv2d_wgrad_ckpt_scratch_floats(int32_t cout, int32_t cin, int32_t ksize, int32_t stride,
                                                        int32_t batch, int32_t in_h, int32_t in_w) {
  Plan p;
  if (int rc = make_plan(cout, cin, ksize, stride, batch, in_h, in_w, &p, "dvc_conv2d_wgrad_ckpt_scratch_floats")) return rc;
  return slab_floats(p) + (int64_t)p.nsplit * p.cout_pad;
}

extern "C" int dvc_conv2d_wgrad_ckpt(const DvcCkpt* srcs, int32_t n_src, int32_t batch, int32_t in_h, int32_t in_w,
                                     const float* grad_out, int32_t out_channels, int32_t ksize, int32_t stride,
                                     float* scratch, float* grad_weight, float* grad_bias, void* stream) {
  const char* const who = "dvc_conv2d_wgrad_ckpt";
  int cin;
  if (int rc = check_srcs(srcs, n_src, &cin, who)) return rc;
  DVC_REQUIRE(grad_out != nullptr && scratch != nullptr && grad_weight != nullptr, "%s: null pointer", who);
  DVC_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "%s: scratch must start on 16 bytes", who);
  Plan p;
  if (int rc = make_plan(out_channels, cin, ksize, stride, batch, in_h, in_w, &p, who)) return rc;
  Args a{};
  int first = 0;
  for (int s = 0; s < DVC_MAX_SRC; ++s) {
    const bool have = s < n_src;
    a.codes[s] = have ? srcs[s].codes : srcs[0].codes;
    a.scales[s] = have ? srcs[s].scales : srcs[0].scales;
    a.first[s] = have ? first : cin;
    a.chans[s] = have ? srcs[s].channels : 1;
    first += have ? srcs[s].channels : 0;
  }
  a.e4m3 = srcs[0].format == DVC_CKPT_E4M3;
  a.cin = cin;
  a.h = in_h;
  a.w = in_w;
  a.blocks = (int)(((long long)in_h * in_w + 31) / 32);
  a.cout = out_channels;
  a.ho = p.ho;
  a.wo = p.wo;
  a.g = grad_out;
  a.partial = scratch;
  a.bias_partial = grad_bias != nullptr ? scratch + slab_floats(p) : nullptr;
  a.cout_pad = p.cout_pad;
  a.cin_pad = p.cin_pad;
  a.n_cib = p.n_cib;
  a.tiles_x = p.tiles_x;
  a.tiles_y = p.tiles_y;
  a.seg_tiles = p.seg_tiles;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool aligned = in_w % 4 == 0 && p.wo % 4 == 0 && reinterpret_cast<uintptr_t>(grad_out) % 16 == 0 &&
                       16LL * p.ho * p.wo < (1LL << 31);
  const long long units = (long long)out_channels * p.taps * ((cin + 3) / 4) + (out_channels + 3) / 4;
  // Blocks of 64 units by 16 groups (64->64 3x3 in 256 slabs: 8 us, 16 by 64 10); where those are fewer than half the CUs, 16 by
  // 64 (3->64 3x3 in 1024 slabs: 42 us in 10 blocks, 18 in 37); of few slabs 64 by 4.
#define REDUCE(UNITS, GROUPS)                                                                                                        \
  hipLaunchKernelGGL((wgrad_ckpt_reduce_kernel<UNITS, GROUPS>), dim3((unsigned)((units + UNITS - 1) / UNITS < 16384 ? (units + UNITS - 1) / UNITS : 16384)), \
                     dim3(UNITS * GROUPS), 0, st, scratch, grad_weight, slabs, p.nsplit, p.taps, out_channels, cin, p.cout_pad, p.cin_pad, \
                     a.bias_partial, grad_bias, a.seg0 != 0)
  for (a.seg0 = 0; a.seg0 < p.all_segments; a.seg0 += p.segments) {
    const long long step = (long long)p.nsplit * p.seg_tiles, end = step * (a.seg0 + p.segments);
    a.segments = a.seg0 + p.segments < p.all_segments ? p.segments : p.all_segments - a.seg0;
    a.tile0 = (int)(step * a.seg0);
    a.n_tiles = end < p.n_tiles ? (int)end : p.n_tiles;
    if (int rc = aligned ? launch_aligned(ksize, stride, a, p, st) : launch_any(ksize, stride, a, p, st)) return rc;
    const int slabs = a.segments * p.nsplit * p.kg;
    if (slabs < 64) REDUCE(64, 4);
    else if (units < 64 * 128) REDUCE(16, 64);
    else REDUCE(64, 16);
    if (int rc = dvc::check_launch("wgrad_ckpt_reduce_kernel")) return rc;
  }
#undef REDUCE
  return DVC_OK;
}
