// Weight gradient of the 2-D convolutions from 8-bit activation checkpoints: entry points, plan and the reduction of the
// partial results (the kernels are in conv_wgrad_ckpt_impl.h).
#include "conv_wgrad_ckpt_impl.h"

namespace dvc_wgrad_ckpt {

int launch_aligned(int ks, int stride, const Args& a, const Plan& p, hipStream_t st) { return launch_shape<true>(ks, stride, a, p, st); }

namespace {

// gW[co][ci][tap] = sum over slabs of partial[slab][tap][co][ci], gB[co] likewise over splits (indices past the weight's).  A block
// takes 64 results; each of its WAVES waves adds every WAVES-th slab, with the loads of four slabs in flight, and the sums are
// added in a fixed order.  16 waves for many slabs (256 of a 64 x 64 3x3 layer: 9 us, 20 with four waves and one load after
// the other), 4 for few.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void wgrad_ckpt_reduce_kernel(const float* partial, float* gw, int slabs, int nsplit, int taps, int cout, int cin,
                                                                 int cout_pad, int cin_pad, const float* bias_partial, float* gb) {
  __shared__ float part[WAVES][64];
  const long long total = (long long)cout * taps * cin;
  const long long total_all = total + (gb != nullptr ? cout : 0);
  const int lane = threadIdx.x & 63, kg = threadIdx.x >> 6;
  for (long long i0 = blockIdx.x * 64LL; i0 < total_all; i0 += (long long)gridDim.x * 64) {
    const long long i = i0 + lane;
    const float* p = nullptr;
    long long step = 0, dst = -1;
    int count = slabs;
    if (i < total) {
      const unsigned r = (unsigned)i, ci = r % (unsigned)cin, q = r / (unsigned)cin;      // (a weight has below 2^31 elements)
      const unsigned tap = q % (unsigned)taps, co = q / (unsigned)taps;
      p = partial + ((long long)tap * cout_pad + co) * cin_pad + ci;
      step = (long long)taps * cout_pad * cin_pad;
      dst = ((long long)co * cin + ci) * taps + tap;
    } else if (i < total_all) {
      p = bias_partial + (i - total);
      step = cout_pad;
      count = nsplit;
    }
    float s = 0.f;
    if (p != nullptr) {
      int k = kg;
      for (; k + 3 * WAVES < count; k += 4 * WAVES) {
        const float v0 = p[k * step], v1 = p[(k + WAVES) * step], v2 = p[(k + 2 * WAVES) * step], v3 = p[(k + 3 * WAVES) * step];
        s += (v0 + v1) + (v2 + v3);
      }
      for (; k < count; k += WAVES) s += p[k * step];
    }
    part[kg][lane] = s;
    __syncthreads();
    if (kg == 0 && p != nullptr) {
      float v = part[0][lane];
#pragma unroll
      for (int k = 1; k < WAVES; ++k) v += part[k][lane];
      if (dst >= 0) gw[dst] = v;
      else gb[i - total] = v;
    }
    __syncthreads();
  }
}

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
  const int kg = ks == 7 ? 1 : 4 / (p->mt * p->ct), pieces = p->th * p->tw / 16 / kg;
  p->seg_tiles = (ks == 7 ? 512 : 256) / pieces;
  const int most = (p->n_tiles + p->nsplit - 1) / p->nsplit;      // tiles of a workgroup
  p->segments = (most + p->seg_tiles - 1) / p->seg_tiles;
  p->slabs = p->segments * p->nsplit * kg;
  return DVC_OK;
}

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
  return (int64_t)p.slabs * p.taps * p.cout_pad * p.cin_pad + (int64_t)p.nsplit * p.cout_pad;
}

extern "C" int dvc_conv2d_wgrad_ckpt(const DvcCkpt* srcs, int32_t n_src, int32_t batch, int32_t in_h, int32_t in_w,
                                     const float* grad_out, int32_t out_channels, int32_t ksize, int32_t stride,
                                     float* scratch, float* grad_weight, float* grad_bias, void* stream) {
  const char* const who = "dvc_conv2d_wgrad_ckpt";
  int cin;
  if (int rc = check_srcs(srcs, n_src, &cin, who)) return rc;
  DVC_REQUIRE(grad_out != nullptr && scratch != nullptr && grad_weight != nullptr, "%s: null pointer", who);
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
  a.bias_partial = grad_bias != nullptr ? scratch + (long long)p.slabs * p.taps * p.cout_pad * p.cin_pad : nullptr;
  a.cout_pad = p.cout_pad;
  a.cin_pad = p.cin_pad;
  a.n_cib = p.n_cib;
  a.tiles_x = p.tiles_x;
  a.tiles_y = p.tiles_y;
  a.n_tiles = p.n_tiles;
  a.seg_tiles = p.seg_tiles;
  a.segments = p.segments;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool aligned = in_w % 4 == 0 && p.wo % 4 == 0 && reinterpret_cast<uintptr_t>(grad_out) % 16 == 0 &&
                       4LL * out_channels * p.ho * p.wo < (1LL << 31);
  if (int rc = aligned ? launch_aligned(ksize, stride, a, p, st) : launch_any(ksize, stride, a, p, st)) return rc;
  const long long total = (long long)out_channels * cin * p.taps + out_channels;
  const dim3 grid((unsigned)((total + 63) / 64 < 16384 ? (total + 63) / 64 : 16384));
#define REDUCE(WAVES) hipLaunchKernelGGL(wgrad_ckpt_reduce_kernel<WAVES>, grid, dim3(64 * WAVES), 0, st, scratch, grad_weight, p.slabs, p.nsplit, \
                                         p.taps, out_channels, cin, p.cout_pad, p.cin_pad, a.bias_partial, grad_bias)
  if (p.slabs >= 64) REDUCE(16);
  else REDUCE(4);
#undef REDUCE
  return dvc::check_launch("wgrad_ckpt_reduce_kernel");
}
