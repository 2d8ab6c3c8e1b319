// drb_block_norms: what lies between two blocks, in one pass over the rows.
//
//   t  = rmsnorm(o) * post_w                      (o itself without post_w)
//   x' = alpha * x + sigmoid(gate[row]) * scale[c] * t
//   h  = rmsnorm(x') * pre_w
//
// Every value is read once and stays in registers through both norms; sums of squares in fp32, by thread, then a butterfly, then the
// warps in order, so a row's result does not depend on how many rows there are. Bound by HBM for many rows (4 + 4 bytes of x a value
// beside o and h), by the launch and two block-wide sums for few.
#pragma once

#include "common.cuh"


namespace bn {

constexpr int MAX_D = 8192;  // eight values a thread
enum Type { F32 = 0, BF16 = 1, F16 = 2 };

struct Args {
  const void* o;
  const float *post_w, *gate, *scale, *x, *pre_w;
  float* x_out;
  void* h;
  int o_type, h_type, d;
  float alpha, eps;
};

DRB_DEV float clamp_f16(float v) { return v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v; }  // a NaN stays one

DRB_DEV float widen(uint16_t b, int type) {
  return type == BF16 ? __uint_as_float((uint32_t)b << 16) : __half2float(__ushort_as_half(b));
}
DRB_DEV uint16_t narrow(float v, int type) {
  return type == BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(clamp_f16(v)));
}

// The block's sum of v in every thread; `red` holds one value per warp and is used once.
DRB_DEV float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

// Eight values of a row a thread: eight consecutive ones (WIDE: 16-byte accesses, d a multiple of 8 and every pointer aligned), or every
// blockDim-th one for any other row. A block keeps its part of the weights in registers and goes through rows blockIdx, + gridDim, ...; the
// next row is requested before the current one's sums, so that the stream does not wait for them.
template <bool WIDE>
struct Cols {
  int c0, step, d;
  DRB_DEV Cols(int d) : c0(threadIdx.x * (WIDE ? 8 : 1)), step(WIDE ? 1 : blockDim.x), d(d) {}
  DRB_DEV bool in(int j) const { return WIDE ? c0 < d : c0 + j * step < d; }
  DRB_DEV void load(const float* p, float (&v)[8]) const {
    if constexpr (WIDE) {
      if (!in(0)) return;
      const float4 a = __ldcg(reinterpret_cast<const float4*>(p + c0)), b = __ldcg(reinterpret_cast<const float4*>(p + c0) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (in(j)) v[j] = __ldcg(p + c0 + j * step);
    }
  }
  DRB_DEV void store(float* p, const float (&v)[8]) const {
    if constexpr (WIDE) {
      if (!in(0)) return;
      reinterpret_cast<float4*>(p + c0)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p + c0)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (in(j)) p[c0 + j * step] = v[j];
    }
  }
  // 16-bit values stay as they are until they are used: w[j] holds values 2 j and 2 j + 1
  DRB_DEV void load16(const uint16_t* p, uint32_t (&w)[4]) const {
    if constexpr (WIDE) {
      if (!in(0)) return;
      const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p + c0));
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = in(2 * j) ? __ldcg(p + c0 + 2 * j * step) : 0u, hi = in(2 * j + 1) ? __ldcg(p + c0 + (2 * j + 1) * step) : 0u;
        w[j] = lo | hi << 16;
      }
    }
  }
  DRB_DEV void store16(uint16_t* p, const float (&v)[8], int type) const {
    if constexpr (WIDE) {
      if (!in(0)) return;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)narrow(v[2 * j], type) | (uint32_t)narrow(v[2 * j + 1], type) << 16;
      *reinterpret_cast<uint4*>(p + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (in(j)) p[c0 + j * step] = narrow(v[j], type);
    }
  }
};

template <bool WIDE, bool O16, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? 3 : 1) k_block_norms(Args a, int rows) {
  __shared__ float red[2][32];
  const int d = a.d;
  const Cols<WIDE> cols(d);
  pdl_launch_dependents();
  pdl_wait();
  float xn[8] = {}, on[8] = {}, gn = 0.f;
  uint32_t hn[4] = {};
  auto fetch = [&](int row) {
    const size_t at = (size_t)row * d;
    cols.load(a.x + at, xn);
    if constexpr (O16) cols.load16(static_cast<const uint16_t*>(a.o) + at, hn);
    else cols.load(static_cast<const float*>(a.o) + at, on);
    if (a.gate) gn = __ldcg(a.gate + row);
  };
  fetch(blockIdx.x);
  float wt[8], wn[8] = {};  // post_w * scale, pre_w
  {
    float w[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = s[j] = 1.f;
    if (a.post_w) cols.load(a.post_w, w);
    if (a.scale) cols.load(a.scale, s);
    if (a.pre_w) cols.load(a.pre_w, wn);
#pragma unroll
    for (int j = 0; j < 8; ++j) wt[j] = w[j] * s[j];
  }
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const size_t at = (size_t)row * d;
    float x[8], t[8];
    const float gate = gn;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = xn[j];
      if constexpr (O16) t[j] = widen((uint16_t)(hn[j / 2] >> (j & 1 ? 16 : 0)), a.o_type);
      else t[j] = on[j];
    }
    if (row + (int)gridDim.x < rows) fetch(row + gridDim.x);
    float f = 1.f;
    if (a.post_w) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(t[j], t[j], ss);
      f = rsqrtf(block_sum(ss, red[0]) / (float)d + a.eps);
    }
    if (a.gate) f *= sigmoid_f(gate);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(f, t[j] * wt[j], a.alpha * x[j]), ss = fmaf(x[j], x[j], ss);
    cols.store(a.x_out + at, x);
    if (a.pre_w) {
      const float r = rsqrtf(block_sum(ss, red[1]) / (float)d + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * wn[j];
      if (a.h_type == F32) cols.store(static_cast<float*>(a.h) + at, x);
      else cols.store16(static_cast<uint16_t*>(a.h) + at, x, a.h_type);
    }
    // a warp writes its slot of one sum again only behind the other sum's barrier; with one sum a row it has to be kept apart
    if (!a.post_w || !a.pre_w) __syncthreads();
  }
}

// As many blocks as are resident at once go through the rows together.
template <bool WIDE, bool O16, int MAXT>
static void launch(const Args& a, int rows, cudaStream_t st, const DrbDevice& dev) {
  const int threads = ((a.d + 7) / 8 + 31) / 32 * 32;
  const int fit = dev.sms * (MAXT == 256 ? 768 / threads : 1);
  drb_launch(k_block_norms<WIDE, O16, MAXT>, dim3(rows < fit ? rows : fit), dim3(threads), 0, st, dev.pdl, a, rows);
}

template <bool WIDE, bool O16>
static void launch_any(const Args& a, int rows, cudaStream_t st, const DrbDevice& dev) {
  if (a.d <= 2048) launch<WIDE, O16, 256>(a, rows, st, dev);
  else if (a.d <= 4096) launch<WIDE, O16, 512>(a, rows, st, dev);
  else launch<WIDE, O16, 1024>(a, rows, st, dev);
}

template <bool WIDE, bool O16>
static cudaError_t configure() {
  cudaError_t e;
  if ((e = drb_carveout(k_block_norms<WIDE, O16, 256>)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_block_norms<WIDE, O16, 512>)) != cudaSuccess) return e;
  return drb_carveout(k_block_norms<WIDE, O16, 1024>);
}
static cudaError_t configure_all() {
  cudaError_t e;
  if ((e = configure<true, true>()) != cudaSuccess) return e;
  if ((e = configure<true, false>()) != cudaSuccess) return e;
  if ((e = configure<false, true>()) != cudaSuccess) return e;
  return configure<false, false>();
}

}  // namespace bn

extern "C" int drb_block_norms(const void* o, int o_type, const float* post_w, const float* gate, const float* scale, float alpha, const float* x,
                               float* x_out, const float* pre_w, void* h, int h_type, int rows, int d, float eps, cudaStream_t st) {
  if (d < 1 || d > bn::MAX_D || rows < 0 || o_type < 0 || o_type > 2 || h_type < 0 || h_type > 2 || !o || !x || !x_out || (pre_w && !h)) return -1;
  const auto off = [](const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) != 0; };
  // every value lies on a multiple of its own size
  if (off(o, o_type ? 2 : 4) || off(x, 4) || off(x_out, 4) || off(post_w, 4) || off(gate, 4) || off(scale, 4) || off(pre_w, 4) || (pre_w && off(h, h_type ? 2 : 4)))
    return -3;
  const DrbDevice& dev = drb_device(st);
  if (!dev.ready) return -2;
  if (rows == 0) return 0;
  const bn::Args a = {o, post_w, gate, scale, x, pre_w, x_out, h, o_type, h_type, d, alpha, eps};
  const bool wide = d % 8 == 0 && !off(o, 16) && !off(x, 16) && !off(x_out, 16) && !off(post_w, 16) && !off(scale, 16) && !off(pre_w, 16) && !(pre_w && off(h, 16));
  if (wide) o_type ? bn::launch_any<true, true>(a, rows, st, dev) : bn::launch_any<true, false>(a, rows, st, dev);
  else o_type ? bn::launch_any<false, true>(a, rows, st, dev) : bn::launch_any<false, false>(a, rows, st, dev);
  return 0;
}
