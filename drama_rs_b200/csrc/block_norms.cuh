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

constexpr int MAX_D = 8192;
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

// A block per row. Thread t holds VEC consecutive values at (t + i * threads) * VEC, i < NCH. VEC = 8: 16-byte accesses, d a multiple
// of 8 and every pointer aligned; VEC = 1 for any other row.
template <int VEC, int NCH>
__global__ void __launch_bounds__(VEC == 8 ? 256 : 1024) k_block_norms(Args a) {
  __shared__ float red[2][32];
  const int d = a.d, step = (int)blockDim.x * VEC, c0 = (int)threadIdx.x * VEC;
  const size_t row = (size_t)blockIdx.x * d;
  pdl_launch_dependents();
  pdl_wait();
  float t[NCH][VEC], x[NCH][VEC];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = c0 + i * step;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t[i][j] = 0.f, x[i][j] = 0.f;
    if (c >= d) continue;
    if constexpr (VEC == 8) {
      const float4* xp = reinterpret_cast<const float4*>(a.x + row + c);
      const float4 x0 = __ldcg(xp), x1 = __ldcg(xp + 1);
      x[i][0] = x0.x, x[i][1] = x0.y, x[i][2] = x0.z, x[i][3] = x0.w, x[i][4] = x1.x, x[i][5] = x1.y, x[i][6] = x1.z, x[i][7] = x1.w;
      if (a.o_type == F32) {
        const float4* op = reinterpret_cast<const float4*>(static_cast<const float*>(a.o) + row + c);
        const float4 o0 = __ldcg(op), o1 = __ldcg(op + 1);
        t[i][0] = o0.x, t[i][1] = o0.y, t[i][2] = o0.z, t[i][3] = o0.w, t[i][4] = o1.x, t[i][5] = o1.y, t[i][6] = o1.z, t[i][7] = o1.w;
      } else {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.o) + row + c));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) t[i][2 * j] = widen((uint16_t)w[j], a.o_type), t[i][2 * j + 1] = widen((uint16_t)(w[j] >> 16), a.o_type);
      }
    } else {
      x[i][0] = __ldcg(a.x + row + c);
      t[i][0] = a.o_type == F32 ? __ldcg(static_cast<const float*>(a.o) + row + c)
                                : widen(__ldcg(static_cast<const uint16_t*>(a.o) + row + c), a.o_type);
    }
  }
  float f = 1.f;
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss = fmaf(t[i][j], t[i][j], ss);
    f = rsqrtf(block_sum(ss, red[0]) / (float)d + a.eps);
  }
  if (a.gate) f *= sigmoid_f(__ldcg(a.gate + blockIdx.x));
  auto weights = [&](const float* w, int c, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
      const float4 w0 = __ldcg(reinterpret_cast<const float4*>(w + c)), w1 = __ldcg(reinterpret_cast<const float4*>(w + c) + 1);
      v[0] = w0.x, v[1] = w0.y, v[2] = w0.z, v[3] = w0.w, v[4] = w1.x, v[5] = w1.y, v[6] = w1.z, v[7] = w1.w;
    } else {
      v[0] = __ldcg(w + c);
    }
  };
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = c0 + i * step;
    if (c >= d) continue;
    float w[VEC];
    if (a.post_w) {
      weights(a.post_w, c, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) t[i][j] *= w[j];
    }
    if (a.scale) {
      weights(a.scale, c, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) t[i][j] *= w[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[i][j] = fmaf(f, t[i][j], a.alpha * x[i][j]), ss = fmaf(x[i][j], x[i][j], ss);
    if constexpr (VEC == 8) {
      float4* xp = reinterpret_cast<float4*>(a.x_out + row + c);
      xp[0] = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      xp[1] = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
    } else {
      a.x_out[row + c] = x[i][0];
    }
  }
  if (!a.pre_w) return;
  const float r = rsqrtf(block_sum(ss, red[1]) / (float)d + a.eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = c0 + i * step;
    if (c >= d) continue;
    float w[VEC];
    weights(a.pre_w, c, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] = x[i][j] * r * w[j];
    if constexpr (VEC == 8) {
      if (a.h_type == F32) {
        float4* hp = reinterpret_cast<float4*>(static_cast<float*>(a.h) + row + c);
        hp[0] = make_float4(w[0], w[1], w[2], w[3]);
        hp[1] = make_float4(w[4], w[5], w[6], w[7]);
      } else {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = (uint32_t)narrow(w[2 * j], a.h_type) | (uint32_t)narrow(w[2 * j + 1], a.h_type) << 16;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.h) + row + c) = make_uint4(p[0], p[1], p[2], p[3]);
      }
    } else {
      if (a.h_type == F32) static_cast<float*>(a.h)[row + c] = w[0];
      else static_cast<uint16_t*>(a.h)[row + c] = narrow(w[0], a.h_type);
    }
  }
}

template <int VEC, int NCH>
static void launch(const Args& a, int rows, cudaStream_t st, bool pdl) {
  const int threads = ((a.d + VEC * NCH - 1) / (VEC * NCH) + 31) / 32 * 32;
  drb_launch(k_block_norms<VEC, NCH>, dim3(rows), dim3(threads), 0, st, pdl, a);
}

static cudaError_t configure_all() {
  cudaError_t e;
  if ((e = drb_carveout(k_block_norms<8, 1>)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_block_norms<8, 2>)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_block_norms<8, 4>)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_block_norms<1, 2>)) != cudaSuccess) return e;
  return drb_carveout(k_block_norms<1, 8>);
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
  if (wide) {
    if (d <= 2048) bn::launch<8, 1>(a, rows, st, dev.pdl);
    else if (d <= 4096) bn::launch<8, 2>(a, rows, st, dev.pdl);
    else bn::launch<8, 4>(a, rows, st, dev.pdl);
  } else if (d <= 2048) {
    bn::launch<1, 2>(a, rows, st, dev.pdl);
  } else {
    bn::launch<1, 8>(a, rows, st, dev.pdl);
  }
  return 0;
}
