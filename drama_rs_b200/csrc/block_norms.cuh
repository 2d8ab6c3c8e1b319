// drb_block_norms: what lies between two blocks, in one pass over the rows.
//
//   t  = rmsnorm(o) * post_w                      (o itself without post_w)
//   x' = alpha * x + sigmoid(gate[row]) * scale[c] * t
//   h  = rmsnorm(x') * pre_w
//
// Every value is read once and stays in registers through both norms; sums of squares in fp32, by thread, then a butterfly, then the
// warps in order, so a row's result does not depend on how many rows there are. Bound by HBM for many rows (4 + 4 bytes of x a value
// beside o and h), by the launch and two block-wide sums for few. Queued: 8192 rows of 2048 33.9 us (5.9 TB/s, 0.91 of a copy's rate; rows through registers,
// one ahead, 40.8), 300 rows 3.6, one row 2.4; 777 rows of 1501, whose values are loaded one by one, 8.5: two such rows in 96 registers spill 124 to 152 bytes. Beyond 2048 columns a
// multiprocessor has one block: 1500 rows of 8192 29.0, 3000 of 4096 32.0, 6000 of 2052 46.2 (22.5 us of bytes each), 6000 of 2049, one by one, 134.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace bn {

constexpr int MAX_D = 8192;  // sixteen values a thread
constexpr int MAX_ROWS = 1 << 30;  // a block looks a few thousand rows ahead: no row number passes 31 bits
constexpr int BLOCKS = 5;    // of 128 threads a multiprocessor
constexpr int depth(int maxt) { return maxt == 128 ? 4 : 3; }  // rows under way and in use
constexpr int SMEM_MAX = 220 * 1024;  // of a multiprocessor, beside what the system takes of it
enum Type { F32 = 0, BF16 = 1, F16 = 2 };

struct Args {
  const void* o;
  const float *post_w, *gate, *scale, *x, *pre_w;
  float* x_out;
  void* h;
  int d;
  float alpha, eps;
};

DRB_DEV float clamp_f16(float v) { return v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v; }  // a NaN stays one

template <int TYPE>
DRB_DEV float2 widen(uint32_t w) {
  return TYPE == BF16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int TYPE>
DRB_DEV uint32_t narrow(float lo, float hi) {
  if (TYPE == BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(clamp_f16(lo), clamp_f16(hi));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The block's sum of v in every thread: butterfly, then the warps in fours. `red` is one value per warp, zeros behind the last.
DRB_DEV float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (int)blockDim.x; w += 128) {
    const float4 q = *reinterpret_cast<const float4*>(red + (w >> 5));
    s += (q.x + q.y) + (q.z + q.w);
  }
  return s;
}

// Sixteen values of a row a thread: four times four consecutive ones (WIDE: 16- and 8-byte accesses next to one another, d a multiple of 4 and
// every pointer aligned), or every blockDim-th one for any other row. A block keeps its part of the weights in registers and goes
// through rows blockIdx, + gridDim, ...; the next rows (WIDE: three, through shared memory; else one, in registers) are requested before the
// current one's sums, so that the stream does not wait for them. (Eight values a thread took two thirds longer over the sums: as many shuffles and barriers for half the values.)
constexpr int V = 16;
template <bool WIDE>
struct Cols {
  int c0, step, d;
  DRB_DEV Cols(int d) : c0(threadIdx.x * (WIDE ? 4 : 1)), step(blockDim.x * (WIDE ? 4 : 1)), d(d) {}
  // value j lies in column at(j); WIDE: values 4 i .. 4 i + 3 are in the row together
  DRB_DEV int at(int j) const { return WIDE ? c0 + (j >> 2) * step + (j & 3) : c0 + j * step; }
  DRB_DEV bool in(int j) const { return at(j) < d; }
  DRB_DEV void load(const float* p, float (&v)[V]) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        if (in(j)) {
          const float4 a = __ldcg(reinterpret_cast<const float4*>(p + at(j)));
          v[j] = a.x, v[j + 1] = a.y, v[j + 2] = a.z, v[j + 3] = a.w;
        }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (in(j)) v[j] = __ldcg(p + at(j));
    }
  }
  DRB_DEV void store(float* p, const float (&v)[V]) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        if (in(j)) *reinterpret_cast<float4*>(p + at(j)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (in(j)) p[at(j)] = v[j];
    }
  }
  // 16-bit values stay as they are until they are used: w[j] holds values 2 j and 2 j + 1
  DRB_DEV void load16(const uint16_t* p, uint32_t (&w)[V / 2]) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        if (in(j)) {
          const uint2 a = __ldcg(reinterpret_cast<const uint2*>(p + at(j)));
          w[j / 2] = a.x, w[j / 2 + 1] = a.y;
        }
    } else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const uint32_t lo = in(2 * j) ? __ldcg(p + at(2 * j)) : 0u, hi = in(2 * j + 1) ? __ldcg(p + at(2 * j + 1)) : 0u;
        w[j] = lo | hi << 16;
      }
    }
  }
  template <int TYPE>
  DRB_DEV void store16(uint16_t* p, const float (&v)[V]) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        if (in(j)) *reinterpret_cast<uint2*>(p + at(j)) = make_uint2(narrow<TYPE>(v[j], v[j + 1]), narrow<TYPE>(v[j + 2], v[j + 3]));
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const uint32_t w = narrow<TYPE>(v[j], v[j + 1]);
        if (in(j)) p[at(j)] = (uint16_t)w;
        if (in(j + 1)) p[at(j + 1)] = (uint16_t)(w >> 16);
      }
    }
  }
};

template <bool WIDE, int OT, int HT, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? BLOCKS : 1) k_block_norms(Args a, int rows) {
  __shared__ __align__(16) float red[2][32];
  constexpr int OSIZE = OT == F32 ? 16 : 8;  // bytes of four values of o
  constexpr int DEPTH = MAXT == 128 ? 4 : 3;
  const int d = a.d;
  const Cols<WIDE> cols(d);
  if (threadIdx.x < 64) red[0][threadIdx.x] = 0.f;  // a block has 32 threads at least
  if (blockDim.x == 32) red[1][threadIdx.x] = 0.f;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  float xn[V] = {}, on[V] = {}, gn = 0.f;  // !WIDE: the next row
  uint32_t hn[V / 2] = {};
  extern __shared__ __align__(16) unsigned char ring[];
  auto fetch = [&](int row) {
    const size_t at = (size_t)row * d;
    cols.load(a.x + at, xn);
    if constexpr (OT != F32) cols.load16(static_cast<const uint16_t*>(a.o) + at, hn);
    else cols.load(static_cast<const float*>(a.o) + at, on);
  };
  // WIDE: rows on their way into DEPTH slots of shared memory, where every thread finds what it copied itself: no barrier, no registers
  const uint32_t slots = smem_u32(ring) + 16 * threadIdx.x, pitch = 16 * blockDim.x, oslots = smem_u32(ring) + 4 * pitch + OSIZE * threadIdx.x;
  const uint32_t opitch = OSIZE * blockDim.x, slot_bytes = 4 * (pitch + opitch);
  auto request = [&](int row, int slot) {
    if (row < rows) {
      const float* x = a.x + (size_t)row * d;
      const unsigned char* o = static_cast<const unsigned char*>(a.o) + (size_t)row * d * (OSIZE / 4);
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        if (cols.in(4 * i)) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slots + slot * slot_bytes + i * pitch), "l"(x + cols.at(4 * i)) : "memory");
          if constexpr (OT == F32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(oslots + slot * slot_bytes + i * opitch), "l"(o + 4 * (size_t)cols.at(4 * i)) : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(oslots + slot * slot_bytes + i * opitch), "l"(o + 2 * (size_t)cols.at(4 * i)) : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (WIDE) {
#pragma unroll
    for (int k = 0; k < DEPTH - 1; ++k) request(blockIdx.x + k * gridDim.x, k);
  } else {
    fetch(blockIdx.x);
  }
  if (a.gate) gn = __ldcg(a.gate + blockIdx.x);
  float wt[V], wn[V] = {};  // post_w * scale, pre_w
  {
    float w[V], s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = s[j] = 1.f;
    if (a.post_w) cols.load(a.post_w, w);
    if (a.scale) cols.load(a.scale, s);
    if (a.pre_w) cols.load(a.pre_w, wn);
#pragma unroll
    for (int j = 0; j < V; ++j) wt[j] = w[j] * s[j];
  }
  int slot = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const size_t at = (size_t)row * d;
    float x[V], t[V];
    const float gate = gn;
    const bool more = row + (int)gridDim.x < rows;
    if (a.gate && more) gn = __ldcg(a.gate + row + gridDim.x);
    if constexpr (WIDE) {
      request(row + (DEPTH - 1) * gridDim.x, slot == 0 ? DEPTH - 1 : slot - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u = v;
        if (cols.in(4 * i)) {
          v = *static_cast<const float4*>(__cvta_shared_to_generic(slots + slot * slot_bytes + i * pitch));
          const uint32_t q = oslots + slot * slot_bytes + i * opitch;
          if constexpr (OT == F32) {
            u = *static_cast<const float4*>(__cvta_shared_to_generic(q));
          } else {
            const uint2 w = *static_cast<const uint2*>(__cvta_shared_to_generic(q));
            const float2 lo = widen<OT>(w.x), hi = widen<OT>(w.y);
            u = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
        }
        x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        t[4 * i] = u.x, t[4 * i + 1] = u.y, t[4 * i + 2] = u.z, t[4 * i + 3] = u.w;
      }
      if (++slot == DEPTH) slot = 0;
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        x[j] = xn[j], x[j + 1] = xn[j + 1];
        const float2 v = OT == F32 ? make_float2(on[j], on[j + 1]) : widen<OT>(hn[j / 2]);
        t[j] = v.x, t[j + 1] = v.y;
      }
      if (more) fetch(row + gridDim.x);
    }
    float f = 1.f;
    if (a.post_w) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(t[j], t[j], ss);
      f = rsqrtf(block_sum(ss, red[0]) / (float)d + a.eps);
    }
    if (a.gate) f *= sigmoid_f(gate);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = fmaf(f, t[j] * wt[j], a.alpha * x[j]), ss = fmaf(x[j], x[j], ss);
    cols.store(a.x_out + at, x);
    if (a.pre_w) {
      const float r = rsqrtf(block_sum(ss, red[1]) / (float)d + a.eps);
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = x[j] * r * wn[j];
      if constexpr (HT == F32) cols.store(static_cast<float*>(a.h) + at, x);
      else cols.template store16<HT>(static_cast<uint16_t*>(a.h) + at, x);
    }
    // a warp writes its slot of one sum again only behind the other sum's barrier; with one sum a row it has to be kept apart
    if (!a.post_w || !a.pre_w) __syncthreads();
  }
}

// As many blocks as are resident at once go through the rows together.
template <bool WIDE, int OT, int HT, int MAXT>
static void launch(const Args& a, int rows, cudaStream_t st, const DrbDevice& dev) {
  const int threads = ((a.d + V - 1) / V + 31) / 32 * 32, smem = WIDE ? depth(MAXT) * threads * (64 + (OT == F32 ? 64 : 32)) : 0;
  int fit = MAXT == 128 ? BLOCKS * 128 / threads : 1;
  if constexpr (WIDE)
    if (fit > SMEM_MAX / smem) fit = SMEM_MAX / smem;
  drb_launch(k_block_norms<WIDE, OT, HT, MAXT>, dim3(rows < dev.sms * fit ? rows : dev.sms * fit), dim3(threads), smem, st, dev.pdl, a, rows);
}

template <bool WIDE, int OT, int HT, int MAXT>
static cudaError_t configure() {
  if (WIDE) {
    const cudaError_t e = cudaFuncSetAttribute(k_block_norms<WIDE, OT, HT, MAXT>, cudaFuncAttributeMaxDynamicSharedMemorySize, depth(MAXT) * MAXT * 128);
    if (e != cudaSuccess) return e;
  }
  return drb_carveout(k_block_norms<WIDE, OT, HT, MAXT>);
}

// The kernels for every pair of types, as one list for launches and set-up.
template <typename F>
static auto for_types(int o_type, int h_type, F f) {
  using std::integral_constant;
  const auto inner = [&](auto o) {
    return h_type == F32 ? f(o, integral_constant<int, F32>()) : h_type == BF16 ? f(o, integral_constant<int, BF16>()) : f(o, integral_constant<int, F16>());
  };
  return o_type == F32 ? inner(integral_constant<int, F32>()) : o_type == BF16 ? inner(integral_constant<int, BF16>()) : inner(integral_constant<int, F16>());
}

static void launch_any(bool wide, const Args& a, int o_type, int h_type, int rows, cudaStream_t st, const DrbDevice& dev) {
  for_types(o_type, h_type, [&](auto o, auto h) {
    constexpr int OT = decltype(o)::value, HT = decltype(h)::value;
    if (wide) a.d <= 2048 ? launch<true, OT, HT, 128>(a, rows, st, dev) : launch<true, OT, HT, 512>(a, rows, st, dev);
    else a.d <= 2048 ? launch<false, OT, HT, 128>(a, rows, st, dev) : launch<false, OT, HT, 512>(a, rows, st, dev);
    return 0;
  });
}

static cudaError_t configure_all() {
  for (int o = 0; o < 3; ++o)
    for (int h = 0; h < 3; ++h) {
      const cudaError_t e = for_types(o, h, [](auto ot, auto ht) {
        constexpr int OT = decltype(ot)::value, HT = decltype(ht)::value;
        cudaError_t e;
        if ((e = configure<true, OT, HT, 128>()) != cudaSuccess) return e;
        if ((e = configure<true, OT, HT, 512>()) != cudaSuccess) return e;
        if ((e = configure<false, OT, HT, 128>()) != cudaSuccess) return e;
        return configure<false, OT, HT, 512>();
      });
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace bn

extern "C" int drb_block_norms(const void* o, int o_type, const float* post_w, const float* gate, const float* scale, float alpha, const float* x,
                               float* x_out, const float* pre_w, void* h, int h_type, int rows, int d, float eps, cudaStream_t st) {
  if (d < 1 || d > bn::MAX_D || rows < 0 || rows > bn::MAX_ROWS || o_type < 0 || o_type > 2 || h_type < 0 || h_type > 2 || !o || !x || !x_out || (pre_w && !h)) return -1;
  const auto off = [](const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) != 0; };
  // every value lies on a multiple of its own size
  if (off(o, o_type ? 2 : 4) || off(x, 4) || off(x_out, 4) || off(post_w, 4) || off(gate, 4) || off(scale, 4) || off(pre_w, 4) || (pre_w && off(h, h_type ? 2 : 4)))
    return -3;
  const DrbDevice& dev = drb_device(st);
  if (!dev.ready) return -2;
  if (rows == 0) return 0;
  const bn::Args a = {o, post_w, gate, scale, x, pre_w, x_out, h, d, alpha, eps};
  const bool wide = d % 4 == 0 && !off(o, o_type ? 8 : 16) && !off(x, 16) && !off(x_out, 16) && !off(post_w, 16) && !off(scale, 16) && !off(pre_w, 16) && !(pre_w && off(h, h_type ? 8 : 16));
  bn::launch_any(wide, a, o_type, h_type, rows, st, dev);
  return 0;
}
