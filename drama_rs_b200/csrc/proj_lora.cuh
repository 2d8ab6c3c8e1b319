// drb_proj_q8_lora: an int8 projection of several rows, each row's low-rank adapter beside it.
//
//   y_r = W x_r (+ res_r) + scale_a B_a (A_a x_r),  a = adapter_of[r]
//
// Two launches (one without adapters). k_shrink: v_r = scale_a A_a x_r, the adapters' first halves, read once per row that uses them.
// k_proj: the weights' stream. Bound by the bytes of W and of the adapters hit for few rows; from some 64 rows on by mma.sync.
//
// k_proj: 16-bit x meets the int8 codes, which both 16-bit types hold exactly, on mma.sync m16n8k16; a sum over the 128 inputs of a weight
// scale is fp32, scaled in fp32, so no weight is rounded. The 16 weight rows of a tile are M, the rows of x are N (8 to 64 a pass). A
// block keeps its slice of x in shared memory. 64 rows of 2048 inputs would not fit and would cost every multiprocessor 256 KB of L2
// reads, so a cluster of blocks shares the K axis: each holds its slice of x, streams its slice of the cluster's weight rows through
// rings of 16-byte asynchronous copies (one ring a warp, no barrier in a step), and the slices' sums meet through distributed shared
// memory, in rank order.
#pragma once

#include "common.cuh"
#include "moe_few.cuh"

namespace pl {

constexpr int MAX_RANK = 64, MAX_K = 8192;
constexpr int CW = 8, THREADS = CW * 32;
constexpr int SUB = 2048;                  // a step of a warp: 16 weight rows x 128 inputs
constexpr int PP = 20;                     // floats between the columns of a tile of sums: writes of a warp meet no bank twice
constexpr size_t SMEM_MAX = 232448;

struct Args {
  const int8_t* w;
  const __half* s;
  const void* x;
  const __nv_bfloat16 *a, *b;
  const float *scale, *res;
  const int* adapter_of;
  float *y, *v;
  int adapters, rank, rows, n, k;
};

DRB_DEV float widen16(uint32_t b, bool f16) { return f16 ? __half2float(__ushort_as_half((uint16_t)b)) : __uint_as_float(b << 16); }

// ---- v = scale A x ------------------------------------------------------------------------------------------------------
// A block: eight ranks of one row, a warp each.
template <bool F16>
__global__ void __launch_bounds__(256) k_shrink(Args p) {
  const int row = (int)blockIdx.x, j = (int)blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int ad = __ldcg(p.adapter_of + row);
  if (ad < 0 || ad >= p.adapters) return;
  const uint4* xp = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + (size_t)row * p.k) + lane;
  const uint4* ap = reinterpret_cast<const uint4*>(p.a + ((size_t)ad * p.rank + j) * p.k) + lane;
  float acc[2] = {0.f, 0.f};
#pragma unroll 4
  for (int i = lane; i < p.k / 8; i += 32, xp += 32, ap += 32) {
    const uint4 xv = __ldcg(xp), av = __ldg(ap);
    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w}, aw[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      acc[0] = fmaf(widen16(xw[q] & 0xffffu, F16), widen16(aw[q] & 0xffffu, false), acc[0]);
      acc[1] = fmaf(widen16(xw[q] >> 16, F16), widen16(aw[q] >> 16, false), acc[1]);
    }
  }
  const float sum = warp_sum(acc[0] + acc[1]);
  if (lane == 0) p.v[(size_t)row * p.rank + j] = sum * __ldcg(p.scale + ad);
}

// ---- y = W x + res + B v -----------------------------------------------------------------------------------------------
template <bool F16>
DRB_DEV void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four int8 codes as two pairs of 16-bit floats, exactly. fp16: code + 128 below the leading bit of 1024, minus 1152. bf16: the low
// seven bits below the leading bit of 128, minus 128, or minus 256 where the sign bit is set.
template <bool F16>
DRB_DEV void widen_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (F16) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t l = prmt(u, 0x64646464u, 0x4140u), h = prmt(u, 0x64646464u, 0x4342u);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), off), b = __hsub2(*reinterpret_cast<const __half2*>(&h), off);
    lo = *reinterpret_cast<const uint32_t*>(&a), hi = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const uint32_t l = prmt(w, 0x43434343u, 0x4140u), h = prmt(w, 0x43434343u, 0x4342u);
    const uint32_t lm = l & 0xff7fff7fu, hm = h & 0xff7fff7fu;
    const uint32_t ls = lop3_and_or(l, 0x00800080u, 0x43004300u), hs = lop3_and_or(h, 0x00800080u, 0x43004300u);
    const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lm), *reinterpret_cast<const __nv_bfloat162*>(&ls));
    const __nv_bfloat162 b = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&hm), *reinterpret_cast<const __nv_bfloat162*>(&hs));
    lo = *reinterpret_cast<const uint32_t*>(&a), hi = *reinterpret_cast<const uint32_t*>(&b);
  }
}

DRB_DEV unsigned cluster_size() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(v));
  return v;
}
DRB_DEV unsigned cluster_rank() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}
DRB_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
DRB_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
DRB_DEV float ld_peer(uint32_t addr, unsigned rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <int NT>
struct Shape {
  static constexpr int DEPTH = NT == 8 ? 3 : 6;
  static constexpr size_t SUMS = (size_t)CW * 8 * NT * PP * 4;
  static constexpr size_t bytes(int slice) { return (size_t)8 * NT * (2 * slice + 16) + SUMS + (size_t)CW * DEPTH * SUB; }
};
static_assert(Shape<8>::bytes(MAX_K / 8) <= SMEM_MAX && Shape<4>::bytes(MAX_K / 8) <= SMEM_MAX, "eight blocks hold the longest row");

// NT: column tiles (8 rows of x each) of a pass; blockIdx.y: the pass. Cluster c of the pass owns weight tiles [mt c / C, mt (c + 1) / C).
template <bool F16, int NT>
__global__ void __launch_bounds__(THREADS, 1) k_proj(Args p) {
  constexpr int DEPTH = Shape<NT>::DEPTH;
  extern __shared__ __align__(128) unsigned char dyn[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int cs = (int)cluster_size(), cr = (int)cluster_rank(), C = (int)gridDim.x / cs, c = (int)blockIdx.x / cs;
  const int groups = p.k / 128, g0 = groups * cr / cs, ng = groups * (cr + 1) / cs - g0;  // this block's inputs
  const int mt = (p.n + 15) / 16, t0 = (int)((long long)mt * c / C), t1 = (int)((long long)mt * (c + 1) / C);
  const int row0 = (int)blockIdx.y * 8 * NT, cols = min(8 * NT, p.rows - row0);
  const int pitch = 2 * 128 * ((groups + cs - 1) / cs) + 16;
  unsigned char* xs = dyn;
  float* sums = reinterpret_cast<float*>(dyn + (size_t)8 * NT * pitch);
  unsigned char* ring = reinterpret_cast<unsigned char*>(sums) + Shape<NT>::SUMS + warp * DEPTH * SUB;
  pdl_launch_dependents();

  // The weights' stream: tiles t0 + warp, t0 + warp + CW, ..., ng steps each. Rows behind the last one are read as the last one.
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + CW - 1) / CW : 0, steps = mine * ng;
  int nslot = 0, slot = 0, ltile = t0 + warp, lg = 0, left = steps;
  auto issue = [&]() {
    if (left > 0) {
      const uint32_t dst = smem_u32(ring + nslot * SUB);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 3) + 4 * i, q = lane & 7;
        few::cp16(dst + r * 128 + 16 * (q ^ ((r & 1) << 2)), p.w + (size_t)min(16 * ltile + r, p.n - 1) * p.k + (g0 + lg) * 128 + 16 * q);
      }
      --left;
      if (++lg == ng) lg = 0, ltile += CW;
    }
    few::cp_commit();
    if (++nslot == DEPTH) nslot = 0;
  };
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) issue();
  auto scales = [&](int tile, int grp, float& s0, float& s1) {
    s0 = __half2float(__ldg(p.s + (size_t)min(16 * tile + g, p.n - 1) * groups + g0 + grp));
    s1 = __half2float(__ldg(p.s + (size_t)min(16 * tile + g + 8, p.n - 1) * groups + g0 + grp));
  };
  float s0 = 0.f, s1 = 0.f;
  if (steps > 0) scales(t0 + warp, 0, s0, s1);

  pdl_wait();  // x, res, the adapters and v
  {
    const int pieces = ng * 16;  // of 16 bytes a row
    for (int i = threadIdx.x; i < 8 * NT * pieces; i += THREADS) {
      const int r = i / pieces, q = i - r * pieces;
      few::cp16(smem_u32(xs + r * pitch + 16 * q), static_cast<const uint16_t*>(p.x) + (size_t)(row0 + min(r, cols - 1)) * p.k + g0 * 128 + 8 * q);
    }
    few::cp_commit();
    few::cp_wait<0>();
    __syncthreads();
  }

  const int batches = (t1 - t0 + CW - 1) / CW;
  const unsigned char* xb = xs + g * pitch + 32 * t;
  for (int bt = 0; bt < batches; ++bt) {
    const int tile = t0 + bt * CW + warp;
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    if (tile < t1) {
      for (int q = 0; q < ng; ++q) {
        const float f0 = s0, f1 = s1;
        if (q + 1 < ng) scales(tile, q + 1, s0, s1);
        else if (tile + CW < t1) scales(tile + CW, 0, s0, s1);
        few::cp_wait<DEPTH - 1>();
        __syncwarp();
        const unsigned char* r0 = ring + slot * SUB + g * 128;
        float d[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = 64 * (h ^ (g & 1)) + 16 * t;
          const uint4 u = *reinterpret_cast<const uint4*>(r0 + at), v = *reinterpret_cast<const uint4*>(r0 + 8 * 128 + at);
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // inputs 16 t + 8 e .. + 7 of the 64: two multiplications
            uint32_t a[8];
            widen_codes<F16>(uw[2 * e], a[0], a[2]);
            widen_codes<F16>(vw[2 * e], a[1], a[3]);
            widen_codes<F16>(uw[2 * e + 1], a[4], a[6]);
            widen_codes<F16>(vw[2 * e + 1], a[5], a[7]);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const uint4 b = *reinterpret_cast<const uint4*>(xb + (size_t)8 * i * pitch + q * 256 + h * 128 + 16 * e);
              mma16<F16>(d[i], a[0], a[1], a[2], a[3], b.x, b.y);
              mma16<F16>(d[i], a[4], a[5], a[6], a[7], b.z, b.w);
            }
          }
        }
        __syncwarp();
        issue();
        if (++slot == DEPTH) slot = 0;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          acc[i][0] = fmaf(f0, d[i][0], acc[i][0]), acc[i][1] = fmaf(f0, d[i][1], acc[i][1]);
          acc[i][2] = fmaf(f1, d[i][2], acc[i][2]), acc[i][3] = fmaf(f1, d[i][3], acc[i][3]);
        }
      }
    }
    if (bt > 0) cluster_wait();  // everyone has read the batch before
    float* st = sums + warp * 8 * NT * PP;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      st[(8 * i + 2 * t) * PP + g] = acc[i][0], st[(8 * i + 2 * t + 1) * PP + g] = acc[i][1];
      st[(8 * i + 2 * t) * PP + g + 8] = acc[i][2], st[(8 * i + 2 * t + 1) * PP + g + 8] = acc[i][3];
    }
    cluster_arrive();
    cluster_wait();
    // Block cr of the cluster finishes its share of the batch: column r of x, weight row j of tile m.
    const int nt = min(CW, t1 - t0 - bt * CW), outs = nt * 16 * cols;
    for (int i = outs * cr / cs + (int)threadIdx.x; i < outs * (cr + 1) / cs; i += THREADS) {
      const int j = i & 15, m = (i >> 4) % nt, r = (i >> 4) / nt, o = 16 * (t0 + bt * CW + m) + j;
      if (o >= p.n) continue;
      const uint32_t at = smem_u32(sums + (m * 8 * NT + r) * PP + j);
      float v = 0.f;
      for (int q = 0; q < cs; ++q) v += ld_peer(at, (unsigned)q);
      const int row = row0 + r;
      if (p.rank > 0) {
        const int ad = __ldcg(p.adapter_of + row);
        if (ad >= 0 && ad < p.adapters) {
          const uint4* bp = reinterpret_cast<const uint4*>(p.b + ((size_t)ad * p.n + o) * p.rank);
          const float4* vp = reinterpret_cast<const float4*>(p.v + (size_t)row * p.rank);
          float s = 0.f;
          for (int q = 0; q < p.rank / 8; ++q) {
            const uint4 bw = __ldg(bp + q);
            const float4 v0 = __ldcg(vp + 2 * q), v1 = __ldcg(vp + 2 * q + 1);
            s = fmaf(widen16(bw.x & 0xffffu, false), v0.x, s), s = fmaf(widen16(bw.x >> 16, false), v0.y, s);
            s = fmaf(widen16(bw.y & 0xffffu, false), v0.z, s), s = fmaf(widen16(bw.y >> 16, false), v0.w, s);
            s = fmaf(widen16(bw.z & 0xffffu, false), v1.x, s), s = fmaf(widen16(bw.z >> 16, false), v1.y, s);
            s = fmaf(widen16(bw.w & 0xffffu, false), v1.z, s), s = fmaf(widen16(bw.w >> 16, false), v1.w, s);
          }
          v += s;
        }
      }
      const size_t yo = (size_t)row * p.n + o;
      p.y[yo] = p.res ? v + __ldcg(p.res + yo) : v;
    }
    __syncwarp();
    cluster_arrive();
  }
  if (batches > 0) cluster_wait();
  few::cp_wait<0>();
}

// NT column tiles: the smallest form that takes all rows in one pass, 64 rows a pass beyond. Blocks of a cluster share K: more of them for
// longer rows, so that the slice of x fits, and for matrices of so few tiles that the warps of fewer blocks would stand idle.
template <bool F16, int NT>
static int launch(const Args& p, const DrbDevice& dev, cudaStream_t st) {
  const int groups = p.k / 128, mt = (p.n + 15) / 16, passes = (p.rows + 8 * NT - 1) / (8 * NT);
  int cs = 1;
  while (cs < 8 && 2 * cs <= groups && (Shape<NT>::bytes(128 * ((groups + cs - 1) / cs)) > SMEM_MAX || (long long)mt * passes * cs < (long long)CW * dev.sms)) cs *= 2;
  const size_t smem = Shape<NT>::bytes(128 * ((groups + cs - 1) / cs));
  int clusters = dev.sms / cs / passes;
  if (clusters < 1) clusters = 1;
  if (clusters > (mt + CW - 1) / CW) clusters = (mt + CW - 1) / CW;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * cs, passes);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dev.pdl ? 2 : 1;
  cudaLaunchKernelEx(&cfg, k_proj<F16, NT>, p);
  return 0;
}

template <bool F16>
static int launch_any(const Args& p, const DrbDevice& dev, cudaStream_t st) {
  if (p.rank > 0) drb_launch(k_shrink<F16>, dim3(p.rows, p.rank / 8), dim3(256), 0, st, dev.pdl, p);
  if (p.rows <= 8) return launch<F16, 1>(p, dev, st);
  if (p.rows <= 16) return launch<F16, 2>(p, dev, st);
  if (p.rows <= 32) return launch<F16, 4>(p, dev, st);
  return launch<F16, 8>(p, dev, st);
}

template <bool F16, int NT>
static cudaError_t configure() {
  const cudaError_t e = cudaFuncSetAttribute(k_proj<F16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX);
  return e != cudaSuccess ? e : drb_carveout(k_proj<F16, NT>);
}
template <bool F16>
static cudaError_t configure_type() {
  cudaError_t e;
  if ((e = configure<F16, 1>()) != cudaSuccess) return e;
  if ((e = configure<F16, 2>()) != cudaSuccess) return e;
  if ((e = configure<F16, 4>()) != cudaSuccess) return e;
  if ((e = configure<F16, 8>()) != cudaSuccess) return e;
  return drb_carveout(k_shrink<F16>);
}
static cudaError_t configure_all() {
  const cudaError_t e = configure_type<false>();
  return e != cudaSuccess ? e : configure_type<true>();
}

}  // namespace pl

extern "C" int drb_proj_q8_lora(const int8_t* w, const __half* s, const void* x, int x_type, const __nv_bfloat16* a, const __nv_bfloat16* b,
                                const float* scale, const int* adapter_of, int adapters, int rank, const float* res, float* y, float* v, int rows, int n,
                                int k, cudaStream_t st) {
  if ((x_type != 1 && x_type != 2) || rows < 0 || n < 1 || k < 128 || k > pl::MAX_K || k % 128 || rank < 0 || rank > pl::MAX_RANK || rank % 8 || adapters < 0)
    return -1;
  if (!w || !s || !x || !y || (rank > 0 && (!a || !b || !scale || !adapter_of || !v))) return -1;
  const auto off = [](const void* p, unsigned m) { return ((uintptr_t)p & (m - 1)) != 0; };
  if (off(w, 16) || off(s, 2) || off(x, 16) || off(y, 4) || off(res, 4)) return -3;
  if (rank > 0 && (off(a, 16) || off(b, 16) || off(v, 16) || off(scale, 4) || off(adapter_of, 4))) return -3;
  const DrbDevice& dev = drb_device(st);
  if (!dev.ready) return -2;
  if (rows == 0) return 0;
  if (rows > 65535 * 64) return -1;
  const pl::Args p = {w, s, x, a, b, scale, res, adapter_of, y, v, adapters, adapters > 0 ? rank : 0, rows, n, k};
  return x_type == 2 ? pl::launch_any<true>(p, dev, st) : pl::launch_any<false>(p, dev, st);
}
