// drb_proj_q8_lora: an int8 projection of several rows, each row's low-rank adapter beside it.
//
//   y_r = W x_r (+ res_r) + scale_a B_a (A_a x_r),  a = adapter_of[r]
//
// Two launches (one without adapters). v_r = scale_a A_a x_r: k_shrink, a warp a dot product, or k_shrink_rows, sixteen rows a block on
// the tensor cores. Then the weights' stream, with the adapters' second half on its sums: k_proj behind the first, or, for many rows of few adapters or wide W (the rule and its
// measurements: pr::many), k_proj_rows (tcgen05) behind the second.
// Bound by the bytes of W and of the adapters hit for few rows, by the conversion of the codes for many.
//
// k_proj: 16-bit x meets the int8 codes, which both 16-bit types hold exactly, on mma.sync m16n8k16; a sum over the 128 inputs of a weight
// scale is fp32, scaled in fp32, so no weight is rounded. The 16 weight rows of a tile are M, the rows of x are N (8 to 32 a pass). A
// block keeps its slice of x in shared memory. 32 rows of 2048 inputs would cost every multiprocessor 128 KB of L2 reads, so a cluster
// of blocks shares the K axis: each holds its slice of x, streams its slice of the cluster's weight rows through rings of 16-byte
// asynchronous copies (one ring a warp, no barrier in a step), and the slices' sums meet through distributed shared memory, in rank
// order. The weights' first steps are requested before the launch before has ended, and x is read and multiplied while k_shrink still
// runs: k_shrink lets this kernel in behind its own wait, so what came before k_shrink is complete.
//
// Queued (without adapters in brackets): 1 row of 2048 x 4096 7.2 us (5.4), 17 rows of 8192 x 2048 14.6 (8.8), 64 rows of 4096 x 2048 and as many adapters 17.6
// (10.9). A step of 17 rows takes 0.8 us, of which mma.sync, conversion and reads of shared memory would each take half alone; no unit is busy for more than 0.4 of
// the time, so what bounds it is a warp's way through its step, one after another with three slots. A pass takes up to 32 rows.
#pragma once

#include "common.cuh"
#include "moe_few.cuh"

namespace pl {

constexpr int MAX_RANK = 64, MAX_K = 8192;
constexpr int CW = 8, THREADS = CW * 32;
constexpr int SUB = 2048;                  // a step of a warp: 16 weight rows x 128 inputs
constexpr int DEPTH = 3;
constexpr int PP = 20;                     // floats between the columns of a tile of sums: writes of a warp meet no bank twice
constexpr size_t SMEM_MAX = 232448, SMEM_TWO = 113 * 1024;  // up to the second, two blocks share a multiprocessor

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
DRB_DEV int adapter(const Args& p, int row) {  // -1: none
  const int a = __ldcg(p.adapter_of + row);
  return a >= 0 && a < p.adapters ? a : -1;
}

// ---- v = scale A x ------------------------------------------------------------------------------------------------------
// A block: eight ranks of one row, a warp each. Up to SK inputs of x and of the eight rows of A come by asynchronous copies at once: plain loads
// are few lines at a time beside the largest shared memory, and their registers kept blocks of k_proj off the multiprocessor.
constexpr int SK = 4096;
static int shrink_bytes(int k) { return 9 * 2 * (k < SK ? k : SK); }
template <bool F16>
__global__ void __launch_bounds__(256, 6) k_shrink(Args p) {
  extern __shared__ __align__(128) unsigned char dyn[];
  const int row = (int)blockIdx.x, warp = threadIdx.x >> 5, j = (int)blockIdx.y * 8 + warp, lane = threadIdx.x & 31;
  const int most = min(p.k, SK);
  const uint32_t xs = smem_u32(dyn), as = xs + 2 * most * (1 + warp);
  const uint16_t* xp = static_cast<const uint16_t*>(p.x) + (size_t)row * p.k;
  pdl_wait();
  pdl_launch_dependents();  // behind the wait: see above
  auto load_x = [&](int k0) {
    for (int i = threadIdx.x; i < min(SK, p.k - k0) / 8; i += 256) few::cp16(xs + 16 * i, xp + k0 + 8 * i);
  };
  load_x(0);
  const int ad = adapter(p, row);
  if (ad < 0) {
    few::cp_commit();
    few::cp_wait<0>();
    return;
  }
  const __nv_bfloat16* ap = p.a + ((size_t)ad * p.rank + j) * p.k;
  const float scale = __ldcg(p.scale + ad);
  float acc[2] = {0.f, 0.f};
  for (int k0 = 0; k0 < p.k; k0 += SK) {
    if (k0 > 0) {
      __syncthreads();
      load_x(k0);
    }
    const int n = min(SK, p.k - k0) / 8;
    for (int i = lane; i < n; i += 32) few::cp16(as + 16 * i, ap + k0 + 8 * i);
    few::cp_commit();
    few::cp_wait<0>();
    __syncthreads();
#pragma unroll 4
    for (int i = lane; i < n; i += 32) {
      const uint4 xv = few::lds<uint4>(xs + 16 * i), av = few::lds<uint4>(as + 16 * i);
      const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w}, aw[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[0] = fmaf(widen16(xw[e] & 0xffffu, F16), widen16(aw[e] & 0xffffu, false), acc[0]);
        acc[1] = fmaf(widen16(xw[e] >> 16, F16), widen16(aw[e] >> 16, false), acc[1]);
      }
    }
  }
  const float sum = warp_sum(acc[0] + acc[1]);
  if (lane == 0) p.v[(size_t)row * p.rank + j] = sum * scale;
}

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

// Sums of bf16 numbers. An infinity less its first term is a NaN; the minimum of that and the largest rest that a finite number leaves is the latter, and infinity
// and any finite rest add up to the infinity (set to zero by comparisons: 300 fp16 rows 19.2 -> 20.2 us).

// Two f16 numbers as the sum of two pairs of bf16 numbers, exactly (eleven bits; eight and the rest).
DRB_DEV void split_f16(uint32_t h, uint32_t& hi, uint32_t& lo) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y);
  const __nv_bfloat162 b = __hmin2(__floats2bfloat162_rn(f.x - __low2float(a), f.y - __high2float(a)), __float2bfloat162_rn(128.f));
  hi = *reinterpret_cast<const uint32_t*>(&a), lo = *reinterpret_cast<const uint32_t*>(&b);
}

// Four fp32 numbers as pairs of bf16 numbers in three terms (eight bits each, the third rounded).
DRB_DEV void split3(const float4& v, uint32_t (&b0)[3], uint32_t (&b1)[3]) {
  float4 r = v;
#pragma unroll
  for (int l = 0; l < 3; ++l) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(r.x, r.y), c = __floats2bfloat162_rn(r.z, r.w);
    b0[l] = *reinterpret_cast<const uint32_t*>(&a), b1[l] = *reinterpret_cast<const uint32_t*>(&c);
    r = make_float4(r.x - __low2float(a), r.y - __high2float(a), r.z - __low2float(c), r.w - __high2float(c));
    if (l == 0) r = make_float4(fminf(r.x, 0x1p119f), fminf(r.y, 0x1p119f), fminf(r.z, 0x1p119f), fminf(r.w, 0x1p119f));
  }
}

// A block: eight ranks of sixteen rows, every adapter among them in turn; each of the eight warps an eighth of the inputs, 64 at a time.
// Rows are M, ranks are N; fp16 rows meet the bf16 adapters as two bf16 terms. x and A come by asynchronous copies of whole lines into
// a ring of each warp's own (fragments straight from L2 are half lines, and beside the largest shared memory few lines of loads are under way at once:
// 2 us for 64 inputs a warp). 256 threads of 64 registers and 52 KB are what a multiprocessor has left beside a block of k_proj_rows, which starts
// while this kernel runs.
constexpr int SH_STAGE = 24 * 128, SH_DEPTH = 2, SH_BYTES = 8 * SH_DEPTH * SH_STAGE;
template <bool F16>
__global__ void __launch_bounds__(256, 4) k_shrink_rows(Args p) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ float part[8][16][8];
  const int row0 = (int)blockIdx.x * 16, j0 = (int)blockIdx.y * 8, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rows = min(16, p.rows - row0);
  pdl_wait();
  pdl_launch_dependents();
  const int who = lane < rows ? adapter(p, row0 + lane) : -1;  // lane r: of row r
  const unsigned same = __match_any_sync(0xffffffffu, who);
  unsigned firsts = __ballot_sync(0xffffffffu, who >= 0 && __ffs(same) - 1 == lane);
  const int groups = p.k / 64, c0 = groups * warp / 8, nc = groups * (warp + 1) / 8 - c0;
  // Piece c (16 bytes) of row r lies where reads of two rows at once meet no bank twice. A lane copies piece lane % 8 of rows lane / 8, + 4, ...
  const uint32_t ring = smem_u32(dyn) + warp * SH_DEPTH * SH_STAGE, put = (lane >> 3) * 128 + 16 * ((lane & 7) ^ (((lane >> 3) & 1) << 2));
  const uint32_t get = g * 128 + 64 * (g & 1) + 16 * t;
  const uint16_t* xr[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) xr[i] = static_cast<const uint16_t*>(p.x) + (size_t)(row0 + min((lane >> 3) + 4 * i, rows - 1)) * p.k + 64 * c0 + 8 * (lane & 7);
  for (; firsts; firsts &= firsts - 1u) {  // the different adapters
    const int r = __ffs(firsts) - 1, ad = __shfl_sync(0xffffffffu, who, r);
    const unsigned mine = __shfl_sync(0xffffffffu, same, r);
    const float scale = __ldcg(p.scale + ad);
    const uint16_t* ar = reinterpret_cast<const uint16_t*>(p.a) + ((size_t)ad * p.rank + j0 + (lane >> 3)) * p.k + 64 * c0 + 8 * (lane & 7);
    auto issue = [&](int c) {
      if (c < nc) {
        const uint32_t dst = ring + (c & (SH_DEPTH - 1)) * SH_STAGE + put;
#pragma unroll
        for (int i = 0; i < 4; ++i) few::cp16(dst + 512 * i, xr[i] + 64 * c);
#pragma unroll
        for (int i = 0; i < 2; ++i) few::cp16(dst + 2048 + 512 * i, ar + (size_t)4 * i * p.k + 64 * c);
      }
      few::cp_commit();
    };
    float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < SH_DEPTH; ++c) issue(c);
#pragma unroll 1
    for (int c = 0; c < nc; ++c) {
      few::cp_wait<SH_DEPTH - 1>();
      __syncwarp();
      const uint32_t at = ring + (c & (SH_DEPTH - 1)) * SH_STAGE + get;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = few::lds<uint4>(at ^ (64 * h)), v = few::lds<uint4>((at ^ (64 * h)) + 1024), b = few::lds<uint4>((at ^ (64 * h)) + 2048);
        if constexpr (F16) {
          uint32_t uh[4], ul[4], vh[4], vl[4];
          split_f16(u.x, uh[0], ul[0]), split_f16(u.y, uh[1], ul[1]), split_f16(u.z, uh[2], ul[2]), split_f16(u.w, uh[3], ul[3]);
          split_f16(v.x, vh[0], vl[0]), split_f16(v.y, vh[1], vl[1]), split_f16(v.z, vh[2], vl[2]), split_f16(v.w, vh[3], vl[3]);
          mma16<false>(d, uh[0], vh[0], uh[1], vh[1], b.x, b.y);
          mma16<false>(e, uh[2], vh[2], uh[3], vh[3], b.z, b.w);
          mma16<false>(d, ul[0], vl[0], ul[1], vl[1], b.x, b.y);
          mma16<false>(e, ul[2], vl[2], ul[3], vl[3], b.z, b.w);
        } else {
          mma16<false>(d, u.x, v.x, u.y, v.y, b.x, b.y);
          mma16<false>(e, u.z, v.z, u.w, v.w, b.z, b.w);
        }
      }
      __syncwarp();
      issue(c + SH_DEPTH);
    }
    few::cp_wait<0>();
    *reinterpret_cast<float2*>(&part[warp][g][2 * t]) = make_float2(d[0] + e[0], d[1] + e[1]);
    *reinterpret_cast<float2*>(&part[warp][g + 8][2 * t]) = make_float2(d[2] + e[2], d[3] + e[3]);
    __syncthreads();
    const int m = (int)threadIdx.x >> 3, j = threadIdx.x & 7;
    if (m < 16 && (mine >> m) & 1u) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += part[q][m][j];
      p.v[(size_t)(row0 + m) * p.rank + j0 + j] = s * scale;
    }
    __syncthreads();
  }
}

// ---- y = W x + res + B v -----------------------------------------------------------------------------------------------
DRB_DEV unsigned cluster_rank() {
  unsigned v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}
DRB_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
DRB_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
DRB_DEV float4 ld_peer(uint32_t addr, unsigned rank) {
  uint32_t a;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

// v of a row: three terms (see split3) of 64 ranks, pieces of eight ranks where reads of two terms at once meet no bank twice
constexpr int V_BYTES = 3 * MAX_RANK * 2;
DRB_DEV uint32_t v_at(int term, int piece) { return 128 * term + 16 * (piece ^ ((term & 1) << 2)); }

// NT column tiles (8 rows of x each) a pass; a slice of K inputs.
template <int NT>
struct Shape {
  static constexpr size_t SUMS = (size_t)CW * 8 * NT * PP * 4, RING = (size_t)CW * DEPTH * SUB;
  static constexpr size_t VS = (size_t)8 * NT * V_BYTES;  // v of the pass
  static constexpr size_t bytes(int slice) { return 256 + (size_t)8 * NT * (2 * slice + 16) + SUMS + RING + VS; }
};
static_assert(Shape<4>::bytes(MAX_K / 8) <= SMEM_MAX, "eight blocks hold the longest row");

// How a launch shares out its tiles and K: `each` tiles a cluster and one more for the first `more`; clusters of 1 << lcs blocks, 1 << lkw warps a
// tile. All divisions are made on the host (a few dozen runtime divisions a thread took 3 us of 15).
struct Split {
  int each, more, lcs, lkw, pitch;
};

// blockIdx.y: the pass of 8 NT rows of x.
template <bool F16, int NT>
__global__ void __launch_bounds__(THREADS, 2) k_proj(Args p, Split sp) {
  extern __shared__ __align__(128) unsigned char dyn[];
  int* who = reinterpret_cast<int*>(dyn);  // adapters of the pass's rows
  unsigned char* xs = dyn + 256;
  float* sums = reinterpret_cast<float*>(xs + (size_t)8 * NT * sp.pitch);
  unsigned char* vs = reinterpret_cast<unsigned char*>(sums) + Shape<NT>::SUMS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(vs) + Shape<NT>::VS + warp * DEPTH * SUB;
  const int lcs = sp.lcs, lkw = sp.lkw, cs = 1 << lcs, kw = 1 << lkw, pitch = sp.pitch;
  const int cr = (int)cluster_rank(), c = (int)blockIdx.x >> lcs;
  const int tw = CW >> lkw, wt = warp >> lkw, wk = warp & (kw - 1);                               // tiles of a batch; this warp's tile and share of K
  const int groups = p.k >> 7, b0 = groups * cr >> lcs, bn = (groups * (cr + 1) >> lcs) - b0;     // this block's inputs, in 128s
  const int g0 = bn * wk >> lkw, ng = (bn * (wk + 1) >> lkw) - g0;                                // this warp's, of the block's
  const int t0 = sp.each * c + min(sp.more, c), t1 = t0 + sp.each + (c < sp.more ? 1 : 0);
  const int row0 = (int)blockIdx.y * 8 * NT, cols = min(8 * NT, p.rows - row0);

  pdl_launch_dependents();

  // The weights' stream: tiles t0 + wt, t0 + wt + tw, ..., ng steps each. Rows behind the last one are read as the last one.
  const int mine = t1 - t0 > wt ? (t1 - t0 - wt + tw - 1) >> (3 - lkw) : 0;
  int nslot = 0, slot = 0, ltile = t0 + wt, lg = 0, left = mine * ng;
  const uint32_t put = (lane >> 3) * 128 + 16 * ((lane & 7) ^ (((lane >> 3) & 1) << 2));
  const int8_t* src = p.w;  // this lane's piece of the next step in row 16 ltile, and its four rows from there
  int over[4] = {0, 0, 0, 0};
  auto aim = [&]() {
    src = p.w + (size_t)16 * ltile * p.k + (b0 + g0) * 128 + 16 * (lane & 7);
#pragma unroll
    for (int i = 0; i < 4; ++i) over[i] = min((lane >> 3) + 4 * i, p.n - 1 - 16 * ltile) * p.k;
    // the tile's scales, which are read a step ahead of use, come to L2 with its first weights
    if (lane < 16) prefetch_line_l2(p.s + (size_t)min(16 * ltile + lane, p.n - 1) * groups + b0 + g0);
  };
  if (left > 0) aim();
  auto issue = [&]() {
    if (left > 0) {
      const uint32_t dst = ring + nslot * SUB + put;
#pragma unroll
      for (int i = 0; i < 4; ++i) few::cp16(dst + 512 * i, src + over[i]);
      src += 128;
      --left;
      if (++lg == ng) {
        lg = 0, ltile += tw;
        if (left > 0) aim();
      }
    }
    few::cp_commit();
    if (++nslot == DEPTH) nslot = 0;
  };
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) issue();
  __half s0 = __half(), s1 = __half();  // the next step's; converted when they are used, so that nothing waits for them before
  auto scales = [&](int tile, int grp) {
    s0 = __ldg(p.s + (size_t)min(16 * tile + g, p.n - 1) * groups + b0 + g0 + grp);
    s1 = __ldg(p.s + (size_t)min(16 * tile + g + 8, p.n - 1) * groups + b0 + g0 + grp);
  };
  if (mine * ng > 0) scales(t0 + wt, 0);

  if (p.rank == 0) pdl_wait();  // with adapters x and the rest are older than k_shrink, and only v is awaited, below
  // x by plain loads, so that nothing here waits for the weights: a warp takes NT rows, 16 bytes a lane, two pieces of each at once
  const int ad = p.rank > 0 && lane < cols ? adapter(p, row0 + lane) : -1;  // lane r: of row r
  {
    const uint4* src[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) src[i] = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + (size_t)(row0 + min(warp + CW * i, cols - 1)) * p.k + b0 * 128);
    for (int q = lane; q < 16 * bn; q += 64) {
      uint4 v[2][NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        v[0][i] = __ldcg(src[i] + q);
        if (q + 32 < 16 * bn) v[1][i] = __ldcg(src[i] + q + 32);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint4* dst = reinterpret_cast<uint4*>(xs + (warp + CW * i) * pitch);
        dst[q] = v[0][i];
        if (q + 32 < 16 * bn) dst[q + 32] = v[1][i];
      }
    }
  }
  const bool any = __ballot_sync(0xffffffffu, ad >= 0) != 0u;  // the same in every warp
  if (warp == 0) who[lane] = ad;
  // The adapters' second half: a warp takes the sixteen weight rows of a tile for a row of x, whose v is the other operand, a term a column; the pairs
  // of a batch are dealt out over the cluster and its warps. The rows of B for the first batch come to L2 meanwhile.
  const int lr = lane >> 1, half = lane & 1;
  auto pair_row = [&](int tile, int a) { return p.b + ((size_t)a * p.n + min(16 * tile + lr, p.n - 1)) * p.rank; };
  if (any)
    for (int i = cr * CW + warp; i < min(tw, t1 - t0) * 8 * NT; i += cs * CW) {
      const int a = __shfl_sync(0xffffffffu, ad, i % (8 * NT));
      if (a >= 0 && 32 * half < p.rank) prefetch_line_l2(pair_row(t0 + i / (8 * NT), a) + 32 * half);
    }
  __syncthreads();

  const int batches = (t1 - t0 + tw - 1) >> (3 - lkw);
  const uint32_t xb = smem_u32(xs) + g * pitch + 32 * t + 256 * g0;
  for (int bt = 0; bt < batches; ++bt) {
    const int tile = t0 + bt * tw + wt;
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    if (tile < t1) {
#pragma unroll 1
      for (int q = 0; q < ng; ++q) {
        const __half h0 = s0, h1 = s1;
        if (q + 1 < ng) scales(tile, q + 1);
        else if (tile + tw < t1) scales(tile + tw, 0);
        few::cp_wait<DEPTH - 1>();
        __syncwarp();
        const uint32_t r0 = ring + slot * SUB + g * 128 + 64 * (g & 1) + 16 * t;
        float d[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 u = few::lds<uint4>(r0 ^ (64 * h)), v = few::lds<uint4>((r0 ^ (64 * h)) + 1024);
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
              const uint4 b = few::lds<uint4>(xb + 8 * i * pitch + q * 256 + h * 128 + 16 * e);
              mma16<F16>(d[i], a[0], a[1], a[2], a[3], b.x, b.y);
              mma16<F16>(d[i], a[4], a[5], a[6], a[7], b.z, b.w);
            }
          }
        }
        __syncwarp();
        issue();
        if (++slot == DEPTH) slot = 0;
        const float f0 = __half2float(h0), f1 = __half2float(h1);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          acc[i][0] = fmaf(f0, d[i][0], acc[i][0]), acc[i][1] = fmaf(f0, d[i][1], acc[i][1]);
          acc[i][2] = fmaf(f1, d[i][2], acc[i][2]), acc[i][3] = fmaf(f1, d[i][3], acc[i][3]);
        }
      }
    }
    if (p.rank > 0 && bt == 0) {
      pdl_wait();  // v
      if (any) {
        for (int i = threadIdx.x; i < 8 * NT * (MAX_RANK / 4); i += THREADS) {
          const int r = i / (MAX_RANK / 4), q = i % (MAX_RANK / 4);
          const float4 f = r < cols && who[r] >= 0 && 4 * q < p.rank ? __ldcg(reinterpret_cast<const float4*>(p.v + (size_t)(row0 + r) * p.rank) + q)
                                                                     : make_float4(0.f, 0.f, 0.f, 0.f);
          uint32_t b0[3], b1[3];
          split3(f, b0, b1);
#pragma unroll
          for (int l = 0; l < 3; ++l) *reinterpret_cast<uint2*>(vs + r * V_BYTES + v_at(l, q >> 1) + 8 * (q & 1)) = make_uint2(b0[l], b1[l]);
        }
        __syncthreads();
      }
    }
    __syncwarp();
    if (bt > 0) cluster_wait();  // everyone has read the batch before
    float* st = sums + warp * 8 * NT * PP;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      st[(8 * i + 2 * t) * PP + g] = acc[i][0], st[(8 * i + 2 * t + 1) * PP + g] = acc[i][1];
      st[(8 * i + 2 * t) * PP + g + 8] = acc[i][2], st[(8 * i + 2 * t + 1) * PP + g + 8] = acc[i][3];
    }
    const int nt = min(tw, t1 - t0 - bt * tw);
    if (any) {
      __syncthreads();
      constexpr int PAIRS = NT == 1 ? 2 : 4;  // on the way at once: of few pairs a warp has one or two, and every one more is code to fetch
      for (int i0 = cr * CW + warp; i0 < nt * 8 * NT; i0 += PAIRS * cs * CW) {
        float d[PAIRS][4];
        const __nv_bfloat16* bp[PAIRS];  // this lane's row g; row g + 8 lies `down` numbers on
        int r[PAIRS], down[PAIRS];
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          const int i = i0 + e * cs * CW, o = 16 * (t0 + bt * tw + i / (8 * NT)) + g;
          r[e] = i % (8 * NT), d[e][0] = d[e][1] = d[e][2] = d[e][3] = 0.f;
          bp[e] = who[r[e]] < 0 || i >= nt * 8 * NT ? nullptr : p.b + ((size_t)who[r[e]] * p.n + min(o, p.n - 1)) * p.rank + 8 * t;
          down[e] = (min(o + 8, p.n - 1) - min(o, p.n - 1)) * p.rank;
        }
        for (int q = 0; q < p.rank; q += 32) {
          uint4 u[PAIRS], v[PAIRS];
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            u[e] = v[e] = make_uint4(0u, 0u, 0u, 0u);
            if (bp[e] && q + 8 * t < p.rank)
              u[e] = __ldcg(reinterpret_cast<const uint4*>(bp[e] + q)), v[e] = __ldcg(reinterpret_cast<const uint4*>(bp[e] + q + down[e]));
          }
#pragma unroll
          for (int e = 0; e < PAIRS; ++e) {
            const uint4 c = g < 3 ? *reinterpret_cast<const uint4*>(vs + r[e] * V_BYTES + v_at(g, q / 8 + t)) : make_uint4(0u, 0u, 0u, 0u);
            mma16<false>(d[e], u[e].x, v[e].x, u[e].y, v[e].y, c.x, c.y);
            mma16<false>(d[e], u[e].z, v[e].z, u[e].w, v[e].w, c.z, c.w);
          }
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {  // the three terms' columns: two in lanes t = 0, one in t = 1
          float lo = d[e][0] + d[e][1], hi = d[e][2] + d[e][3];
          lo += __shfl_xor_sync(0xffffffffu, lo, 1), hi += __shfl_xor_sync(0xffffffffu, hi, 1);
          float* at = sums + ((i0 + e * cs * CW) / (8 * NT) * kw * 8 * NT + r[e]) * PP + g;
          if (t == 0 && bp[e]) at[0] += lo, at[8] += hi;
        }
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    // Block cr of the cluster finishes its share of the batch, four weight rows of a column (a row of x) at a time
    for (int i = cr * THREADS + (int)threadIdx.x; i < tw * 4 * cols; i += cs * THREADS) {
      const int j = 4 * (i & 3), m = (i >> 2) & (tw - 1), r = i >> (5 - lkw), o = 16 * (t0 + bt * tw + m) + j, row = row0 + r;
      if (m >= nt || o >= p.n) continue;
      const uint32_t at = smem_u32(sums + (m * kw * 8 * NT + r) * PP + j);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < kw; ++k) {
        float4 f[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = q < cs ? ld_peer(at + k * 8 * NT * PP * 4, (unsigned)q) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[0] += f[q].x, v[1] += f[q].y, v[2] += f[q].z, v[3] += f[q].w;
      }
      const size_t yo = (size_t)row * p.n + o;
      if (p.n % 4 == 0 && (((uintptr_t)p.y | (uintptr_t)p.res) & 15) == 0) {
        if (p.res) {
          const float4 a = __ldcg(reinterpret_cast<const float4*>(p.res + yo));
          v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
        }
        *reinterpret_cast<float4*>(p.y + yo) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        for (int l = 0; l < 4 && o + l < p.n; ++l) p.y[yo + l] = p.res ? v[l] + __ldcg(p.res + yo + l) : v[l];
      }
    }
    __syncwarp();
    cluster_arrive();
  }
  if (batches > 0) cluster_wait();
  few::cp_wait<0>();
}

template <bool F16>
static void launch_shrink(const Args& p, const DrbDevice& dev, bool many, cudaStream_t st) {
  if (many) drb_launch(k_shrink_rows<F16>, dim3((p.rows + 15) / 16, p.rank / 8), dim3(256), SH_BYTES, st, dev.pdl, p);
  else drb_launch(k_shrink<F16>, dim3(p.rows, p.rank / 8), dim3(256), shrink_bytes(p.k), st, dev.pdl, p);
}

// Clusters of cs blocks that are resident at once, with one block a multiprocessor and with two: a property of the device, asked once.
constexpr int MAX_DEVICES = 32;
static int g_clusters[MAX_DEVICES][2][4];

// The rows of x decide NT, up to 32 a pass. Blocks of a cluster (cs) and warps of a block (kw) share K. Of all splits whose slice of x fits, the one
// with the least work on a warp's way (of equals the widest cluster, whose blocks read least of x): batches of tiles, each (in halves of a step) its steps and about three steps of a
// batch's end, which grows with the slices whose sums meet there. `resident`: clusters of 1, 2, 4
// and 8 blocks that the device holds at once, [0] with one block a multiprocessor, [1] with two; 0: it runs none of that width.
struct Plan {
  int cs, kw, clusters;  // clusters 0: no width runs
};
template <int NT>
static Plan plan(const int (&resident)[2][4], int rows, int n, int k) {
  const int groups = k / 128, mt = (n + 15) / 16, passes = (rows + 8 * NT - 1) / (8 * NT);
  Plan best = {0, 0, 0};
  long long least = -1;
  for (int lg = 0; lg < 4 && 1 << lg <= groups; ++lg) {
    const int slice = (groups + (1 << lg) - 1) >> lg;
    const size_t bytes = Shape<NT>::bytes(128 * slice);
    if (bytes > SMEM_MAX) continue;
    const int all = resident[bytes <= SMEM_TWO][lg], avail = all / passes;
    if (all < 1) continue;
    for (int w = 1; w <= 4 && w <= slice; w *= 2) {
      const int need = (int)(((long long)mt * w + CW - 1) / CW), have = avail < 1 ? 1 : avail < need ? avail : need;
      const int waves = avail < 1 ? (passes + all - 1) / all : 1;
      const long long cost = (long long)waves * ((need + have - 1) / have) * (2 * ((slice + w - 1) / w) + 6 + w * (1 << lg) / 2);
      if (least < 0 || cost <= least) least = cost, best = {1 << lg, w, have};
    }
  }
  return best;
}

template <bool F16, int NT>
static int launch(const Args& p, const DrbDevice& dev, cudaStream_t st) {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= MAX_DEVICES) return -2;
  const int groups = p.k / 128, mt = (p.n + 15) / 16, passes = (p.rows + 8 * NT - 1) / (8 * NT);
  const Plan pn = plan<NT>(g_clusters[d], p.rows, p.n, p.k);
  if (pn.clusters == 0) return -1;
  const int cs = pn.cs, kw = pn.kw, clusters = pn.clusters;
  if (p.rank > 0) launch_shrink<F16>(p, dev, false, st);
  const size_t smem = Shape<NT>::bytes(128 * ((groups + cs - 1) / cs));
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
  const auto lg2 = [](int v) { return v == 1 ? 0 : v == 2 ? 1 : v == 4 ? 2 : 3; };
  const Split sp = {mt / clusters, mt % clusters, lg2(cs), lg2(kw), 2 * 128 * ((groups + cs - 1) / cs) + 16};
  cudaLaunchKernelEx(&cfg, k_proj<F16, NT>, p, sp);
  return 0;
}

template <bool F16>
static int launch_few(const Args& p, const DrbDevice& dev, cudaStream_t st) {
  if (p.rows <= 8) return launch<F16, 1>(p, dev, st);
  if (p.rows <= 16) return launch<F16, 2>(p, dev, st);
  if (p.rows <= 24) return launch<F16, 3>(p, dev, st);
  return launch<F16, 4>(p, dev, st);
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
  if ((e = configure<F16, 3>()) != cudaSuccess) return e;
  if ((e = configure<F16, 4>()) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(k_shrink_rows<F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SH_BYTES)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_shrink_rows<F16>)) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(k_shrink<F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, shrink_bytes(SK))) != cudaSuccess) return e;
  return drb_carveout(k_shrink<F16>);
}
static cudaError_t configure_all() {
  cudaError_t e = configure_type<false>();
  if (e != cudaSuccess || (e = configure_type<true>()) != cudaSuccess) return e;
  int d = 0;
  if ((e = cudaGetDevice(&d)) != cudaSuccess) return e;
  if (d < 0 || d >= MAX_DEVICES) return cudaErrorInvalidDevice;
  for (int two = 0; two < 2; ++two)
    for (int lg = 0; lg < 4; ++lg) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1 << lg), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = two ? SMEM_TWO : SMEM_MAX;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1 << lg, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr, cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&g_clusters[d][two][lg], k_proj<true, 4>, &cfg) != cudaSuccess) g_clusters[d][two][lg] = 0, cudaGetLastError();
    }
  return cudaSuccess;
}

}  // namespace pl
