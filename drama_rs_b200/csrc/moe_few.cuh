// drb_moe_few: one whole MoE layer for 1 to 16 tokens in ONE cooperative kernel.
//
//   y_r = x_r + sigmoid(l_r[e]) shared(xh_r) + sum_k w_rk expert_{idx_rk}(xh_r),  xh = rmsnorm(x) * nw,  l = R xh
//
// For few tokens nearly every (token, expert) pair has an expert of its own: 1.8 MB of int4 weights that are read once and meet one or
// two rows, so the weights' stream is the floor and what lies between is latency. One block per multiprocessor, all resident:
//
//   logits     block b: some router rows for a group of four tokens; handed over as tagged words (payload, call number), which every
//              block polls, so that every block derives the same routing and the same list of the experts hit
//   gate/up    tiles of 8 gate rows and their 8 up rows, [experts hit] x 64 in one list that the blocks share out in equal
//              runs; four warps a tile, 512 inputs each. The shared expert's 64 tiles go to sixteen blocks before the routing exists.
//   down       tiles of 16 output rows, one warp each, [shared, experts hit] x 128 in one list. A block's run spans two
//              experts at most; it waits for their activations (a counter each), while its weights are on the way
//   combine    every tile's weighted result goes to memory; once all blocks have finished, each adds up its share of the outputs,
//              in rank order
//
// Weights come by 16-byte asynchronous copies into a ring of each warp's own (no barrier in a step), which runs on from gate/up into
// down. They are multiplied by mma.sync m16n8k32 s8 (the few rows cannot fill a tcgen05 tile, and the operands need no tensor memory): the
// codes are exact, and the activations are three signed 8-bit digits of a 24-bit fixed-point number per 64 inputs (error 2^-24 of
// the largest of the 64, as fp32 has it), one column a digit. Sums over 64 inputs are exact integers; scale, min and the digits'
// weights are applied in fp32. Int4 costs three logic operations per eight weights this way.
//
// Every wait is bounded: one that runs out sets the device error word and the block's abort flag, after which no wait of the block
// spins again and the kernel runs to its end.
#pragma once

#include <stddef.h>

#include <type_traits>

#include "gemv.cuh"
#include "moe_decode.cuh"
#include "stack_decode.cuh"

namespace few {

using moe::H;
using moe::I;

constexpr int CW = 16, THREADS = CW * 32;
constexpr int MAX_TOK = 16, MAX_K = 8, MAX_E = 256, MAX_HIT = MAX_TOK * MAX_K;
constexpr int SHARED_BLOCKS = 16;             // blocks of the shared expert's gate/up: a tile for each group of four warps
constexpr int GU_TILES = I / 8, DN_TILES = H / 16;
constexpr int MIN_GRID = 144, MAX_GRID = 1024;  // runs of at most 64 gate/up and 128 down tiles: two experts a block
constexpr int LOGIT_STRIDE = MAX_E + 8;       // words a token

// Workspace: the head is the same for every size, activations and weighted results follow.
struct alignas(256) Head {
  unsigned epoch, seen;  // calls so far; blocks that have read `epoch` in this call
  unsigned pad[62];
  unsigned act_done[2][MAX_HIT + 8];   // [call parity][expert hit, MAX_HIT = shared]: gate/up tiles finished; [MAX_HIT + 1]: blocks finished
  unsigned long long logits[MAX_TOK * LOGIT_STRIDE];
};
static_assert(sizeof(Head) % 256 == 0 && offsetof(Head, logits) % 16 == 0, "aligned sections");

constexpr int SUB = 2048;                // a step of a warp: 16 rows x 128 bytes
constexpr int SLOT = SUB + 256;          // and 16 bytes of scales a row
constexpr int PITCH = H + 64, DPITCH = I + 64;    // bytes between digit planes: neighbouring planes on different banks
constexpr int MP = H / 64 + 1, DMP = I / 64 + 1;  // per 64 inputs, tokens apart: (delta, sum, 65536 delta, 0), see Cols

template <int TOK>
struct Shape {
  static constexpr int DEPTH = TOK > 8 ? 3 : 4;
  static constexpr int PLANES = 3 * TOK * PITCH, META = TOK * MP * 16, RING = CW * DEPTH * SLOT, RED = CW * 16 * 8 * 4;
  static constexpr int CTL = 3072;
  static constexpr size_t BYTES = CTL + PLANES + META + RING + RED;
  static_assert(BYTES <= 232448 && 2 * 3 * TOK * DPITCH <= PLANES && 2 * TOK * DMP * 16 <= META, "shared memory");
};

struct Seg {  // the tokens of one expert in this block's run
  int count;
  float wt[16];           // weight of the expert's result
  float rr[16];           // 1 / rms of the token
  short row[16];          // row of the activations and of the weighted results
  unsigned char pos[16];  // digit planes
};

struct Ctl {
  Seg seg[2];
  uint64_t arrived[4][4];   // [group of four warps][tile mod 4]: warps whose sums of a tile lie in shared memory
  int idx[MAX_TOK][MAX_K];
  float wts[MAX_TOK][MAX_K];
  float sgate[MAX_TOK], rr[MAX_TOK], rr_own[MAX_TOK], ss[CW];
  unsigned mask[MAX_E];     // tokens that chose the expert
  unsigned char hit[MAX_HIT];
  int wsum[8];
  int nhit, abort;
  int range[4];             // this block's gate/up tiles and down tiles
};
static_assert(sizeof(Ctl) <= Shape<16>::CTL, "control block");

DRB_DEV void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
DRB_DEV void cp4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
DRB_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
DRB_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

DRB_DEV unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
DRB_DEV unsigned atom_add_acq_rel(unsigned* p, unsigned v) {
  unsigned r;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(r) : "l"(p), "r"(v) : "memory");
  return r;
}
DRB_DEV void quad_sync(int quad) { asm volatile("bar.sync %0, 128;" ::"r"(1 + quad) : "memory"); }

// Four inputs of a lane (sixteen lanes share 64) as the digits of round(v / delta), delta = max|v| / 8,355,000 (127 (1 + 256 + 65536) is the
// largest number that three signed bytes hold). n + 0x808080 has the digits plus 128 as its bytes. 16 bytes of a plane hold 16
// inputs as words of {0,2,4,6}, {1,3,5,7}, {8,10,12,14}, {9,11,13,15}, the order in which the nibbles of eight bytes come.
// A NaN or an infinity among the 64 makes delta NaN or infinite, and with it every sum that the 64 enter. Also the sum of the 64.
DRB_DEV void digits4(const float4& v, unsigned char* plane, int pitch, float4* meta, int lane) {
  unsigned mb = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                    max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
  float sum = (v.x + v.y) + (v.z + v.w);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const float m = __uint_as_float(mb);
  // kept away from the subnormals, whose reciprocal is infinite
  const float delta = mb < 0x7f800000u ? fmaxf(m * (1.f / 8355000.f), 1.1754944e-38f) : m;
  const float inv = 1.f / delta;  // 0 or NaN beside an infinity or a NaN: the digits do not matter then
  const uint32_t n0 = (uint32_t)(__float2int_rn(v.x * inv) + 0x808080) ^ 0x808080u, n1 = (uint32_t)(__float2int_rn(v.y * inv) + 0x808080) ^ 0x808080u;
  const uint32_t n2 = (uint32_t)(__float2int_rn(v.z * inv) + 0x808080) ^ 0x808080u, n3 = (uint32_t)(__float2int_rn(v.w * inv) + 0x808080) ^ 0x808080u;
  const uint32_t e01 = prmt(n0, n2, 0x5140u), e2 = prmt(n0, n2, 0x0062u), o01 = prmt(n1, n3, 0x5140u), o2 = prmt(n1, n3, 0x0062u);
  unsigned char* w = plane + 8 * (lane >> 1) + 2 * (lane & 1);  // the even inputs; the odd ones four bytes on
  *reinterpret_cast<uint16_t*>(w) = (uint16_t)e01, *reinterpret_cast<uint16_t*>(w + 4) = (uint16_t)o01;
  w += pitch;
  *reinterpret_cast<uint16_t*>(w) = (uint16_t)(e01 >> 16), *reinterpret_cast<uint16_t*>(w + 4) = (uint16_t)(o01 >> 16);
  w += pitch;
  *reinterpret_cast<uint16_t*>(w) = (uint16_t)e2, *reinterpret_cast<uint16_t*>(w + 4) = (uint16_t)o2;
  if ((lane & 15) == 0) meta[lane >> 4] = make_float4(delta, sum, 65536.f * delta, 0.f);
}

// The weights of a warp's tiles on their way. A tile's rows are contiguous; the next tile of the same expert lies dp (ds) bytes on.
enum Mode { SHARED_GU, GU, DN, OVER };
struct Loader {
  const unsigned char *p;   // this lane's first row and piece of the next step
  const unsigned char *sp;  // this lane's row of scales (lanes 0..15)
  uint32_t at;              // where they go in a slot
  int stride, gap;          // bytes over four rows, and from row r to row r + 8
  int sub, nsub, u, uend, ustep, dp, ds, mode;
  bool int8;
};

struct Params {
  drb_moe_layer w;
  const float* x;
  float* y;
  const uint8_t* live;
  Head* ws;
  float *act, *part;
  int n, e, topk;
  float eps;
  unsigned poll_limit;
};

// One warp's share of a tile: 16 rows against the tokens of a segment. TG = 0: one or two tokens, four columns each (three digits);
// TG = 1, 2: up to 8 or 16 tokens, a column tile per digit and eight tokens.
template <int TG>
struct Acc {
  float v[TG ? TG * 4 : 2];
};

template <int TG>
struct Cols {
  const unsigned char* b[TG ? TG : 1];         // this lane's column: its token's digit planes
  const unsigned char* m[TG ? 2 * TG : 1];     // delta and sum of the columns whose sums this lane holds. TG = 0: lanes of the third digit
                                               // take 65536 delta and no sum
  int second;                                  // TG = 0: weight of this lane's second column
};

template <int TG>
DRB_DEV void cols_set(Cols<TG>& c, const Seg& s, const unsigned char* planes, int pitch, const float4* meta, int mp, int lane) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (TG == 0) {
    c.b[0] = planes + (3 * s.pos[min(g >> 2, s.count - 1)] + min(g & 3, 2)) * pitch + 16 * t;
    c.m[0] = reinterpret_cast<const unsigned char*>(meta + s.pos[min(t >> 1, s.count - 1)] * mp) + 8 * (t & 1);
    c.second = t & 1 ? 0 : 256;
  } else {
#pragma unroll
    for (int i = 0; i < TG; ++i) {
      c.b[i] = planes + 3 * s.pos[min(8 * i + g, s.count - 1)] * pitch + 16 * t;
      c.m[2 * i] = reinterpret_cast<const unsigned char*>(meta + s.pos[min(8 * i + 2 * t, s.count - 1)] * mp);
      c.m[2 * i + 1] = reinterpret_cast<const unsigned char*>(meta + s.pos[min(8 * i + 2 * t + 1, s.count - 1)] * mp);
    }
  }
}

DRB_DEV void mma_s8_zero(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// 64 inputs: A in the operand's registers, group kg of the planes; s0, m0: scale and min of row g, s1, m1 of row g + 8. A digit's sum stays
// below 2^20.1 (int8 codes), so it and 256 times the next one's fit an integer.
template <int TG, bool MIN>
DRB_DEV void group64(Acc<TG>& acc, const Cols<TG>& c, int pitch, int kg, const uint32_t (&a)[8], float s0, float m0, float s1, float m1) {
  if constexpr (TG == 0) {
    const uint4 b = *reinterpret_cast<const uint4*>(c.b[0] + 64 * kg);
    int d[4];
    mma_s8_zero(d, a[0], a[1], a[2], a[3], b.x, b.y);
    gemv::q8::mma_s8(d, a[4], a[5], a[6], a[7], b.z, b.w);
    const float2 m = *reinterpret_cast<const float2*>(c.m[0] + 16 * kg);
    acc.v[0] = fmaf(s0 * m.x, (float)(d[1] * c.second + d[0]), acc.v[0]);
    acc.v[1] = fmaf(s1 * m.x, (float)(d[3] * c.second + d[2]), acc.v[1]);
    if (MIN) acc.v[0] = fmaf(m0, m.y, acc.v[0]), acc.v[1] = fmaf(m1, m.y, acc.v[1]);
  } else {
#pragma unroll
    for (int i = 0; i < TG; ++i) {
      int d[3][4];
#pragma unroll
      for (int l = 0; l < 3; ++l) {
        const uint4 b = *reinterpret_cast<const uint4*>(c.b[i] + l * pitch + 64 * kg);
        mma_s8_zero(d[l], a[0], a[1], a[2], a[3], b.x, b.y);
        gemv::q8::mma_s8(d[l], a[4], a[5], a[6], a[7], b.z, b.w);
      }
      const float2 c0 = *reinterpret_cast<const float2*>(c.m[2 * i] + 16 * kg), c1 = *reinterpret_cast<const float2*>(c.m[2 * i + 1] + 16 * kg);
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = fmaf((float)d[2][j], 65536.f, (float)(d[1][j] * 256 + d[0][j]));
      float* v = acc.v + 4 * i;
      v[0] = fmaf(s0, f[0] * c0.x, v[0]), v[1] = fmaf(s0, f[1] * c1.x, v[1]);
      v[2] = fmaf(s1, f[2] * c0.x, v[2]), v[3] = fmaf(s1, f[3] * c1.x, v[3]);
      if (MIN) {
        v[0] = fmaf(m0, c0.y, v[0]), v[1] = fmaf(m0, c1.y, v[1]);
        v[2] = fmaf(m1, c0.y, v[2]), v[3] = fmaf(m1, c1.y, v[3]);
      }
    }
  }
}

// One step of 128 bytes a row: 256 int4 or 128 int8 inputs from group kg on. The ring keeps 16-byte pieces where reads of 8 rows meet
// no bank twice (see `issue`).
template <int TG, bool INT8>
DRB_DEV void step(Acc<TG>& acc, const Cols<TG>& c, int pitch, int kg, const unsigned char* slot, int sub, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const unsigned char* r0 = slot + g * 128;
  const unsigned char* r1 = r0 + 8 * 128;
  uint32_t a[8];
  if constexpr (INT8) {
    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(slot + SUB + 16 * g), w1 = *reinterpret_cast<const uint32_t*>(slot + SUB + 16 * g + 128);
    const float s0 = __half2float(__ushort_as_half((uint16_t)(sub & 1 ? w0 >> 16 : w0)));
    const float s1 = __half2float(__ushort_as_half((uint16_t)(sub & 1 ? w1 >> 16 : w1)));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int at = 64 * (q ^ (g & 1)) + 16 * t;
      const uint4 u = *reinterpret_cast<const uint4*>(r0 + at), v = *reinterpret_cast<const uint4*>(r1 + at);
      a[0] = prmt(u.x, u.y, 0x6420u), a[1] = prmt(v.x, v.y, 0x6420u), a[2] = prmt(u.x, u.y, 0x7531u), a[3] = prmt(v.x, v.y, 0x7531u);
      a[4] = prmt(u.z, u.w, 0x6420u), a[5] = prmt(v.z, v.w, 0x6420u), a[6] = prmt(u.z, u.w, 0x7531u), a[7] = prmt(v.z, v.w, 0x7531u);
      group64<TG, false>(acc, c, pitch, kg + q, a, s0, 0.f, s1, 0.f);
    }
  } else {
    const uint4 w0 = *reinterpret_cast<const uint4*>(slot + SUB + 16 * g), w1 = *reinterpret_cast<const uint4*>(slot + SUB + 16 * g + 128);
    const uint32_t sm0[4] = {w0.x, w0.y, w0.z, w0.w}, sm1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 32 * (q ^ (g & 3)) + 8 * t;
      const uint2 u = *reinterpret_cast<const uint2*>(r0 + at), v = *reinterpret_cast<const uint2*>(r1 + at);
      a[0] = u.x & 0x0F0F0F0Fu, a[1] = v.x & 0x0F0F0F0Fu, a[2] = (u.x >> 4) & 0x0F0F0F0Fu, a[3] = (v.x >> 4) & 0x0F0F0F0Fu;
      a[4] = u.y & 0x0F0F0F0Fu, a[5] = v.y & 0x0F0F0F0Fu, a[6] = (u.y >> 4) & 0x0F0F0F0Fu, a[7] = (v.y >> 4) & 0x0F0F0F0Fu;
      const float2 c0 = __half22float2(*reinterpret_cast<const __half2*>(&sm0[q])), c1 = __half22float2(*reinterpret_cast<const __half2*>(&sm1[q]));
      group64<TG, true>(acc, c, pitch, kg + q, a, c0.x, c0.y, c1.x, c1.y);
    }
  }
}

// What a tile costs with `count` tokens, in quarters of one with one or two: instructions, which grow with the column tiles.
DRB_DEV int tile_cost(int count) { return count <= 2 ? 4 : count <= 8 ? 6 : 11; }
constexpr int SHARED_HEAD_START = 8;  // the shared expert's gate/up, in tiles of one or two tokens that its blocks do less of

template <int TOK>
__global__ void __launch_bounds__(THREADS, 1) k_moe_few(Params P) {
  using S = Shape<TOK>;
  constexpr int DEPTH = S::DEPTH;
  extern __shared__ __align__(128) unsigned char dyn[];
  Ctl& ctl = *reinterpret_cast<Ctl*>(dyn);
  unsigned char* planes = dyn + S::CTL;
  float4* meta = reinterpret_cast<float4*>(planes + S::PLANES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp >> 2, kq = warp & 3;
  unsigned char* ring = planes + S::PLANES + S::META + warp * DEPTH * SLOT;
  float* red = reinterpret_cast<float*>(planes + S::PLANES + S::META + S::RING);
  const int n = P.n, E = P.e, topk = P.topk, E1 = E + 1;
  const int G = (int)gridDim.x, b = (int)blockIdx.x;
  volatile int* abort_flag = &ctl.abort;
  const int GN = G - SHARED_BLOCKS, shared_block = b - GN;  // >= 0: one of them

  // ---------------- the weights' stream
  Loader ld;
  ld.mode = OVER;
  int nslot = 0, slot = 0;  // ring positions: next to fill, next to use
  auto point = [&](const void* w, const void* s, bool int8, int row_bytes, int row0, int gap_rows, int off, int srow_bytes, int soff, int nsub, int rows_on) {
    ld.int8 = int8;
    ld.stride = 4 * row_bytes, ld.gap = gap_rows * row_bytes;
    const int r = lane >> 3, c = lane & 7, sr = lane & 15;
    // Piece c (16 bytes) of row r lies where reads of eight rows at once meet no bank twice: int4 rows are read 32 bytes (four
    // lanes) at a time, int8 rows 64.
    ld.at = r * 128 + 16 * (int8 ? c ^ ((r & 1) << 2) : c ^ ((r & 3) << 1));
    ld.p = static_cast<const unsigned char*>(w) + (size_t)(row0 + r) * row_bytes + off + 16 * c;
    ld.sp = static_cast<const unsigned char*>(s) + (size_t)(row0 + (sr < 8 ? sr : sr - 8 + gap_rows)) * srow_bytes + soff;
    ld.sub = 0, ld.nsub = nsub;
    ld.dp = rows_on * row_bytes - 128 * nsub, ld.ds = rows_on * srow_bytes;
  };
  int gu0 = 0, gu1 = 0, dn0 = 0, dn1 = 0;  // this block's tiles: expert hit x GU_TILES; shared, then expert hit x DN_TILES
  auto aim_gu = [&]() {
    const int h = ld.u / GU_TILES;
    ld.mode = GU, ld.ustep = 4, ld.uend = min(gu1, (h + 1) * GU_TILES);
    point(P.w.gu_q, P.w.gu_sm, false, H / 2, ctl.hit[h] * 2 * I + 8 * (ld.u % GU_TILES), I, kq * 256, H / 64 * 4, kq * 32, 2, 32);
  };
  auto aim_dn = [&]() {
    const int h = ld.u / DN_TILES - 1, row0 = 16 * (ld.u % DN_TILES);
    ld.mode = DN, ld.ustep = CW, ld.uend = min(dn1, (h + 2) * DN_TILES);
    if (h < 0) point(P.w.sd_q, P.w.sd_s, true, I, row0, 8, 0, I / 128 * 2, 0, 4, 16 * CW);
    else point(P.w.d_q, P.w.d_sm, false, I / 2, ctl.hit[h] * H + row0, 8, 0, I / 64 * 4, 0, 2, 16 * CW);
  };
  auto issue = [&]() {  // requests the next step, if there is one
    if (ld.mode != OVER) {
      const uint32_t dst = smem_u32(ring + nslot * SLOT), d = dst + ld.at;
      cp16(d, ld.p);
      cp16(d + 512, ld.p + ld.stride);
      cp16(d + 1024, ld.p + ld.gap);
      cp16(d + 1536, ld.p + ld.gap + ld.stride);
      if (lane < 16) {
        if (ld.int8) cp4(dst + SUB + 16 * lane, ld.sp + 4 * (ld.sub >> 1));
        else cp16(dst + SUB + 16 * lane, ld.sp + 16 * ld.sub);
      }
      ld.p += 128;
      if (++ld.sub == ld.nsub) {
        ld.sub = 0, ld.u += ld.ustep;
        if (ld.u < ld.uend) {
          ld.p += ld.dp, ld.sp += ld.ds;
        } else if (ld.mode == SHARED_GU) {
          ld.mode = OVER;
        } else if (ld.mode == GU && ld.u < gu1) {
          aim_gu();
        } else {
          if (ld.mode == GU) ld.u = dn0 + warp;
          if (ld.u < dn1) aim_dn();
          else ld.mode = OVER;
        }
      }
    }
    cp_commit();
    if (++nslot == DEPTH) nslot = 0;
  };
  auto next_slot = [&]() -> const unsigned char* {
    cp_wait<DEPTH - 1>();
    __syncwarp();
    return ring + slot * SLOT;
  };
  auto used = [&]() {
    __syncwarp();
    issue();
    if (++slot == DEPTH) slot = 0;
  };
  if (shared_block >= 0) {
    ld.mode = SHARED_GU, ld.u = 0, ld.ustep = 1, ld.uend = 1;
    point(P.w.sgu_q, P.w.sgu_s, true, H, 8 * (4 * shared_block + quad), I, kq * 512, H / 128 * 2, kq * 8, 4, 0);
#pragma unroll 1
    for (int i = 0; i < DEPTH; ++i) issue();
  }

  // ---------------- logits: token group tg (four tokens), router rows [r0, r1); thread t holds inputs 4 t .. 4 t + 3
  const int tgs = (n + 3) / 4, per = G / tgs, tg = b / per;
  const bool part_of = tg < tgs;
  constexpr int RP = 7;  // rows a pass
  const int r0 = part_of ? E1 * (b % per) / per : 0, r1 = part_of ? E1 * (b % per + 1) / per : 0;
  uint2 rw[RP];
  auto router_rows = [&](int rb) {
#pragma unroll
    for (int i = 0; i < RP; ++i)
      rw[i] = rb + i < r1 ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(P.w.router) + (size_t)(rb + i) * H) + threadIdx.x) : make_uint2(0u, 0u);
  };
  router_rows(r0);
  const bool on = lane < n && (!P.live || __ldcg(P.live + lane) != 0);
  const unsigned live = __ballot_sync(0xffffffffu, on);
  float4 xs[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int r = 4 * tg + m;
    xs[m] = part_of && ((live >> r) & 1u) ? __ldcg(reinterpret_cast<const float4*>(P.x + (size_t)r * H) + threadIdx.x) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float4 nw4 = __ldcg(reinterpret_cast<const float4*>(P.w.post_norm) + threadIdx.x);
  const unsigned ep = ld_acquire(&P.ws->epoch), tag = 2u * ep + 1u;  // this call's number
  for (int i = threadIdx.x; i < MAX_E; i += THREADS) ctl.mask[i] = 0u;
  if (threadIdx.x == 0) {
    ctl.abort = 0;
    for (int i = 0; i < 16; ++i) mbar_init(&ctl.arrived[i >> 2][i & 3], 4);
  }
  __syncthreads();
  if (threadIdx.x == THREADS - 1 && atom_add_acq_rel(&P.ws->seen, 1u) == (unsigned)G - 1u) {  // every block has read the number
    P.ws->seen = 0u;
    P.ws->epoch = ep + 1u;
  }
  if (b == 0 && threadIdx.x < MAX_HIT + 8) P.ws->act_done[(ep + 1) & 1][threadIdx.x] = 0u;  // the next call's counters
  if (live == 0u) {
    cp_wait<0>();
    return;
  }
  unsigned* act_done = P.ws->act_done[ep & 1];
  if (part_of) {
    for (int rb = r0; rb < r1 || rb == r0; rb += RP) {
      if (rb != r0) router_rows(rb);
      float v[32];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (4 * tg + m >= n) {
#pragma unroll
          for (int i = 0; i < RP; ++i) v[4 * i + m] = 0.f;
          v[28 + m] = 0.f;
          continue;
        }
        const float4 q = xs[m];
        v[28 + m] = (q.x * q.x + q.y * q.y) + (q.z * q.z + q.w * q.w);
        const float4 h = make_float4(q.x * nw4.x, q.y * nw4.y, q.z * nw4.z, q.w * nw4.w);
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const float a0 = __uint_as_float(rw[i].x << 16), a1 = __uint_as_float(rw[i].x & 0xffff0000u);
          const float a2 = __uint_as_float(rw[i].y << 16), a3 = __uint_as_float(rw[i].y & 0xffff0000u);
          v[4 * i + m] = fmaf(a3, h.w, fmaf(a2, h.z, fmaf(a1, h.y, a0 * h.x)));
        }
      }
      // 32 sums over the warp: lane l ends with sum l
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int j = 0; j < o; ++j) {
          const bool up = lane & o;
          const float keep = up ? v[j + o] : v[j], give = up ? v[j] : v[j + o];
          v[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      red[warp * 33 + lane] = v[0];
      __syncthreads();
      if (warp == 0) {
        float tot = 0.f;
#pragma unroll
        for (int q = 0; q < CW; ++q) tot += red[q * 33 + lane];
        const int m = lane & 3, row = rb + (lane >> 2), tok = 4 * tg + m;
        const float rr = rsqrtf(__shfl_sync(0xffffffffu, tot, 28 + m) / (float)H + P.eps);
        if (lane < 28 && row < r1 && (live >> tok) & 1u) {
          unsigned long long* dst = P.ws->logits + tok * LOGIT_STRIDE + row;
          stack::ll_store(dst, __float_as_uint(tot * rr), tag);
          if (row == E1 - 1) {  // behind the logits: 1 / rms, and a word that evens them out, for they are polled in pairs
            stack::ll_store(dst + 1, __float_as_uint(rr), tag);
            if (E & 1) stack::ll_store(dst + 2, 0u, tag);
          }
        }
        if (lane < 4) ctl.rr_own[4 * tg + lane] = rr;
      }
      __syncthreads();
    }
  }

  // ---------------- digit planes of the tokens in `want`: as many warps a token as there are to spare
  auto convert_tokens = [&](unsigned want, bool squares) {
    const int m = __popc(want), lg = m <= 1 ? 4 : m <= 2 ? 3 : m <= 4 ? 2 : m <= 8 ? 1 : 0, nth = warp >> lg, part = warp & ((1 << lg) - 1);
    if (nth >= m) return;
    unsigned left = want;
    for (int i = 0; i < nth; ++i) left &= left - 1u;
    const int tok = __ffs(left) - 1, its = 16 >> lg, k0 = part * its;
    const float4* xp = reinterpret_cast<const float4*>(P.x + (size_t)tok * H) + 32 * k0 + lane;
    const float4* np = reinterpret_cast<const float4*>(P.w.post_norm) + 32 * k0 + lane;
    unsigned char* plane = planes + 3 * tok * PITCH + 128 * k0;
    float4* mt = meta + tok * MP + 2 * k0;
    float ss = 0.f;
#pragma unroll 4
    for (int i = 0; i < its; ++i) {
      const float4 a = __ldcg(xp + 32 * i), c = __ldcg(np + 32 * i);
      ss += (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w);
      digits4(make_float4(a.x * c.x, a.y * c.y, a.z * c.z, a.w * c.w), plane + 128 * i, PITCH, mt + 2 * i, lane);
    }
    if (squares) {
      ss = warp_sum(ss);
      if (lane == 0) ctl.ss[warp] = ss;
    }
  };
  // The tokens of expert `e` (-1: all live ones, the shared expert), by one warp
  auto list = [&](Seg& s, int e, bool by_place, int base, const float* rr) {
    const unsigned m = e < 0 ? live : ctl.mask[e];
    if (lane < MAX_TOK && (m >> lane) & 1u) {
      const int p = __popc(m & ((1u << lane) - 1u));
      int k = 0;
      if (e >= 0)
        while (k + 1 < topk && ctl.idx[lane][k] != e) ++k;
      s.pos[p] = (unsigned char)(by_place ? base + p : lane);
      s.row[p] = (short)(e < 0 ? n * topk + lane : lane * topk + k);
      s.wt[p] = e < 0 ? sigmoid_f(ctl.sgate[lane]) : ctl.wts[lane][k];
      s.rr[p] = rr[lane];
    }
    if (lane == 0) s.count = __popc(m);
  };

  // A quad's gate/up tiles u, u + 4, ... < end of one expert: each warp a quarter of the inputs; the sums meet in shared memory. With one
  // or two tokens the warps take turns at a tile's end and need not wait for one another: a warp is at most three tiles ahead of the one
  // whose turn it is, its own turn stops it, and four buffers and barriers serve. The finished tiles are counted once for the block, at
  // its end (a fence a tile, which also waits for the copies under way, took as long as the tile).
  int turn = 0;
  auto gate_up = [&](auto tg_c, auto int8_c, const Seg& s, int u, int end) {
    constexpr int TG = decltype(tg_c)::value;
    constexpr bool INT8 = decltype(int8_c)::value;
    const int g = lane >> 2, t = lane & 3;
    float* mine = red + quad * 512;
    if (TG) quad_sync(quad);
    Cols<TG> c;
    cols_set<TG>(c, s, planes, PITCH, meta, MP, lane);
#pragma unroll 1
    for (; u < end; u += 4) {
      Acc<TG> acc = {};
#pragma unroll 1
      for (int sub = 0; sub < (INT8 ? 4 : 2); ++sub) {
        step<TG, INT8>(acc, c, PITCH, 8 * kq + (INT8 ? 2 : 4) * sub, next_slot(), sub, lane);
        used();
      }
      const int tile = u % GU_TILES;
      if constexpr (TG == 0) {
        const float a0 = acc.v[0] + __shfl_xor_sync(0xffffffffu, acc.v[0], 1), a1 = acc.v[1] + __shfl_xor_sync(0xffffffffu, acc.v[1], 1);
        float* buf = mine + (turn & 3) * 128;  // [quarter][16 rows][2 tokens]
        if ((t & 1) == 0) buf[32 * kq + 2 * g + (t >> 1)] = a0, buf[32 * kq + 2 * (g + 8) + (t >> 1)] = a1;
        uint64_t* bar = &ctl.arrived[quad][turn & 3];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        if (kq == (turn & 3)) {
          mbar_wait_hot(bar, (unsigned)(turn >> 2) & 1u, DRB_ERR_GRID_WAIT);
          const int j = (lane >> 1) & 7, p = lane & 1;
          if (lane < 16 && p < s.count) {
            const float* gp = buf + 2 * j + p;
            const float rr = s.rr[p];
            const float gate = ((gp[0] + gp[32]) + (gp[64] + gp[96])) * rr, up = ((gp[16] + gp[48]) + (gp[80] + gp[112])) * rr;
            __stcg(P.act + (size_t)s.row[p] * I + 8 * tile + j, silu_f(gate) * up);
          }
        }
        ++turn;
      } else {
        const int th = threadIdx.x & 127;
#pragma unroll
        for (int i = 0; i < TG; ++i) {
          float* st = mine + 128 * kq;  // [16 rows][8 tokens]
          *reinterpret_cast<float2*>(st + 8 * g + 2 * t) = make_float2(acc.v[4 * i], acc.v[4 * i + 1]);
          *reinterpret_cast<float2*>(st + 8 * (g + 8) + 2 * t) = make_float2(acc.v[4 * i + 2], acc.v[4 * i + 3]);
          quad_sync(quad);
          const int j = th & 7, p = 8 * i + (th >> 3);  // unit of the tile, token
          if (th < 64 && p < s.count) {
            const float* gp = mine + 8 * j + (th >> 3);
            const float rr = s.rr[p];
            const float gate = ((gp[0] + gp[128]) + (gp[256] + gp[384])) * rr, up = ((gp[64] + gp[192]) + (gp[320] + gp[448])) * rr;
            __stcg(P.act + (size_t)s.row[p] * I + 8 * tile + j, silu_f(gate) * up);
          }
          quad_sync(quad);
        }
      }
    }
  };
  using std::integral_constant;
  auto gate_up_any = [&](auto int8_c, const Seg& s, int u, int end) {
    if (s.count <= 2) gate_up(integral_constant<int, 0>(), int8_c, s, u, end);
    else if (TOK <= 8 || s.count <= 8) gate_up(integral_constant<int, 1>(), int8_c, s, u, end);
    else gate_up(integral_constant<int, 2>(), int8_c, s, u, end);
  };

  const bool early = tgs == 1 || shared_block >= 0;
  if (early) {
    convert_tokens(live, tgs > 1);
    if (shared_block >= 0) {
      if (tgs > 1) {  // 1 / rms of the tokens whose logits are other blocks' work
        __syncthreads();
        const int m = __popc(live), lg = m <= 1 ? 4 : m <= 2 ? 3 : m <= 4 ? 2 : m <= 8 ? 1 : 0;
        if (threadIdx.x < MAX_TOK && (live >> threadIdx.x) & 1u) {
          const int at = __popc(live & ((1u << threadIdx.x) - 1u)) << lg;
          float ss = 0.f;
          for (int i = 0; i < 1 << lg; ++i) ss += ctl.ss[at + i];
          ctl.rr_own[threadIdx.x] = rsqrtf(ss / (float)H + P.eps);
        }
        __syncwarp();
      }
      if (warp == 0) list(ctl.seg[0], -1, false, 0, ctl.rr_own);
      __syncthreads();
      gate_up_any(integral_constant<bool, true>(), ctl.seg[0], 4 * shared_block + quad, 4 * shared_block + quad + 1);
    }
  }

  // ---------------- routing: a warp a token; every block for itself
  if ((live >> warp) & 1u) {
    const unsigned long long* src = P.ws->logits + warp * LOGIT_STRIDE;
    const int pieces = (E + 3) / 2;
    uint32_t v[10];
    unsigned need = 0u;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      v[2 * i] = v[2 * i + 1] = 0u;
      if (lane + 32 * i < pieces) need |= 1u << i;
    }
    for (unsigned it = 0; !*abort_flag; ++it) {  // all requests of a round go out before any is looked at
      unsigned long long q[10];
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if ((need >> i) & 1u) stack::ll_load2(src + 2 * (lane + 32 * i), q[2 * i], q[2 * i + 1]);
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (((need >> i) & 1u) && (uint32_t)(q[2 * i] >> 32) == tag && (uint32_t)(q[2 * i + 1] >> 32) == tag) {
          v[2 * i] = (uint32_t)q[2 * i], v[2 * i + 1] = (uint32_t)q[2 * i + 1];
          need &= ~(1u << i);
        }
      if (need == 0u || stack::poll_failed(it, P.poll_limit, abort_flag)) break;
    }
    __syncwarp();
    // larger logit = larger key, never 0; 0: no entry, or taken. A NaN counts as the lowest logit
    uint32_t key[8];
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const int id = 2 * (lane + 32 * (i >> 1)) + (i & 1);
      if (id == E) ctl.sgate[warp] = __uint_as_float(v[i]);
      if (id == E + 1) ctl.rr[warp] = __uint_as_float(v[i]);
      if (i < 8) {
        const uint32_t o = (v[i] & 0x7fffffffu) > 0x7f800000u ? 1u : (v[i] & 0x80000000u) ? ~v[i] : (v[i] | 0x80000000u);
        key[i] = id < E ? o : 0u;
      }
    }
    uint32_t mykey = 0u;
    int myid = 0;
    for (int k = 0; k < topk; ++k) {
      uint32_t bk[4];
      int bi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // ids ascend within a lane: an equal key further on does not win
        const bool second = key[2 * i + 1] > key[2 * i];
        bk[i] = second ? key[2 * i + 1] : key[2 * i], bi[i] = 2 * i + (second ? 1 : 0);
      }
      if (bk[1] > bk[0]) bk[0] = bk[1], bi[0] = bi[1];
      if (bk[3] > bk[2]) bk[2] = bk[3], bi[2] = bi[3];
      if (bk[2] > bk[0]) bk[0] = bk[2], bi[0] = bi[2];
      const int id = 2 * (lane + 32 * (bi[0] >> 1)) + (bi[0] & 1);
      const uint32_t best = __reduce_max_sync(0xffffffffu, bk[0]);
      const unsigned tie = __ballot_sync(0xffffffffu, bk[0] == best);
      int who;
      if (tie & (tie - 1u)) who = (int)__reduce_min_sync(0xffffffffu, bk[0] == best ? (unsigned)id : (unsigned)MAX_E);
      else who = __shfl_sync(0xffffffffu, id, __ffs(tie) - 1);
      const bool winner = id == who;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (winner && bi[0] == i) key[i] = 0u;
      if (lane == k) mykey = best, myid = who;
    }
    const float val = mykey == 1u ? __uint_as_float(0x7fffffffu) : __uint_as_float((mykey & 0x80000000u) ? (mykey & 0x7fffffffu) : ~mykey);
    const float top = __shfl_sync(0xffffffffu, val, 0), ex = lane < topk ? expf(val - top) : 0.f;
    const float sum = warp_sum(ex);
    if (lane < topk) {
      ctl.idx[warp][lane] = myid, ctl.wts[warp][lane] = ex / sum;
      atomicOr(&ctl.mask[myid], 1u << warp);
    }
  }
  __syncthreads();
  // ---------------- experts hit, in ascending order, and this block's runs of their tiles: equal shares of what the tiles cost
  {
    const int ec = threadIdx.x < MAX_E ? __popc(ctl.mask[threadIdx.x]) : 0;
    const unsigned any = __ballot_sync(0xffffffffu, ec > 0), mid = __ballot_sync(0xffffffffu, ec > 2), big = __ballot_sync(0xffffffffu, ec > 8);
    if (warp < 8 && lane == 0) ctl.wsum[warp] = __popc(any) | __popc(mid) << 8 | __popc(big) << 16;
    if (threadIdx.x < 4) ctl.range[threadIdx.x] = -1;
    __syncthreads();
    if (warp < 8) {
      int base = 0, all = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int c = ctl.wsum[w];
        base += w < warp ? c : 0;
        all += c;
      }
      const unsigned below = (1u << lane) - 1u;
      base += __popc(any & below) | __popc(mid & below) << 8 | __popc(big & below) << 16;
      const auto cost = [](int c) { return 4 * (c & 0xff) + 2 * ((c >> 8) & 0xff) + 5 * (c >> 16); };  // tile_cost of so many experts
      const int h = base & 0xff, nhit = all & 0xff, before = cost(base), total = cost(all);
      if (ec > 0) ctl.hit[h] = (unsigned char)threadIdx.x;
      if (threadIdx.x == 0) ctl.nhit = nhit;
      // gate/up: the shared expert's blocks have done SHARED_HEAD_START tiles more, more yet with many tokens
      const int head = SHARED_HEAD_START * tile_cost(__popc(live)), sum = GU_TILES * total;
      const int mine = min(sum, (sum + SHARED_BLOCKS * head) / G * GN);  // what the other blocks do
      const int c = tile_cost(ec);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int bb = b + q;
        const int at = bb <= GN ? mine * bb / GN : mine + (sum - mine) * (bb - GN) / SHARED_BLOCKS;
        const int off = at - GU_TILES * before;
        if (ec > 0 && off >= 0 && off < GU_TILES * c) ctl.range[q] = h * GU_TILES + (off + c - 1) / c;
        if (threadIdx.x == 0 && at >= sum) ctl.range[q] = nhit * GU_TILES;
      }
      // down: the shared expert's tiles first; twice the bytes
      const int cs = tile_cost(__popc(live)) + 4, dsum = DN_TILES * (total + cs);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int at = (int)((long long)dsum * (b + q) / G);
        const int off = at - DN_TILES * (cs + before);
        if (ec > 0 && off >= 0 && off < DN_TILES * c) ctl.range[2 + q] = (h + 1) * DN_TILES + (off + c - 1) / c;
        if (threadIdx.x == 0 && at < DN_TILES * cs) ctl.range[2 + q] = (at + cs - 1) / cs;
        if (threadIdx.x == 0 && at >= dsum) ctl.range[2 + q] = (nhit + 1) * DN_TILES;
      }
    }
    __syncthreads();
  }
  gu0 = ctl.range[0], gu1 = ctl.range[1], dn0 = ctl.range[2], dn1 = ctl.range[3];
  if (gu0 + quad < gu1) {
    ld.u = gu0 + quad;
    aim_gu();
  } else if (dn0 + warp < dn1) {
    ld.u = dn0 + warp;
    aim_dn();
  }
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) issue();

  const int h0 = gu0 / GU_TILES, split = min(gu1, (h0 + 1) * GU_TILES);  // the second expert's tiles start there
  if (gu1 > gu0) {
    const int e0 = ctl.hit[h0], e1 = gu1 > split ? ctl.hit[h0 + 1] : e0;
    if (warp < 2) list(ctl.seg[warp], warp ? e1 : e0, false, 0, ctl.rr);
    if (!early) convert_tokens(ctl.mask[e0] | ctl.mask[e1], false);
  }
  __syncthreads();
  if (gu1 > gu0) {
    gate_up_any(integral_constant<bool, false>(), ctl.seg[0], gu0 + quad, split);
    if (gu1 > split) gate_up_any(integral_constant<bool, false>(), ctl.seg[1], split + ((gu0 + quad - split) & 3), gu1);
  }
  __syncthreads();  // the planes are free
  if (threadIdx.x == 0) {
    __threadfence();
    if (split > gu0) atomicAdd(act_done + h0, (unsigned)(split - gu0));
    if (gu1 > split) atomicAdd(act_done + h0 + 1, (unsigned)(gu1 - split));
    if (shared_block >= 0) atomicAdd(act_done + MAX_HIT, 4u);
  }

  // ---------------- down: digit planes of the (at most two) experts' activations; h = -1: the shared expert
  const int d0 = dn0 / DN_TILES - 1, d1 = dn1 > dn0 ? (dn1 - 1) / DN_TILES - 1 : d0, dsplit = min(dn1, (d0 + 2) * DN_TILES);
  if (warp < 2 && dn1 > dn0) {
    const int h = warp == 0 ? d0 : d1;
    list(ctl.seg[warp], h < 0 ? -1 : ctl.hit[h], true, warp * TOK, ctl.rr);
    if (lane == 0 && !*abort_flag)
      for (unsigned it = 0; ld_acquire(act_done + (h < 0 ? MAX_HIT : h)) < (unsigned)GU_TILES; ++it)
        if (stack::poll_failed(it, P.poll_limit, abort_flag)) break;
  }
  __syncthreads();
  if (dn1 > dn0) {
    const int c0 = ctl.seg[0].count, all = c0 + (d1 != d0 ? ctl.seg[1].count : 0);
    for (int i = warp; i < 4 * all; i += CW) {  // 128 inputs of a token
      const int a = i >> 2, part = i & 3;
      const Seg& s = ctl.seg[a >= c0];
      const int p = a >= c0 ? a - c0 : a, pos = s.pos[p];
      const float4 v = __ldcg(reinterpret_cast<const float4*>(P.act + (size_t)s.row[p] * I) + 32 * part + lane);
      digits4(v, planes + 3 * pos * DPITCH + 128 * part, DPITCH, meta + pos * DMP + 2 * part, lane);
    }
  }
  __syncthreads();

  auto down = [&](auto tg_c, auto int8_c, const Seg& s, int u, int end) {
    constexpr int TG = decltype(tg_c)::value;
    constexpr bool INT8 = decltype(int8_c)::value;
    Cols<TG> c;
    cols_set<TG>(c, s, planes, DPITCH, meta, DMP, lane);
    const int g = lane >> 2, t = lane & 3;
#pragma unroll 1
    for (; u < end; u += CW) {
      Acc<TG> acc = {};
#pragma unroll 1
      for (int sub = 0; sub < (INT8 ? 4 : 2); ++sub) {
        step<TG, INT8>(acc, c, DPITCH, (INT8 ? 2 : 4) * sub, next_slot(), sub, lane);
        used();
      }
      float* out = P.part + 16 * (u % DN_TILES) + g;
      auto put = [&](int p, float lo, float hi) {
        if (p < s.count) {
          float* o = out + (size_t)s.row[p] * H;
          __stcg(o, lo * s.wt[p]);
          __stcg(o + 8, hi * s.wt[p]);
        }
      };
      if constexpr (TG == 0) {
        const float a0 = acc.v[0] + __shfl_xor_sync(0xffffffffu, acc.v[0], 1), a1 = acc.v[1] + __shfl_xor_sync(0xffffffffu, acc.v[1], 1);
        if ((t & 1) == 0) put(t >> 1, a0, a1);
      } else {
#pragma unroll
        for (int i = 0; i < TG; ++i) {
          put(8 * i + 2 * t, acc.v[4 * i], acc.v[4 * i + 2]);
          put(8 * i + 2 * t + 1, acc.v[4 * i + 1], acc.v[4 * i + 3]);
        }
      }
    }
  };
  auto down_any = [&](auto int8_c, const Seg& s, int u, int end) {
    if (s.count <= 2) down(integral_constant<int, 0>(), int8_c, s, u, end);
    else if (TOK <= 8 || s.count <= 8) down(integral_constant<int, 1>(), int8_c, s, u, end);
    else down(integral_constant<int, 2>(), int8_c, s, u, end);
  };
  if (dn1 > dn0) {
    int u = dn0 + warp;
    if (d0 < 0) down_any(integral_constant<bool, true>(), ctl.seg[0], u, dsplit);
    else down_any(integral_constant<bool, false>(), ctl.seg[0], u, dsplit);
    if (u < dsplit) u += (dsplit - u + CW - 1) / CW * CW;
    if (dn1 > dsplit) down_any(integral_constant<bool, false>(), ctl.seg[1], u, dn1);
  }
  cp_wait<0>();

  // ---------------- combine: once every block has written its results, each adds up its share of the outputs, in rank order
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(act_done + MAX_HIT + 1, 1u);
    if (!*abort_flag)
      for (unsigned it = 0; ld_acquire(act_done + MAX_HIT + 1) < (unsigned)G; ++it)
        if (stack::poll_failed(it, P.poll_limit, abort_flag)) break;
  }
  __syncthreads();
  const int outs = n * H / 4, o0 = outs / G * b + min(outs % G, b), o1 = outs / G * (b + 1) + min(outs % G, b + 1);  // in fours
  for (int i = o0 + (int)threadIdx.x; i < o1; i += THREADS) {
    const int r = i / (H / 4), col = 4 * (i % (H / 4));
    if (!((live >> r) & 1u)) continue;
    float4 v[MAX_K];
#pragma unroll
    for (int k = 0; k < MAX_K; ++k)
      v[k] = k < topk ? __ldcg(reinterpret_cast<const float4*>(P.part + (size_t)(r * topk + k) * H + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 x = __ldcg(reinterpret_cast<const float4*>(P.x + (size_t)r * H + col));
    const float4 sh = __ldcg(reinterpret_cast<const float4*>(P.part + (size_t)(n * topk + r) * H + col));
    float4 rest = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < MAX_K; ++k) rest.x += v[k].x, rest.y += v[k].y, rest.z += v[k].z, rest.w += v[k].w;
    float* y = P.y + (size_t)r * H + col;
    y[0] = x.x + sh.x + rest.x, y[1] = x.y + sh.y + rest.y, y[2] = x.z + sh.z + rest.z, y[3] = x.w + sh.w + rest.w;
  }
}

static size_t workspace_bytes(int n, int topk) { return sizeof(Head) + (size_t)n * (topk + 1) * (I + H) * sizeof(float); }

static cudaError_t configure_all() {
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(k_moe_few<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<8>::BYTES)) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(k_moe_few<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<16>::BYTES)) != cudaSuccess) return e;
  if ((e = drb_carveout(k_moe_few<8>)) != cudaSuccess) return e;
  return drb_carveout(k_moe_few<16>);
}

}  // namespace few

extern "C" int drb_moe_few_workspace_bytes(int n, int topk) {
  if (n < 1 || n > few::MAX_TOK || topk < 1 || topk > few::MAX_K) return -1;
  return (int)few::workspace_bytes(n, topk);
}

extern "C" int drb_moe_few(const drb_moe_layer* w, const float* x, float* y, const uint8_t* live, int n, int e, int topk, int h, int i, float eps,
                           void* workspace, cudaStream_t st) {
  if (h != few::H || i != few::I || n < 0 || n > few::MAX_TOK || topk < 1 || topk > few::MAX_K || e < topk || e > few::MAX_E) return -1;
  if (!w || !x || !y || !workspace) return -1;
  const void* ptrs[] = {w->router, w->post_norm, w->gu_q, w->gu_sm, w->d_q, w->d_sm, w->sgu_q, w->sgu_s, w->sd_q, w->sd_s};
  for (const void* p : ptrs)
    if (!p) return -1;
  for (const void* p : ptrs)
    if ((uintptr_t)p & 15) return -3;
  if (((uintptr_t)x & 15) || ((uintptr_t)y & 3) || ((uintptr_t)workspace & 255)) return -3;
  const DrbDevice& dev = drb_device(st);
  if (!dev.ready) return -2;
  if (dev.sms < few::MIN_GRID || dev.sms > few::MAX_GRID) return -1;
  if (n == 0) return 0;
  few::Params p;
  p.w = *w, p.x = x, p.y = y, p.live = live;
  p.ws = static_cast<few::Head*>(workspace);
  p.act = reinterpret_cast<float*>(p.ws + 1);
  p.part = p.act + (size_t)n * (topk + 1) * few::I;
  p.n = n, p.e = e, p.topk = topk, p.eps = eps, p.poll_limit = stack::POLL_LIMIT;
  void* args[] = {&p};
  const bool small = n <= 8;
  const cudaError_t err = cudaLaunchCooperativeKernel(small ? (const void*)few::k_moe_few<8> : (const void*)few::k_moe_few<16>, dim3(dev.sms),
                                                      dim3(few::THREADS), args, small ? few::Shape<8>::BYTES : few::Shape<16>::BYTES, st);
  return err == cudaSuccess ? 0 : (int)err;
}
