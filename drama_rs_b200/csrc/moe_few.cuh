// drb_moe_few: one whole MoE layer for 1 to 16 tokens in ONE cooperative kernel.
//
//   y_r = x_r + sigmoid(l_r[e]) shared(xh_r) + sum_k w_rk expert_{idx_rk}(xh_r),  xh = rmsnorm(x) * nw,  l = R xh
//
// For few tokens nearly every (token, expert) pair has an expert of its own: 1.8 MB of int4 weights that are read once and meet one or
// two rows, so the weights' stream is the floor and what lies between is latency. One block per multiprocessor, all resident:
//
//   logits     block b: some router rows for a group of four tokens; handed over as tagged words (payload, call number), which every
//              block polls, so that every block derives the same routing and the same list of the experts hit
//   digits     the last blocks, sixteen for each eight live tokens, make the tokens' digit planes (below) for all and the shared expert's 64 tiles of
//              gate/up, before the routing exists
//   gate/up    tiles of 8 gate rows and their 8 up rows, [experts hit] x 64 in one list that the blocks share out in runs
//              of equal cost (by tokens, see tile_cost); four warps a tile, 512 inputs each
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
// Queued, 256 experts, top 8: 1 token 18.8 us (18 MB; k_moe_stack takes 10.9 for it), 5 tokens 30.0 (71 MB), 16 tokens 52.8 (185 MB; 5.4 TB/s while gate/up runs). Of the 53: logits 4.1,
// routing and runs 4, first weights and digits 3, gate/up 19, hand-over of the activations 4, down 9, last block 3, combine and launch 6. With a dozen
// runtime divisions on a thread's way 16 tokens took 1 us more, with a fence a tile instead of one a block and equal counts of tiles a block 94 in all.
//
// Every wait is bounded: one that runs out sets the device error word and the block's abort flag, after which no wait of the block
// spins again and the kernel runs to its end.
#pragma once

#include <stddef.h>

#include "gemv.cuh"
#include "moe_decode.cuh"
#include "stack_decode.cuh"

namespace few {

using moe::H;
using moe::I;

constexpr int CW = 16, THREADS = CW * 32;
constexpr int MAX_TOK = 16, MAX_K = 8, MAX_E = 256, MAX_ENT = MAX_TOK * MAX_K;
constexpr int TOK = 8;                          // tokens that a tile meets at once; an expert of more is two entries of the lists below
constexpr int SHARED_BLOCKS = 16;               // blocks of the shared expert's gate/up (for each eight tokens): a tile for each four warps
constexpr int GU_TILES = I / 8, DN_TILES = H / 16;
constexpr int MIN_GRID = 144, MAX_GRID = 1024;  // a block's share of either list spans two entries at most
constexpr int LOGIT_STRIDE = MAX_E + 8;         // words a token

// Workspace: the head is the same for every size, activations and weighted results follow.
struct alignas(256) Head {
  unsigned epoch, seen;  // calls so far; blocks that have read `epoch` in this call
  unsigned pad[62];
  unsigned done[2][MAX_ENT + 8];  // [call parity][counter, see below]
  unsigned long long logits[MAX_TOK * LOGIT_STRIDE];
};
enum Counter { SHARED_ACT = MAX_ENT, BLOCKS = MAX_ENT + 2, DIGITS };  // gate/up tiles of entry i, of the shared expert's halves; blocks
                                                                      // finished; eighths of tokens whose digits are written
static_assert(sizeof(Head) % 256 == 0 && offsetof(Head, logits) % 16 == 0, "aligned sections");

constexpr int SUB = 2048;                // a step of a warp: 16 rows x 128 bytes
constexpr int SLOT = SUB + 256;          // and 16 bytes of scales a row
constexpr int PITCH = H + 64, DPITCH = I + 64;    // bytes between digit planes: neighbouring planes on different banks
constexpr int TOKEN_PLANES = 3 * PITCH;           // a token's digits, in the workspace and in shared memory
constexpr int MP = H / 64 + 1, DMP = I / 64 + 1;  // per 64 inputs, tokens apart: (delta, sum, 65536 delta, 0), see Cols
constexpr int TOKEN_BYTES = TOKEN_PLANES + MP * 16;

constexpr int DEPTH = 4;
constexpr int CTL_BYTES = 3 * 1024, PLANES_BYTES = TOK * TOKEN_PLANES, META_BYTES = TOK * MP * 16, RING_BYTES = CW * DEPTH * SLOT, RED_BYTES = CW * 16 * 8 * 4;
constexpr size_t SMEM_BYTES = CTL_BYTES + PLANES_BYTES + META_BYTES + RING_BYTES + RED_BYTES;
static_assert(8 * MAX_TOK <= SHARED_BLOCKS * CW, "a warp for every eighth of a token");
static_assert(SMEM_BYTES <= 232448 && 2 * 3 * TOK * DPITCH <= PLANES_BYTES && 2 * TOK * DMP * 16 <= META_BYTES, "shared memory");
static_assert((CTL_BYTES + PLANES_BYTES + META_BYTES) % 128 == 0 && SLOT % 128 == 0, "reads of the ring are told apart by their low bits");

struct Seg {  // the tokens of an entry in this block's run
  int count;
  float wt[TOK];           // weight of the expert's result
  float rr[TOK];           // 1 / rms of the token
  short row[TOK];          // row of the activations and of the weighted results
  unsigned char pos[TOK];  // digit planes
};

struct Ctl {
  Seg seg[2];
  int arrived[4][4], finished[4];  // [group of four warps]: warps whose sums of tile t lie in shared memory (t mod 4), tiles finished
  int idx[MAX_TOK][MAX_K];
  float wts[MAX_TOK][MAX_K];
  float sgate[MAX_TOK], rr[MAX_TOK];
  unsigned mask[MAX_E];            // tokens that chose the expert
  unsigned short ent[MAX_ENT];     // expert, + 256: its tokens from the ninth on
  int wsum[8], range[4];           // this block's gate/up tiles and down tiles
  int abort;
};
static_assert(sizeof(Ctl) <= CTL_BYTES, "control block");

DRB_DEV void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
DRB_DEV void cp8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
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

// The weights of a warp's tiles on their way. The next tile of the same expert lies dp (ds) bytes on.
enum Mode { SHARED_GU, GU, DN, OVER };
struct Loader {
  const unsigned char *p;   // this lane's first row and piece of the next step
  const unsigned char *sp;  // this lane's row of scales
  uint32_t at;              // where the pieces go in a slot
  int stride, gap;          // bytes over four rows, and from row r to row r + 8
  int sub, u, uend, ustep, dp, ds, sstep, mode;
};

struct Params {
  drb_moe_layer w;
  const float* x;
  float* y;
  const uint8_t* live;
  Head* ws;
  float *act, *part;
  unsigned char* digits;  // [n] x (TOKEN_PLANES, MP x 16 bytes)
  int n, e, topk;
  float eps;
  unsigned poll_limit;
  // Divisions by what the host knows, by multiplication: of the grid; with one and with two halves of the shared expert, of the other
  // blocks and of the blocks a group of four tokens (a dozen runtime divisions on a thread's way took 2 us)
  unsigned long long by_grid, by_rest[2], by_per[2];
  int per[2];
};
constexpr int RECIP_BITS = 40;  // x / d = x * ceil(2^40 / d) >> 40, exact while x * d < 2^40
DRB_DEV unsigned times(unsigned x, unsigned long long recip) { return (unsigned)((x * recip) >> RECIP_BITS); }

// One warp's share of a tile: 16 rows against the tokens of an entry. TG = 0: one or two tokens, four columns each (three digits); TG = 1: up
// to eight, a column tile per digit. The sums: rows g and g + 8, or rows g (two), g + 8 (two) of tokens 2 t, 2 t + 1.
// Reads of shared memory by its own 32-bit addresses: behind pointers kept in structs the compiler takes generic loads.
template <typename T>
DRB_DEV T lds(uint32_t a) { return *static_cast<const T*>(__cvta_shared_to_generic(a)); }

struct Cols {
  uint32_t b;     // this lane's column: its token's digit planes
  uint32_t m[2];  // delta and sum of the columns whose sums this lane holds. TG = 0: lanes of the third digit take 65536 delta and no sum
  int second;     // TG = 0: weight of this lane's second column
};

DRB_DEV void cols_set(Cols& c, int tg, const Seg& s, uint32_t planes, int pitch, uint32_t meta, int mp, int lane) {
  const int g = lane >> 2, t = lane & 3, last = s.count - 1;
  if (tg == 0) {
    c.b = planes + (3 * s.pos[min(g >> 2, last)] + min(g & 3, 2)) * pitch + 16 * t;
    c.m[0] = meta + s.pos[min(t >> 1, last)] * mp * 16 + 8 * (t & 1);
    c.second = t & 1 ? 0 : 256;
  } else {
    c.b = planes + 3 * s.pos[min(g, last)] * pitch + 16 * t;
    c.m[0] = meta + s.pos[min(2 * t, last)] * mp * 16;
    c.m[1] = meta + s.pos[min(2 * t + 1, last)] * mp * 16;
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
DRB_DEV void group64(float (&acc)[4], const Cols& c, int pitch, int kg, const uint32_t (&a)[8], float s0, float m0, float s1, float m1) {
  if constexpr (TG == 0) {
    const uint4 b = lds<uint4>(c.b + 64 * kg);
    int d[4];
    mma_s8_zero(d, a[0], a[1], a[2], a[3], b.x, b.y);
    gemv::q8::mma_s8(d, a[4], a[5], a[6], a[7], b.z, b.w);
    const float2 m = lds<float2>(c.m[0] + 16 * kg);
    acc[0] = fmaf(s0 * m.x, (float)(d[1] * c.second + d[0]), acc[0]);
    acc[1] = fmaf(s1 * m.x, (float)(d[3] * c.second + d[2]), acc[1]);
    if (MIN) acc[0] = fmaf(m0, m.y, acc[0]), acc[1] = fmaf(m1, m.y, acc[1]);
  } else {
    int d[3][4];
#pragma unroll
    for (int l = 0; l < 3; ++l) {
      const uint4 b = lds<uint4>(c.b + l * pitch + 64 * kg);
      mma_s8_zero(d[l], a[0], a[1], a[2], a[3], b.x, b.y);
      gemv::q8::mma_s8(d[l], a[4], a[5], a[6], a[7], b.z, b.w);
    }
    const float2 c0 = lds<float2>(c.m[0] + 16 * kg), c1 = lds<float2>(c.m[1] + 16 * kg);
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = fmaf((float)d[2][j], 65536.f, (float)(d[1][j] * 256 + d[0][j]));
    acc[0] = fmaf(s0, f[0] * c0.x, acc[0]), acc[1] = fmaf(s0, f[1] * c1.x, acc[1]);
    acc[2] = fmaf(s1, f[2] * c0.x, acc[2]), acc[3] = fmaf(s1, f[3] * c1.x, acc[3]);
    if (MIN) {
      acc[0] = fmaf(m0, c0.y, acc[0]), acc[1] = fmaf(m0, c1.y, acc[1]);
      acc[2] = fmaf(m1, c0.y, acc[2]), acc[3] = fmaf(m1, c1.y, acc[3]);
    }
  }
}

// One step of 128 bytes a row: 256 int4 or 128 int8 inputs from group kg on. r0: this lane's place in the slot (see `issue`), sc: in its scales.
template <int TG, bool INT8>
DRB_DEV void step(float (&acc)[4], const Cols& c, int pitch, int kg, uint32_t r0, uint32_t sc) {
  uint32_t a[8];
  if constexpr (INT8) {
    const float s0 = __half2float(lds<__half>(sc)), s1 = __half2float(lds<__half>(sc + 128));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 u = lds<uint4>(r0 ^ (64 * q)), v = lds<uint4>((r0 ^ (64 * q)) + 1024);
      a[0] = prmt(u.x, u.y, 0x6420u), a[1] = prmt(v.x, v.y, 0x6420u), a[2] = prmt(u.x, u.y, 0x7531u), a[3] = prmt(v.x, v.y, 0x7531u);
      a[4] = prmt(u.z, u.w, 0x6420u), a[5] = prmt(v.z, v.w, 0x6420u), a[6] = prmt(u.z, u.w, 0x7531u), a[7] = prmt(v.z, v.w, 0x7531u);
      group64<TG, false>(acc, c, pitch, kg + q, a, s0, 0.f, s1, 0.f);
    }
  } else {
    const uint4 w0 = lds<uint4>(sc), w1 = lds<uint4>(sc + 128);
    const uint32_t sm0[4] = {w0.x, w0.y, w0.z, w0.w}, sm1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint2 u = lds<uint2>(r0 ^ (32 * q)), v = lds<uint2>((r0 ^ (32 * q)) + 1024);
      a[0] = u.x & 0x0F0F0F0Fu, a[1] = v.x & 0x0F0F0F0Fu, a[2] = (u.x >> 4) & 0x0F0F0F0Fu, a[3] = (v.x >> 4) & 0x0F0F0F0Fu;
      a[4] = u.y & 0x0F0F0F0Fu, a[5] = v.y & 0x0F0F0F0Fu, a[6] = (u.y >> 4) & 0x0F0F0F0Fu, a[7] = (v.y >> 4) & 0x0F0F0F0Fu;
      const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&sm0[q])), f1 = __half22float2(*reinterpret_cast<const __half2*>(&sm1[q]));
      group64<TG, true>(acc, c, pitch, kg + q, a, f0.x, f0.y, f1.x, f1.y);
    }
  }
}

// What a tile costs, in quarters of one with one or two tokens: instructions, which grow with the column tiles.
DRB_DEV int tile_cost(int count) { return count <= 2 ? 4 : 6; }
constexpr int SHARED_HEAD_START = 8;  // the shared expert's gate/up, in tiles of its number of tokens that its blocks do less of

__global__ void __launch_bounds__(THREADS, 1) k_moe_few(Params P) {
  extern __shared__ __align__(128) unsigned char dyn[];
  Ctl& ctl = *reinterpret_cast<Ctl*>(dyn);
  unsigned char* planes = dyn + CTL_BYTES;
  float4* meta = reinterpret_cast<float4*>(planes + PLANES_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp >> 2, kq = warp & 3;
  float* red = reinterpret_cast<float*>(planes + PLANES_BYTES + META_BYTES + RING_BYTES);
  const uint32_t ring = smem_u32(planes) + PLANES_BYTES + META_BYTES + warp * DEPTH * SLOT, ring_end = ring + DEPTH * SLOT;
  const int n = P.n, E = P.e, topk = P.topk, E1 = E + 1;
  const int G = (int)gridDim.x, b = (int)blockIdx.x;
  volatile int* abort_flag = &ctl.abort;
  const bool on = lane < n && (!P.live || __ldcg(P.live + lane) != 0);
  const unsigned live = __ballot_sync(0xffffffffu, on);
  const int nlive = __popc(live), halves = nlive > TOK ? 2 : 1;
  const int GN = G - halves * SHARED_BLOCKS, shared_block = b - GN;  // >= 0: one of the shared expert's blocks

  // ---------------- the weights' stream
  Loader ld;
  ld.mode = OVER;
  uint32_t slot = ring;  // the next step's place
  auto point = [&](const void* w, const void* s, bool int8, int row_bytes, int row0, int gap_rows, int off, int srow_bytes, int soff, int rows_on) {
    ld.stride = 4 * row_bytes, ld.gap = gap_rows * row_bytes;
    const int r = lane >> 3, c = lane & 7, sr = lane & 15;
    // Piece c (16 bytes) of row r lies where reads of eight rows at once meet no bank twice: int4 rows are read 32 bytes (four
    // lanes) at a time, int8 rows 64.
    ld.at = r * 128 + 16 * (int8 ? c ^ ((r & 1) << 2) : c ^ ((r & 3) << 1));
    ld.p = static_cast<const unsigned char*>(w) + (size_t)(row0 + r) * row_bytes + off + 16 * c;
    // 16 bytes of scales a row: int4 a step's; int8 the ones around the tile's, of one row or two
    ld.sp = static_cast<const unsigned char*>(s) + (((size_t)(row0 + (sr < 8 ? sr : sr - 8 + gap_rows)) * srow_bytes + soff) & ~(size_t)15);
    ld.sub = int8 ? 4 : 2, ld.sstep = int8 ? 0 : 16;
    ld.dp = rows_on * row_bytes - 128 * ld.sub, ld.ds = rows_on * srow_bytes - ld.sub * ld.sstep;
  };
  int gu0 = 0, gu1 = 0, dn0 = 0, dn1 = 0;  // this block's tiles: entry x GU_TILES; shared halves, then entry x DN_TILES
  auto aim_gu = [&]() {
    const int h = ld.u / GU_TILES;
    ld.mode = GU, ld.ustep = 4, ld.uend = min(gu1, (h + 1) * GU_TILES);
    point(P.w.gu_q, P.w.gu_sm, false, H / 2, (ctl.ent[h] & 255) * 2 * I + 8 * (ld.u % GU_TILES), I, kq * 256, H / 64 * 4, kq * 32, 32);
  };
  auto aim_dn = [&]() {
    const int h = ld.u / DN_TILES - halves, row0 = 16 * (ld.u % DN_TILES);
    ld.mode = DN, ld.ustep = CW, ld.uend = min(dn1, (h + halves + 1) * DN_TILES);
    if (h < 0) point(P.w.sd_q, P.w.sd_s, true, I, row0, 8, 0, I / 128 * 2, 0, 16 * CW);
    else point(P.w.d_q, P.w.d_sm, false, I / 2, (ctl.ent[h] & 255) * H + row0, 8, 0, I / 64 * 4, 0, 16 * CW);
  };
  auto next_run = [&]() {  // behind the last tile of an expert
    if (ld.mode == GU && ld.u < gu1) return aim_gu();
    if (ld.mode == GU) ld.mode = DN, ld.u = dn0 + warp;
    if (ld.mode == DN && ld.u < dn1) return aim_dn();
    ld.mode = OVER;
  };
  auto issue = [&](uint32_t dst) {  // requests the next step, if there is one
    if (ld.mode != OVER) {
      const uint32_t d = dst + ld.at;
      const unsigned char* q = ld.p + ld.gap;
      cp16(d, ld.p);
      cp16(d + 512, ld.p + ld.stride);
      cp16(d + 1024, q);
      cp16(d + 1536, q + ld.stride);
      cp16(dst + SUB + 16 * (lane & 15), ld.sp);  // both halves of the warp the same
      ld.p += 128, ld.sp += ld.sstep;
      if (--ld.sub == 0) {
        ld.u += ld.ustep;
        if (ld.u < ld.uend) ld.sub = ld.sstep ? 2 : 4, ld.p += ld.dp, ld.sp += ld.ds;
        else next_run();
      }
    }
    cp_commit();
  };
  auto prime = [&]() {  // the ring is empty and `slot` at its next place
#pragma unroll 1
    for (int i = 0; i < DEPTH; ++i) {
      issue(slot);
      slot = slot + SLOT == ring_end ? ring : slot + SLOT;
    }
  };
  // ---------------- logits: token group tg (four tokens), router rows [r0, r1); thread t holds inputs 4 t .. 4 t + 3. The rows come by copies
  // of each thread's own eight bytes into the planes, which are free so far; behind them the shared expert's weights are requested.
  const int tgs = (n + 3) >> 2, per = P.per[halves - 1], tg = shared_block < 0 ? (int)times(b, P.by_per[halves - 1]) : tgs;
  const int part = b - tg * per;
  const int r0 = tg < tgs ? times(E1 * part, P.by_per[halves - 1]) : 0, r1 = tg < tgs ? times(E1 * (part + 1), P.by_per[halves - 1]) : 0;
  {
    const unsigned char* src = static_cast<const unsigned char*>(P.w.router) + 8 * threadIdx.x;
    for (int r = r0; r < r1; ++r) cp8(smem_u32(planes + (r - r0) * 2 * H + 8 * threadIdx.x), src + (size_t)r * 2 * H);
    cp_commit();
  }
  if (shared_block >= 0) {
    ld.mode = SHARED_GU, ld.u = 0, ld.ustep = 1, ld.uend = 1;
    point(P.w.sgu_q, P.w.sgu_s, true, H, 8 * (4 * (shared_block % SHARED_BLOCKS) + quad), I, kq * 512, H / 128 * 2, kq * 8, 0);
  }
  prime();  // empty groups in the other blocks
  float4 xs[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int r = 4 * tg + m;
    xs[m] = r < n && ((live >> r) & 1u) ? __ldcg(reinterpret_cast<const float4*>(P.x + (size_t)r * H) + threadIdx.x) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float4 nw4 = __ldcg(reinterpret_cast<const float4*>(P.w.post_norm) + threadIdx.x);
  const unsigned ep = ld_acquire(&P.ws->epoch), tag = 2u * ep + 1u;  // this call's number
  if (threadIdx.x < MAX_E) ctl.mask[threadIdx.x] = 0u;
  if (threadIdx.x == 0) ctl.abort = 0;
  if (threadIdx.x < 20) (&ctl.arrived[0][0])[threadIdx.x] = 0;
  unsigned* done = P.ws->done[ep & 1];
  // Digits: the shared expert's blocks, which have no logits to make, turn the tokens into them for all blocks, 256 inputs a warp
  const int item = shared_block + warp * halves * SHARED_BLOCKS, itok = item >> 3;
  if (shared_block >= 0 && item < 8 * n && ((live >> itok) & 1u)) {
    unsigned char* dst = P.digits + (size_t)itok * TOKEN_BYTES;
    const float4* xp = reinterpret_cast<const float4*>(P.x + (size_t)itok * H) + 64 * (item & 7) + lane;
    const float4* np = reinterpret_cast<const float4*>(P.w.post_norm) + 64 * (item & 7) + lane;
    const float4 x0 = __ldcg(xp), x1 = __ldcg(xp + 32), w0 = __ldcg(np), w1 = __ldcg(np + 32);
    float4* mt = reinterpret_cast<float4*>(dst + TOKEN_PLANES) + 4 * (item & 7);
    dst += 256 * (item & 7);
    digits4(make_float4(x0.x * w0.x, x0.y * w0.y, x0.z * w0.z, x0.w * w0.w), dst, PITCH, mt, lane);
    digits4(make_float4(x1.x * w1.x, x1.y * w1.y, x1.z * w1.z, x1.w * w1.w), dst + 128, PITCH, mt + 2, lane);
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      atomicAdd(done + DIGITS, 1u);
    }
  }

  // Four sums over the warp (one for each token): lane l gets the one of token l >> 3
  auto sums4 = [&](float v0, float v1, float v2, float v3) {
    const bool hi = lane & 16, mid = lane & 8;
    const float a = (hi ? v2 : v0) + __shfl_xor_sync(0xffffffffu, hi ? v0 : v2, 16);
    const float c = (hi ? v3 : v1) + __shfl_xor_sync(0xffffffffu, hi ? v1 : v3, 16);
    float s = (mid ? c : a) + __shfl_xor_sync(0xffffffffu, mid ? a : c, 8);
    s += __shfl_xor_sync(0xffffffffu, s, 4);
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    return s + __shfl_xor_sync(0xffffffffu, s, 1);
  };
  if (tg < tgs) {
    float sq[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float4& q = xs[m];
      sq[m] = (q.x * q.x + q.y * q.y) + (q.z * q.z + q.w * q.w);
      q = make_float4(q.x * nw4.x, q.y * nw4.y, q.z * nw4.z, q.w * nw4.w);
    }
    const float s = sums4(sq[0], sq[1], sq[2], sq[3]);
    if ((lane & 7) == 0) red[4 * warp + (lane >> 3)] = s;  // [row, squares first][warp][token]
  }
  cp_wait<DEPTH>();  // the router's rows
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    const uint2 w = *reinterpret_cast<const uint2*>(planes + (r - r0) * 2 * H + 8 * threadIdx.x);
    const float a0 = __uint_as_float(w.x << 16), a1 = __uint_as_float(w.x & 0xffff0000u);
    const float a2 = __uint_as_float(w.y << 16), a3 = __uint_as_float(w.y & 0xffff0000u);
    float v[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) v[m] = fmaf(a3, xs[m].w, fmaf(a2, xs[m].z, fmaf(a1, xs[m].y, a0 * xs[m].x)));
    const float s = sums4(v[0], v[1], v[2], v[3]);
    if ((lane & 7) == 0) red[64 * (r - r0 + 1) + 4 * warp + (lane >> 3)] = s;
  }
  __syncthreads();
  if (threadIdx.x == THREADS - 1 && atom_add_acq_rel(&P.ws->seen, 1u) == (unsigned)G - 1u) {  // every block has read the number
    P.ws->seen = 0u;
    P.ws->epoch = ep + 1u;
  }
  if (b == 0 && threadIdx.x < MAX_ENT + 8) P.ws->done[(ep + 1) & 1][threadIdx.x] = 0u;  // the next call's counters
  if (live == 0u) {
    cp_wait<0>();
    return;
  }
  for (int i = threadIdx.x; i < 4 * (r1 - r0); i += THREADS) {  // router row r0 + i / 4, token i % 4 of the group
    const int m = i & 3, row = r0 + (i >> 2), tok = 4 * tg + m;
    float ss = 0.f, v = 0.f;
#pragma unroll
    for (int q = 0; q < CW; ++q) ss += red[4 * q + m], v += red[64 * ((i >> 2) + 1) + 4 * q + m];
    const float rr = rsqrtf(ss / (float)H + P.eps);
    if ((live >> tok) & 1u) {
      unsigned long long* dst = P.ws->logits + tok * LOGIT_STRIDE + row;
      stack::ll_store(dst, __float_as_uint(v * rr), tag);
      if (row == E1 - 1) {  // behind the logits: 1 / rms, and a word that evens them out, for they are polled in pairs
        stack::ll_store(dst + 1, __float_as_uint(rr), tag);
        if (E & 1) stack::ll_store(dst + 2, 0u, tag);
      }
    }
  }

  // The tokens of an entry: `code` as in ctl.ent, -1, -2: the shared expert's halves
  auto tokens = [&](int code) {
    unsigned m = code < 0 ? live : ctl.mask[code & 255];
    const bool second = code < 0 ? code == -2 : code > 255;
    if (__popc(m) > TOK) {
      unsigned rest = m;
      for (int i = 0; i < TOK; ++i) rest &= rest - 1u;
      m = second ? rest : m ^ rest;
    }
    return m;
  };
  // They become a segment, with digit planes from `base` on; by one warp
  auto list = [&](Seg& s, int code, int base) {
    const unsigned m = tokens(code);
    if ((m >> lane) & 1u) {
      const int p = __popc(m & ((1u << lane) - 1u));
      int k = 0;
      if (code >= 0)
        while (k + 1 < topk && ctl.idx[lane][k] != (code & 255)) ++k;
      s.pos[p] = (unsigned char)(base + p);
      s.row[p] = (short)(code < 0 ? n * topk + lane : lane * topk + k);
      s.wt[p] = code < 0 ? sigmoid_f(ctl.sgate[lane]) : ctl.wts[lane][k];
      s.rr[p] = ctl.rr[lane];
    }
    if (lane == 0) s.count = __popc(m);
  };
  auto await = [&](int counter, unsigned count) {
    if (!*abort_flag)
      for (unsigned it = 0; ld_acquire(done + counter) < count; ++it)
        if (stack::poll_failed(it, P.poll_limit, abort_flag)) break;
  };
  // Their digits (which are written) are requested into planes from `base` on
  auto copy_tokens = [&](unsigned want, int base) {
    const int i = threadIdx.x;
    if (i < TOKEN_BYTES / 16)
      for (; want; want &= want - 1u, ++base) {
        const uint32_t dst = i < TOKEN_PLANES / 16 ? smem_u32(planes + base * TOKEN_PLANES) + 16 * i : smem_u32(meta + base * MP) + 16 * i - TOKEN_PLANES;
        cp16(dst, P.digits + (size_t)(__ffs(want) - 1) * TOKEN_BYTES + 16 * i);
      }
    cp_commit();
  };

  // ---------------- three stages with the same body: the shared expert's gate/up (its blocks only, before the routing is known), gate/up, down.
  // Each gets its tiles' tokens as digit planes and goes through its run of tiles, of two entries at most.
  int turn = 0;
#pragma unroll 1
  for (int stage = shared_block >= 0 ? 0 : 1; stage < 3; ++stage) {
    int first = 0, split = 0, end = 0;  // tiles: [first, split) of one entry, [split, end) of the next
    int code1 = 0;                      // the second one, whose tokens' planes follow when the first one is through
    bool later = false;
    if (stage == 0) {
      const int code = -1 - shared_block / SHARED_BLOCKS;
      if (warp == 0) {
        if ((live >> lane) & 1u) {  // 1 / rms, behind the logits
          uint32_t out[2];
          stack::ll_poll<1>(P.ws->logits + lane * LOGIT_STRIDE + ((E + 1) & ~1), tag, out, P.poll_limit, abort_flag);
          ctl.rr[lane] = __uint_as_float(out[E & 1 ? 0 : 1]);
        }
        __syncwarp();
        list(ctl.seg[0], code, 0);
      }
      first = 4 * (shared_block % SHARED_BLOCKS), split = end = first + 4;
      if (threadIdx.x == THREADS - 1) await(DIGITS, 8 * nlive);
      __syncthreads();
      copy_tokens(tokens(code), 0);
      cp_wait<0>();
    } else if (stage == 1) {
      if (threadIdx.x == THREADS - 1) await(DIGITS, 8 * nlive);  // for the copies below
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
        // Larger logit = larger key, never 0; 0: no entry. A NaN counts as the lowest logit.
        uint32_t key[8], low = 0u;
#pragma unroll
        for (int i = 0; i < 10; ++i) {
          const int id = 2 * (lane + 32 * (i >> 1)) + (i & 1);
          if (id == E) ctl.sgate[warp] = __uint_as_float(v[i]);
          if (id == E + 1) ctl.rr[warp] = __uint_as_float(v[i]);
          if (i < 8) {
            const uint32_t o = (v[i] & 0x7fffffffu) > 0x7f800000u ? 1u : (v[i] & 0x80000000u) ? ~v[i] : (v[i] | 0x80000000u);
            key[i] = id < E ? o : 0u;
            low = max(low, key[i]);
          }
        }
        // The smallest of eight groups' maxima (four lanes each) bounds the k-th largest from below, k <= 8. The entries from it on, two or three
        // dozen of 256, go to a list (in the planes, which are free), and everyone's rank in it is counted.
        low = max(low, __shfl_xor_sync(0xffffffffu, low, 1));
        low = max(low, __shfl_xor_sync(0xffffffffu, low, 2));
        low = max(__reduce_min_sync(0xffffffffu, low), 1u);
        uint2* cand = reinterpret_cast<uint2*>(planes) + MAX_E * warp;
        int count = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool in = key[i] >= low;
          const unsigned bal = __ballot_sync(0xffffffffu, in);
          if (in) cand[count + __popc(bal & ((1u << lane) - 1u))] = make_uint2(key[i], 2 * (lane + 32 * (i >> 1)) + (i & 1));
          count += __popc(bal);
        }
        __syncwarp();
        uint2* best = reinterpret_cast<uint2*>(planes + CW * MAX_E * 8) + MAX_K * warp;
        for (int c = lane; c < count; c += 32) {
          const uint2 me = cand[c];
          int rank = 0;
#pragma unroll 4
          for (int j = 0; j < count; ++j) {
            const uint2 o = cand[j];
            rank += o.x > me.x || (o.x == me.x && o.y < me.y) ? 1 : 0;
          }
          if (rank < topk) best[rank] = me;
        }
        __syncwarp();
        const uint2 won = best[lane & (MAX_K - 1)];
        const uint32_t mykey = won.x;
        const int myid = (int)won.y;
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
        // an entry; with more than two tokens; a second entry; with more than two tokens
        const unsigned any = __ballot_sync(0xffffffffu, ec > 0), mid = __ballot_sync(0xffffffffu, ec > 2);
        const unsigned two = __ballot_sync(0xffffffffu, ec > TOK), big = __ballot_sync(0xffffffffu, ec > TOK + 2);
        if (warp < 8 && lane == 0) ctl.wsum[warp] = (__popc(any) + __popc(two)) | (__popc(mid) + __popc(big)) << 8;
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
          base += (__popc(any & below) + __popc(two & below)) | (__popc(mid & below) + __popc(big & below)) << 8;
          const int h = base & 0xff, nent = all & 0xff, before = 4 * h + 2 * (base >> 8), total = 4 * nent + 2 * (all >> 8);  // tile_cost of so many
          const int c0 = tile_cost(ec), c1 = tile_cost(ec - TOK);
          if (ec > 0) ctl.ent[h] = (unsigned short)threadIdx.x;
          if (ec > TOK) ctl.ent[h + 1] = (unsigned short)(threadIdx.x + 256);
          // gate/up: the shared expert's blocks have done SHARED_HEAD_START tiles already; down: its tiles come first, with twice the bytes
          const int lc = tile_cost(nlive), cs = lc + 4, ns = halves * SHARED_BLOCKS;
          const int sum = GU_TILES * total, dsum = DN_TILES * (total + halves * cs), mine = min(sum, (int)times(sum + ns * SHARED_HEAD_START * lc, P.by_grid) * GN);
          // lane q < 4: border q of this block (gate/up from, to; down from, to) on the scale of costs
          const int bb = b + (lane & 1);
          const bool late = !(lane & 2) && bb > GN;
          const unsigned num = lane & 2 ? dsum * bb : late ? (sum - mine) * (bb - GN) : mine * bb;
          const int border = late ? mine + (int)(num / SHARED_BLOCKS >> (halves - 1)) : (int)times(num, lane & 2 ? P.by_grid : P.by_rest[halves - 1]);
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            const int at = __shfl_sync(0xffffffffu, border, q), scale = q < 2 ? GU_TILES : DN_TILES, heads = q < 2 ? 0 : halves, lead = heads * DN_TILES * cs;
            const int off = at - lead - scale * before;
            // gate/up in whole rounds of the four groups of warps. Costs are 4 and 6: a third by multiplication (below 2^16)
            const int round = q < 2 ? 4 : 1, lr = q < 2 ? 2 : 0;
            const auto tiles = [&](int o, int c) { return (c == 4 ? (o + 4 * round - 1) >> (2 + lr) : ((o + 6 * round - 1) >> (1 + lr)) * 43691 >> 17) << lr; };
            if (ec > 0 && off >= 0 && off < scale * c0) ctl.range[q] = (h + heads) * scale + tiles(off, c0);
            if (ec > TOK && off >= scale * c0 && off < scale * (c0 + c1)) ctl.range[q] = (h + heads + 1) * scale + tiles(off - scale * c0, c1);
            if (threadIdx.x == 0 && at < lead) ctl.range[q] = cs == 8 ? (at + 7) >> 3 : (at + 9) / 10;
            if (threadIdx.x == 0 && at >= lead + scale * total) ctl.range[q] = (nent + heads) * scale;
          }
        }
        __syncthreads();
      }
      gu0 = ctl.range[0], gu1 = ctl.range[1], dn0 = ctl.range[2], dn1 = ctl.range[3];
      const int h0 = gu0 / GU_TILES;
      first = gu0, end = gu1, split = min(gu1, (h0 + 1) * GU_TILES);
      unsigned m0 = 0u, m1 = 0u;
      if (first < end) {
        m0 = tokens(ctl.ent[h0]);
        if (split < end) m1 = tokens(code1 = ctl.ent[h0 + 1]);
      }
      later = __popc(m0) + __popc(m1) > TOK;
      ld.mode = GU, ld.u = gu0 + quad;
      if (ld.u < gu1) aim_gu();
      else next_run();
      prime();
      copy_tokens(m0, 0);
      if (!later) copy_tokens(m1, __popc(m0));
      if (warp == 0 && first < end) list(ctl.seg[0], ctl.ent[h0], 0);
      if (warp == 1 && split < end) list(ctl.seg[1], code1, later ? 0 : __popc(m0));
      cp_wait<0>();
    } else {
      // the activations of this block's gate/up run are written: counted once for the block (a fence a tile, which also waits for the copies
      // under way, took as long as the tile)
      if (threadIdx.x == 0) {
        const int h0 = gu0 / GU_TILES, sp = min(gu1, (h0 + 1) * GU_TILES);
        __threadfence();
        if (sp > gu0) atomicAdd(done + h0, (unsigned)(sp - gu0));
        if (gu1 > sp) atomicAdd(done + h0 + 1, (unsigned)(gu1 - sp));
        if (shared_block >= 0) atomicAdd(done + SHARED_ACT + shared_block / SHARED_BLOCKS, 4u);
      }
      const int h0 = dn0 / DN_TILES - halves;  // below 0: the shared expert
      first = dn0, end = dn1, split = min(dn1, (h0 + halves + 1) * DN_TILES);
      if (warp < 2 && (warp ? split : first) < end) {
        const int h = h0 + warp, code = h < 0 ? -1 - (h + halves) : ctl.ent[h];
        list(ctl.seg[warp], code, warp * TOK);
        if (lane == 0) await(h < 0 ? SHARED_ACT + h + halves : h, GU_TILES);
      }
    }
    const bool dn = stage == 2;
    const int pitch = dn ? DPITCH : PITCH, mp = dn ? DMP : MP;
    if (dn) __syncthreads();
    if (dn && first < end) {  // the activations as digits: a warp takes 128 of a token at a time, two of them on the way
      const int c0 = ctl.seg[0].count, all = 4 * (c0 + (split < end ? ctl.seg[1].count : 0));
#pragma unroll 1
      for (int i0 = warp; i0 < all; i0 += 2 * CW) {
        float4 v[2];
        int at[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = min(i0 + j * CW, all - 1), a = i >> 2;  // the last one twice, if need be
          const Seg& s = ctl.seg[a >= c0];
          const int p = a >= c0 ? a - c0 : a;
          at[j] = s.pos[p] * 4 + (i & 3);
          v[j] = __ldcg(reinterpret_cast<const float4*>(P.act + (size_t)s.row[p] * I) + 32 * (i & 3) + lane);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
          digits4(v[j], planes + 3 * (at[j] >> 2) * DPITCH + 128 * (at[j] & 3), DPITCH, meta + (at[j] >> 2) * DMP + 2 * (at[j] & 3), lane);
      }
    }
    __syncthreads();

    const int g = lane >> 2, t = lane & 3, nw = dn ? CW : 4;  // tiles go round the warps, or round the groups of four
    const int kg0 = dn ? 0 : 8 * kq;
    // this lane's rows g and g + 8 in a slot (see `point`), and their scales
    const uint32_t at4 = g * 128 + 32 * (g & 3) + 8 * t, at8 = g * 128 + 64 * (g & 1) + 16 * t, sc8 = SUB + 16 * g + 8 * ((dn ? g : kq) & 1);
    int u = first + (dn ? warp : quad);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int stop = k ? end : split;
      if (k == 1) {
        if (split >= end) break;
        if (later) {
          __syncthreads();
          copy_tokens(tokens(code1), 0);
          cp_wait<0>();
          __syncthreads();
        }
      }
      const Seg& s = ctl.seg[k];
      const bool int8 = stage == 0 || (dn && stop <= halves * DN_TILES);
      const int tg = s.count <= 2 ? 0 : 1;
      float* mine = red + quad * 512;
      if (!dn && tg) quad_sync(quad);
      Cols c;
      if (first < end) cols_set(c, tg, s, smem_u32(planes), pitch, smem_u32(meta), mp, lane);
      const int nsub = int8 ? 4 : 2, kgs = int8 ? 2 : 4;
      const uint32_t at = int8 ? at8 : at4, sc = int8 ? sc8 : SUB + 16 * g, scs = int8 ? 2 : 0;
#pragma unroll 1
      for (; u < stop; u += nw) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        // One copy of the loop's requests for the four kinds of steps: the kernel runs through its code once or a few times, and every kilobyte of
        // it comes from L2
#pragma unroll 1
        for (int sub = 0; sub < nsub; ++sub) {
          cp_wait<DEPTH - 1>();
          __syncwarp();
          const int kg = kg0 + kgs * sub;
          const uint32_t r = slot + at, q = slot + sc + scs * sub;
          if (!int8) {
            if (tg == 0) step<0, false>(acc, c, pitch, kg, r, q);
            else step<1, false>(acc, c, pitch, kg, r, q);
          } else {
            if (tg == 0) step<0, true>(acc, c, pitch, kg, r, q);
            else step<1, true>(acc, c, pitch, kg, r, q);
          }
          __syncwarp();
          issue(slot);
          slot = slot + SLOT == ring_end ? ring : slot + SLOT;
        }
        if (tg == 0) {  // the third digit's lanes join the first two's: rows g, g + 8 of token t >> 1
          acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 1);
          acc[1] += __shfl_xor_sync(0xffffffffu, acc[1], 1);
        }
        if (dn) {
          // 16 output rows of every token, weighted
          auto put = [&](int p, float lo, float hi) {
            if (p < s.count) {
              float* o = P.part + (size_t)s.row[p] * H + 16 * (u % DN_TILES) + g;
              __stcg(o, lo * s.wt[p]);
              __stcg(o + 8, hi * s.wt[p]);
            }
          };
          if (tg == 0) {
            if ((t & 1) == 0) put(t >> 1, acc[0], acc[1]);
          } else {
            put(2 * t, acc[0], acc[2]);
            put(2 * t + 1, acc[1], acc[3]);
          }
          continue;
        }
        // gate/up: each of the four warps holds the sums over a quarter of the inputs
        float* act = P.act + 8 * (u % GU_TILES);
        if (tg == 0) {
          // The last of the four to arrive finishes the tile; the others go on, three tiles ahead of the last finished one at most, for there
          // are four buffers.
          float* buf = mine + (turn & 3) * 128;  // [quarter][16 rows][2 tokens]
          for (unsigned it = 0; turn - *static_cast<volatile int*>(&ctl.finished[quad]) > 3; ++it)
            if (stack::poll_failed(it, P.poll_limit, abort_flag)) break;
          __syncwarp();
          if ((t & 1) == 0) buf[32 * kq + 2 * g + (t >> 1)] = acc[0], buf[32 * kq + 2 * (g + 8) + (t >> 1)] = acc[1];
          __syncwarp();
          int before = 0;
          if (lane == 0) {
            __threadfence_block();
            before = atomicAdd(&ctl.arrived[quad][turn & 3], 1);
            __threadfence_block();
          }
          ++turn;
          if ((__shfl_sync(0xffffffffu, before, 0) & 3) == 3) {
            const int j = (lane >> 1) & 7, p = lane & 1;
            if (lane < 16 && p < s.count) {
              const float* gp = buf + 2 * j + p;
              const float rr = s.rr[p];
              const float gate = ((gp[0] + gp[32]) + (gp[64] + gp[96])) * rr, up = ((gp[16] + gp[48]) + (gp[80] + gp[112])) * rr;
              __stcg(act + (size_t)s.row[p] * I + j, silu_f(gate) * up);
            }
            __syncwarp();
            if (lane == 0) *static_cast<volatile int*>(&ctl.finished[quad]) = turn;
          }
        } else {
          const int th = threadIdx.x & 127, j = th & 7, p = th >> 3;  // unit of the tile, token
          float* st = mine + 128 * kq;                               // [16 rows][8 tokens]
          *reinterpret_cast<float2*>(st + 8 * g + 2 * t) = make_float2(acc[0], acc[1]);
          *reinterpret_cast<float2*>(st + 8 * (g + 8) + 2 * t) = make_float2(acc[2], acc[3]);
          quad_sync(quad);
          if (p < s.count) {
            const float* gp = mine + 8 * j + p;
            const float rr = s.rr[p];
            const float gate = ((gp[0] + gp[128]) + (gp[256] + gp[384])) * rr, up = ((gp[64] + gp[192]) + (gp[320] + gp[448])) * rr;
            __stcg(act + (size_t)s.row[p] * I + j, silu_f(gate) * up);
          }
          quad_sync(quad);
        }
      }
    }
    __syncthreads();  // the planes are free, and what the stage wrote may be counted
  }
  cp_wait<0>();

  // ---------------- combine: once every block has written its results, each adds up its share of the outputs, in rank order
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(done + BLOCKS, 1u);
    await(BLOCKS, G);
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

static size_t workspace_bytes(int n, int topk) { return sizeof(Head) + (size_t)n * ((topk + 1) * (I + H) * sizeof(float) + TOKEN_BYTES); }

static cudaError_t configure_all() {
  const cudaError_t e = cudaFuncSetAttribute(k_moe_few, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
  return e != cudaSuccess ? e : drb_carveout(k_moe_few);
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
  p.digits = reinterpret_cast<unsigned char*>(p.part + (size_t)n * (topk + 1) * few::H);
  p.n = n, p.e = e, p.topk = topk, p.eps = eps, p.poll_limit = stack::POLL_LIMIT;
  const auto recip = [](int d) { return ((1ull << few::RECIP_BITS) + d - 1) / d; };
  p.by_grid = recip(dev.sms);
  for (int halves = 1; halves <= 2; ++halves) {
    const int rest = dev.sms - halves * few::SHARED_BLOCKS;
    p.per[halves - 1] = rest / ((n + 3) / 4);
    p.by_rest[halves - 1] = recip(rest), p.by_per[halves - 1] = recip(p.per[halves - 1]);
  }
  void* args[] = {&p};
  const cudaError_t err = cudaLaunchCooperativeKernel((const void*)few::k_moe_few, dim3(dev.sms), dim3(few::THREADS), args, few::SMEM_BYTES, st);
  return err == cudaSuccess ? 0 : (int)err;
}
