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
//   combine    every tile's weighted result goes to memory; the warp that finishes the last expert of 16 output columns adds
//              them up, in rank order whatever the order of arrival
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
  unsigned act_done[2][MAX_HIT + 8];   // [call parity][expert hit, MAX_HIT = shared]: gate/up tiles finished
  unsigned tile_done[2][DN_TILES];     // [call parity][16 output columns]: experts finished
  unsigned long long logits[MAX_TOK * LOGIT_STRIDE];
};
static_assert(sizeof(Head) % 256 == 0 && offsetof(Head, logits) % 16 == 0, "aligned sections");

constexpr int SUB = 2048;                // a step of a warp: 16 rows x 128 bytes
constexpr int SLOT = SUB + 256;          // and 16 bytes of scales a row
constexpr int PITCH = H + 64, DPITCH = I + 64;   // bytes between digit planes: neighbouring planes on different banks
constexpr int MP = H / 64 + 1, DMP = I / 64 + 1;  // (scale, sum) pairs between tokens

template <int TOK>
struct Shape {
  static constexpr int DEPTH = TOK > 8 ? 3 : 4;
  static constexpr int PLANES = 3 * TOK * PITCH, META = TOK * MP * 8, RING = CW * DEPTH * SLOT, RED = CW * 16 * 8 * 4;
  static constexpr int CTL = 4096;
  static constexpr size_t BYTES = CTL + PLANES + META + RING + RED;
  static_assert(BYTES <= 232448 && 2 * 3 * TOK * DPITCH <= PLANES && 2 * TOK * DMP * 8 <= META, "shared memory");
};

struct Seg {  // the tokens of one expert in this block's run
  int count, slot;       // slot: index of its counter
  unsigned char pos[16];  // digit planes
  short row[16];         // row of the activations and of the weighted results
  float wt[16];
};

struct Ctl {
  Seg seg[2], shared;
  int idx[MAX_TOK][MAX_K];
  float wts[MAX_TOK][MAX_K];
  float sgate[MAX_TOK], rr[MAX_TOK];
  unsigned mask[MAX_E];            // tokens that chose the expert
  unsigned char hit[MAX_HIT];
  int wsum[8];
  int nhit, abort;
  unsigned tag, live;
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

// Sixteen consecutive inputs of a lane (four lanes share 64) as the digits of round(v / delta), delta = max|v| / 8,355,000 (127 (1 +
// 256 + 65536) is the largest number that three signed bytes hold). n + 0x808080 has the digits plus 128 as its bytes. Words of a
// digit: inputs {0,2,4,6}, {1,3,5,7}, {8,10,12,14}, {9,11,13,15}, the order in which the nibbles of eight bytes come.
// A NaN or an infinity among the 64 makes delta NaN or infinite, and with it every sum that the 64 enter.
DRB_DEV float digits16(const float (&v)[16], unsigned char* plane, int pitch) {
  unsigned mb = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) mb = max(mb, __float_as_uint(v[i]) & 0x7fffffffu);
  mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
  mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
  const float m = __uint_as_float(mb);
  const bool finite = mb < 0x7f800000u;
  // kept away from the subnormals, whose reciprocal is infinite
  const float delta = finite ? fmaxf(m * (1.f / 8355000.f), 1.1754944e-38f) : m;
  const float inv = finite ? 1.f / delta : 0.f;
  uint32_t n[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) n[i] = (uint32_t)((finite ? __float2int_rn(v[i] * inv) : 0) + 0x808080) ^ 0x808080u;
#pragma unroll
  for (int l = 0; l < 3; ++l) {
    uint32_t w[4];
    const uint32_t sel = l == 0 ? 0x0040u : l == 1 ? 0x0051u : 0x0062u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int b = 8 * (q >> 1) + (q & 1);
      w[q] = prmt(prmt(n[b], n[b + 2], sel), prmt(n[b + 4], n[b + 6], sel), 0x5410u);
    }
    *reinterpret_cast<uint4*>(plane + l * pitch) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return delta;
}

// The weights of a run of tiles on their way: a warp's cursor and its ring.
struct Loader {
  const unsigned char *p;   // this lane's first row and piece
  const unsigned char *sp;  // this lane's row of scales (lanes 0..15)
  int stride, gap;          // bytes between rows, and from row r to row r + 8
  int sub, nsub, task, ntask;
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

constexpr float MAGIC = 12582912.f;  // 1.5 * 2^23: an integer below 2^22 added to its bits is added to its value
constexpr int MAGIC_BITS = 0x4B400000;

// One warp's share of a tile: 16 rows against the tokens of a segment. TG = 0: one or two tokens, four columns each (three digits);
// TG = 1, 2: up to 8 or 16 tokens, a column tile per digit and eight tokens.
template <int TG>
struct Acc {
  float v[TG ? TG * 4 : 2];
};

template <int TG>
struct Cols {
  const unsigned char* b[TG ? TG : 1];  // this lane's column: its token's digit planes
  const float2* m[TG ? 2 * TG : 1];     // (delta, sum) of the columns whose sums this lane holds
  float ka, kb;                         // TG = 0: weights of this lane's two columns
  bool first;
};

template <int TG>
DRB_DEV void cols_set(Cols<TG>& c, const Seg& s, const unsigned char* planes, int pitch, const float2* meta, int mp, int lane) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (TG == 0) {
    const int mine = s.pos[min(g >> 2, s.count - 1)];
    c.b[0] = planes + (3 * mine + min(g & 3, 2)) * pitch + 16 * t;
    c.m[0] = meta + s.pos[min(t >> 1, s.count - 1)] * mp;
    c.ka = t & 1 ? 65536.f : 1.f;
    c.kb = t & 1 ? 0.f : 256.f;
    c.first = (t & 1) == 0;
  } else {
#pragma unroll
    for (int i = 0; i < TG; ++i) {
      c.b[i] = planes + 3 * s.pos[min(8 * i + g, s.count - 1)] * pitch + 16 * t;
      c.m[2 * i] = meta + s.pos[min(8 * i + 2 * t, s.count - 1)] * mp;
      c.m[2 * i + 1] = meta + s.pos[min(8 * i + 2 * t + 1, s.count - 1)] * mp;
    }
  }
}

// 64 inputs: A in the operand's registers, group kg of the planes; s0, m0: scale and min of row g, s1, m1 of row g + 8.
template <int TG, bool MIN>
DRB_DEV void group64(Acc<TG>& acc, const Cols<TG>& c, int pitch, int kg, const uint32_t (&a)[8], float s0, float m0, float s1, float m1) {
  if constexpr (TG == 0) {
    const uint4 b = *reinterpret_cast<const uint4*>(c.b[0] + 64 * kg);
    int d[4] = {MAGIC_BITS, MAGIC_BITS, MAGIC_BITS, MAGIC_BITS};
    gemv::q8::mma_s8(d, a[0], a[1], a[2], a[3], b.x, b.y);
    gemv::q8::mma_s8(d, a[4], a[5], a[6], a[7], b.z, b.w);
    const float2 m = c.m[0][kg];
    const float f0 = __int_as_float(d[0]) - MAGIC, f1 = __int_as_float(d[1]) - MAGIC;
    const float h0 = __int_as_float(d[2]) - MAGIC, h1 = __int_as_float(d[3]) - MAGIC;
    acc.v[0] = fmaf(s0 * m.x, fmaf(f1, c.kb, f0 * c.ka), acc.v[0]);
    acc.v[1] = fmaf(s1 * m.x, fmaf(h1, c.kb, h0 * c.ka), acc.v[1]);
    if (MIN) {
      const float sum = c.first ? m.y : 0.f;
      acc.v[0] = fmaf(m0, sum, acc.v[0]);
      acc.v[1] = fmaf(m1, sum, acc.v[1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < TG; ++i) {
      float f[4];
#pragma unroll
      for (int l = 2; l >= 0; --l) {
        const uint4 b = *reinterpret_cast<const uint4*>(c.b[i] + l * pitch + 64 * kg);
        int d[4] = {MAGIC_BITS, MAGIC_BITS, MAGIC_BITS, MAGIC_BITS};
        gemv::q8::mma_s8(d, a[0], a[1], a[2], a[3], b.x, b.y);
        gemv::q8::mma_s8(d, a[4], a[5], a[6], a[7], b.z, b.w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = __int_as_float(d[j]) - MAGIC;
          f[j] = l == 2 ? v : fmaf(f[j], 256.f, v);
        }
      }
      const float2 c0 = c.m[2 * i][kg], c1 = c.m[2 * i + 1][kg];
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

template <int TOK>
__global__ void __launch_bounds__(THREADS, 1) k_moe_few(Params P) {
  using S = Shape<TOK>;
  constexpr int DEPTH = S::DEPTH;
  extern __shared__ __align__(128) unsigned char dyn[];
  Ctl& ctl = *reinterpret_cast<Ctl*>(dyn);
  unsigned char* planes = dyn + S::CTL;
  float2* meta = reinterpret_cast<float2*>(planes + S::PLANES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp >> 2, kq = warp & 3;
  unsigned char* ring = planes + S::PLANES + S::META + warp * DEPTH * SLOT;
  float* red = reinterpret_cast<float*>(planes + S::PLANES + S::META + S::RING);
  const int n = P.n, E = P.e, topk = P.topk, E1 = E + 1;
  const int G = (int)gridDim.x, b = (int)blockIdx.x;
  volatile int* abort_flag = &ctl.abort;
  const int shared_block = b - (G - SHARED_BLOCKS);  // >= 0: one of them

  // ---------------- this call's number; the counters of the next call
  if (threadIdx.x == 0) {
    const unsigned ep = ld_acquire(&P.ws->epoch);
    ctl.tag = ep;
    ctl.abort = 0;
    unsigned m = 0u;
    for (int r = 0; r < n; ++r) m |= (!P.live || P.live[r]) ? 1u << r : 0u;
    ctl.live = m;
    if (atom_add_acq_rel(&P.ws->seen, 1u) == (unsigned)G - 1u) {  // every block has read it
      P.ws->seen = 0u;
      P.ws->epoch = ep + 1u;
    }
  }
  for (int i = threadIdx.x; i < MAX_E; i += THREADS) ctl.mask[i] = 0u;

  // ---------------- the weights' stream
  Loader ld;
  ld.task = ld.ntask = 0;
  int nslot = 0, slot = 0;  // ring positions: next to fill, next to use
  int ntile = 0, ndtile = 0, nshared = 0;  // this quad's gate/up tiles; this warp's down tiles; the block's shared down tiles, which come first
  int gu_first = 0, dn_shared0 = 0, dn_first = 0;
  // Task i of the warp: gate/up tiles, then down tiles. kind 0: gate/up, 1: shared down, 2: down
  auto point = [&](const void* w, const void* s, bool int8, int row_bytes, int row0, int gap_rows, int off, int srow_bytes, int soff, int nsub) {
    ld.int8 = int8;
    ld.stride = 4 * row_bytes, ld.gap = gap_rows * row_bytes;
    ld.p = static_cast<const unsigned char*>(w) + (size_t)(row0 + (lane >> 3)) * row_bytes + off + 16 * (lane & 7);
    const int r = lane & 15;
    ld.sp = static_cast<const unsigned char*>(s) + (size_t)(row0 + (r < 8 ? r : r - 8 + gap_rows)) * srow_bytes + soff;
    ld.sub = 0, ld.nsub = nsub;
  };
  auto aim_shared = [&](int tile) {  // shared gate/up
    point(P.w.sgu_q, P.w.sgu_s, true, H, 8 * tile, I, kq * 512, H / 128 * 2, kq * 8, 4);
  };
  auto aim = [&](int task) {
    if (task < ntile) {
      const int u = gu_first + quad + 4 * task, e = ctl.hit[u / GU_TILES];
      point(P.w.gu_q, P.w.gu_sm, false, H / 2, e * 2 * I + 8 * (u % GU_TILES), I, kq * 256, H / 64 * 4, kq * 32, 2);
    } else {
      const int i = warp + CW * (task - ntile);
      if (i < nshared) {
        point(P.w.sd_q, P.w.sd_s, true, I, 16 * (dn_shared0 + i), 8, 0, I / 128 * 2, 0, 4);
      } else {
        const int u = dn_first + i - nshared, e = ctl.hit[u / DN_TILES];
        point(P.w.d_q, P.w.d_sm, false, I / 2, e * H + 16 * (u % DN_TILES), 8, 0, I / 64 * 4, 0, 2);
      }
    }
  };
  // Requests the next step. Piece c (16 bytes) of row r lies where reads of eight rows at once meet no bank twice: int4 rows are
  // read 32 bytes (four lanes) at a time, int8 rows 64.
  auto issue = [&](bool in_run) {
    if (ld.task < ld.ntask) {
      const uint32_t dst = smem_u32(ring + nslot * SLOT);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 3) + 4 * i, c = lane & 7;
        const int at = ld.int8 ? c ^ ((r & 1) << 2) : c ^ ((r & 3) << 1);
        cp16(dst + r * 128 + 16 * at, ld.p + (i & 1) * ld.stride + (i >> 1) * ld.gap);
      }
      if (lane < 16) {
        if (ld.int8) cp4(dst + SUB + 16 * lane, ld.sp + 4 * (ld.sub >> 1));
        else cp16(dst + SUB + 16 * lane, ld.sp + 16 * ld.sub);
      }
      ld.p += 128;
      if (++ld.sub == ld.nsub && ++ld.task < ld.ntask && in_run) aim(ld.task);
    }
    cp_commit();
    if (++nslot == DEPTH) nslot = 0;
  };
  auto next_slot = [&]() -> const unsigned char* {
    cp_wait<DEPTH - 1>();
    __syncwarp();
    return ring + slot * SLOT;
  };
  auto used = [&](bool in_run) {
    __syncwarp();
    issue(in_run);
    if (++slot == DEPTH) slot = 0;
  };
  if (shared_block >= 0) {
    ld.ntask = 1;
    aim_shared(4 * shared_block + quad);
#pragma unroll 1
    for (int i = 0; i < DEPTH; ++i) issue(false);
  }

  // ---------------- logits: token group tg (four tokens), router rows [r0, r1); thread t holds inputs 4 t .. 4 t + 3
  const int tgs = (n + 3) / 4, per = G / tgs, tg = b / per;
  __syncthreads();
  const unsigned live = ctl.live, ep = ctl.tag, tag = 2u * ep + 1u;
  if (b == 0) {
    unsigned* nxt_a = P.ws->act_done[(ep + 1) & 1];
    unsigned* nxt_t = P.ws->tile_done[(ep + 1) & 1];
    for (int i = threadIdx.x; i < MAX_HIT + 8; i += THREADS) nxt_a[i] = 0u;
    for (int i = threadIdx.x; i < DN_TILES; i += THREADS) nxt_t[i] = 0u;
  }
  if (live == 0u) {
    cp_wait<0>();
    return;
  }
  unsigned* act_done = P.ws->act_done[ep & 1];
  unsigned* tile_done = P.ws->tile_done[ep & 1];
  const float4 nw4 = __ldcg(reinterpret_cast<const float4*>(P.w.post_norm) + threadIdx.x);
  if (tg < tgs) {
    constexpr int RP = 7;  // rows a pass
    const int s = b % per, r0 = E1 * s / per, r1 = E1 * (s + 1) / per;
    float4 xs[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int r = 4 * tg + m;
      xs[m] = (live >> r) & 1u ? __ldcg(reinterpret_cast<const float4*>(P.x + (size_t)r * H) + threadIdx.x) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int rb = r0; rb < r1 || rb == r0; rb += RP) {
      uint2 w[RP];
#pragma unroll
      for (int i = 0; i < RP; ++i)
        w[i] = rb + i < r1 ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(P.w.router) + (size_t)(rb + i) * H) + threadIdx.x) : make_uint2(0u, 0u);
      float v[32];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const float4 q = xs[m];
        v[28 + m] = (q.x * q.x + q.y * q.y) + (q.z * q.z + q.w * q.w);
        const float4 h = make_float4(q.x * nw4.x, q.y * nw4.y, q.z * nw4.z, q.w * nw4.w);
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const float a0 = __uint_as_float(w[i].x << 16), a1 = __uint_as_float(w[i].x & 0xffff0000u);
          const float a2 = __uint_as_float(w[i].y << 16), a3 = __uint_as_float(w[i].y & 0xffff0000u);
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
          if (row == E1 - 1 && (E1 & 1)) stack::ll_store(dst + 1, 0u, tag);  // words are polled in pairs
        }
        if (lane < 4) ctl.rr[4 * tg + lane] = rr;
      }
      __syncthreads();
    }
  }

  // ---------------- digit planes of the tokens in `want`
  auto convert = [&](int tok, int i, float (&keep)[2], float& ss) {  // inputs 512 i + 16 lane .. + 15
    const float4* xp = reinterpret_cast<const float4*>(P.x + (size_t)tok * H) + 128 * i + 4 * lane;
    const float4* np = reinterpret_cast<const float4*>(P.w.post_norm) + 128 * i + 4 * lane;
    float v[16], sum = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 a = __ldcg(xp + q), c = __ldcg(np + q);
      ss += (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w);
      v[4 * q] = a.x * c.x, v[4 * q + 1] = a.y * c.y, v[4 * q + 2] = a.z * c.z, v[4 * q + 3] = a.w * c.w;
      sum += (v[4 * q] + v[4 * q + 1]) + (v[4 * q + 2] + v[4 * q + 3]);
    }
    keep[0] = digits16(v, planes + 3 * tok * PITCH + 512 * i + 16 * lane, PITCH);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    keep[1] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
  };
  auto convert_tokens = [&](unsigned want) {
    if (tgs == 1) {  // 1 / rms is known in every block: a warp for each quarter of a token
      const int tok = warp >> 2;
      if ((want >> tok) & 1u) {
        float keep[2], ss = 0.f;
        convert(tok, kq, keep, ss);
        if ((lane & 3) == 0) meta[tok * MP + 8 * kq + (lane >> 2)] = make_float2(keep[0] * ctl.rr[tok], keep[1] * ctl.rr[tok]);
      }
    } else if ((want >> warp) & 1u) {
      float keep[4][2], ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) convert(warp, i, keep[i], ss);
      const float rr = rsqrtf(warp_sum(ss) / (float)H + P.eps);
      if ((lane & 3) == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) meta[warp * MP + 8 * i + (lane >> 2)] = make_float2(keep[i][0] * rr, keep[i][1] * rr);
    }
  };
  // The tokens of expert `e` (-1: all live ones, the shared expert), by one warp
  auto list = [&](Seg& s, int e, int sl, bool by_place, int base) {
    const unsigned m = e < 0 ? live : ctl.mask[e];
    if (lane < MAX_TOK && (m >> lane) & 1u) {
      const int p = __popc(m & ((1u << lane) - 1u));
      int k = 0;
      if (e >= 0)
        while (k + 1 < topk && ctl.idx[lane][k] != e) ++k;
      s.pos[p] = (unsigned char)(by_place ? base + p : lane);
      s.row[p] = (short)(e < 0 ? n * topk + lane : lane * topk + k);
      s.wt[p] = e < 0 ? sigmoid_f(ctl.sgate[lane]) : ctl.wts[lane][k];
    }
    if (lane == 0) s.count = __popc(m), s.slot = sl;
  };

  // A quad's gate/up tile: sums of the four quarters meet in shared memory; then the activations, and the expert's counter.
  auto gate_up = [&](auto tg_c, auto int8_c, const Seg& s, int tile, bool in_run) {
    constexpr int TG = decltype(tg_c)::value;
    constexpr bool INT8 = decltype(int8_c)::value;
    Cols<TG> c;
    cols_set<TG>(c, s, planes, PITCH, meta, MP, lane);
    Acc<TG> acc = {};
#pragma unroll 1
    for (int sub = 0; sub < (INT8 ? 4 : 2); ++sub) {
      step<TG, INT8>(acc, c, PITCH, 8 * kq + (INT8 ? 2 : 4) * sub, next_slot(), sub, lane);
      used(in_run);
    }
    const int g = lane >> 2, t = lane & 3;
    float* mine = red + warp * 128;  // [16 rows][8 tokens]
    const float* first = red + quad * 4 * 128;
    const int th = threadIdx.x & 127;
#pragma unroll
    for (int i = 0; i < (TG ? TG : 1); ++i) {
      if constexpr (TG == 0) {
        const float a0 = acc.v[0] + __shfl_xor_sync(0xffffffffu, acc.v[0], 1), a1 = acc.v[1] + __shfl_xor_sync(0xffffffffu, acc.v[1], 1);
        if ((t & 1) == 0) mine[8 * g + (t >> 1)] = a0, mine[8 * (g + 8) + (t >> 1)] = a1;
      } else {
        *reinterpret_cast<float2*>(mine + 8 * g + 2 * t) = make_float2(acc.v[4 * i], acc.v[4 * i + 1]);
        *reinterpret_cast<float2*>(mine + 8 * (g + 8) + 2 * t) = make_float2(acc.v[4 * i + 2], acc.v[4 * i + 3]);
      }
      quad_sync(quad);
      const int j = th & 7, p = th >> 3;  // unit of the tile, token
      if (p < 8 && 8 * i + p < s.count) {
        const float* gp = first + 8 * j + p;
        const float gate = (gp[0] + gp[128]) + (gp[256] + gp[384]), up = (gp[64] + gp[192]) + (gp[320] + gp[448]);
        __stcg(P.act + (size_t)s.row[8 * i + p] * I + 8 * tile + j, silu_f(gate) * up);
      }
      quad_sync(quad);
    }
    if (th == 0) {
      __threadfence();
      atomicAdd(act_done + s.slot, 1u);
    }
  };
  using std::integral_constant;
  auto gate_up_any = [&](auto int8_c, const Seg& s, int tile, bool in_run) {
    if (s.count <= 2) gate_up(integral_constant<int, 0>(), int8_c, s, tile, in_run);
    else if (TOK <= 8 || s.count <= 8) gate_up(integral_constant<int, 1>(), int8_c, s, tile, in_run);
    else gate_up(integral_constant<int, 2>(), int8_c, s, tile, in_run);
  };

  const bool early = tgs == 1 || shared_block >= 0;
  if (early) {
    convert_tokens(live);
    if (warp == 0) list(ctl.shared, -1, MAX_HIT, false, 0);
    __syncthreads();
  }
  if (shared_block >= 0) gate_up_any(integral_constant<bool, true>(), ctl.shared, 4 * shared_block + quad, false);

  // ---------------- routing: a warp a token; every block for itself
  if ((live >> warp) & 1u) {
    const unsigned long long* src = P.ws->logits + warp * LOGIT_STRIDE;
    const int pieces = (E1 + 1) / 2;
    float v[10];
    int id[10];
    unsigned need = 0u;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      id[2 * i] = 2 * (lane + 32 * i), id[2 * i + 1] = id[2 * i] + 1;
      v[2 * i] = v[2 * i + 1] = 0.f;
      if (lane + 32 * i < pieces) need |= 1u << i;
    }
    for (unsigned it = 0; !*abort_flag; ++it) {  // all requests of a round go out before any is looked at
      unsigned long long q[10];
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if ((need >> i) & 1u) stack::ll_load2(src + id[2 * i], q[2 * i], q[2 * i + 1]);
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (((need >> i) & 1u) && (uint32_t)(q[2 * i] >> 32) == tag && (uint32_t)(q[2 * i + 1] >> 32) == tag) {
          v[2 * i] = __uint_as_float((uint32_t)q[2 * i]), v[2 * i + 1] = __uint_as_float((uint32_t)q[2 * i + 1]);
          need &= ~(1u << i);
        }
      if (need == 0u || stack::poll_failed(it, P.poll_limit, abort_flag)) break;
    }
    __syncwarp();
    uint32_t key[10];  // larger logit = larger key, never 0; 0: no entry, or taken. A NaN counts as the lowest logit
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint32_t u = __float_as_uint(v[i]);
      if (id[i] == E) ctl.sgate[warp] = v[i];
      const uint32_t o = (u & 0x7fffffffu) > 0x7f800000u ? 1u : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
      key[i] = id[i] < E ? o : 0u;
    }
    float top = 0.f, sum = 0.f;
    for (int k = 0; k < topk; ++k) {
      uint32_t bk = 0u;
      int bi = MAX_E;
#pragma unroll
      for (int i = 0; i < 10; ++i)
        if (key[i] > bk) bk = key[i], bi = id[i];  // ids ascend within a lane
      const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
      const int who = (int)__reduce_min_sync(0xffffffffu, bk == best ? (unsigned)bi : (unsigned)MAX_E);
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < 10; ++i)
        if (id[i] == who && key[i] != 0u) mine = v[i], key[i] = 0u;
      const float val = __shfl_sync(0xffffffffu, mine, (who >> 1) & 31);
      if (k == 0) top = val;
      const float ex = expf(val - top);
      sum += ex;
      if (lane == 0) ctl.idx[warp][k] = who, ctl.wts[warp][k] = ex;
    }
    __syncwarp();
    if (lane < topk) {
      ctl.wts[warp][lane] = ctl.wts[warp][lane] / sum;
      atomicOr(&ctl.mask[ctl.idx[warp][lane]], 1u << warp);
    }
  }
  __syncthreads();
  // experts hit, in ascending order
  {
    const bool on = threadIdx.x < MAX_E && ctl.mask[threadIdx.x & (MAX_E - 1)] != 0u;
    const unsigned bal = __ballot_sync(0xffffffffu, on);
    if (warp < 8 && lane == 0) ctl.wsum[warp] = __popc(bal);
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int c = ctl.wsum[w];
      base += w < warp ? c : 0;
      all += c;
    }
    if (on) ctl.hit[base + __popc(bal & ((1u << lane) - 1u))] = (unsigned char)threadIdx.x;
    if (threadIdx.x == 0) ctl.nhit = all;
    __syncthreads();
  }
  const int nhit = ctl.nhit;
  // gate/up: tiles [gu_first, gu_end) of the list; down: units [u0, u1) of 4 KB, two for a tile of the shared expert, which come first
  gu_first = nhit * GU_TILES * b / G;
  const int gu_end = nhit * GU_TILES * (b + 1) / G;
  ntile = gu_end - gu_first > quad ? (gu_end - gu_first - quad + 3) / 4 : 0;
  const int units = (nhit + 2) * DN_TILES, u0 = units * b / G, u1 = units * (b + 1) / G;
  dn_shared0 = min((u0 + 1) / 2, DN_TILES);
  nshared = min((u1 + 1) / 2, DN_TILES) - dn_shared0;
  dn_first = max(u0 - 2 * DN_TILES, 0);
  const int dn_end = max(u1 - 2 * DN_TILES, 0), ndn = nshared + dn_end - dn_first;
  ndtile = ndn > warp ? (ndn - warp + CW - 1) / CW : 0;
  ld.task = 0, ld.ntask = ntile + ndtile;
  if (ld.ntask > 0) aim(0);
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) issue(true);

  const int h0 = gu_first / GU_TILES;
  if (gu_end > gu_first) {
    const int h1 = (gu_end - 1) / GU_TILES;
    if (warp == 0) list(ctl.seg[0], ctl.hit[h0], h0, false, 0);
    if (warp == 1) list(ctl.seg[1], ctl.hit[h1], h1, false, 0);
    if (!early) convert_tokens(ctl.mask[ctl.hit[h0]] | ctl.mask[ctl.hit[h1]]);
  }
  __syncthreads();
  for (int i = 0; i < ntile; ++i) {
    const int u = gu_first + quad + 4 * i;
    gate_up_any(integral_constant<bool, false>(), ctl.seg[u / GU_TILES - h0 ? 1 : 0], u % GU_TILES, true);
  }
  __syncthreads();  // the planes are free

  // ---------------- down: digit planes of the (at most two) experts' activations
  const int d0 = nshared > 0 ? -1 : dn_first / DN_TILES;                 // first segment, -1: the shared expert
  const int d1 = dn_end > dn_first ? (dn_end - 1) / DN_TILES : d0;       // last one
  if (warp < 2 && ndn > 0) {
    const int h = warp == 0 ? d0 : d1;
    Seg& s = ctl.seg[warp];
    list(s, h < 0 ? -1 : ctl.hit[h], h < 0 ? MAX_HIT : h, true, warp * TOK);
    if (lane == 0 && !*abort_flag)
      for (unsigned it = 0; ld_acquire(act_done + (h < 0 ? MAX_HIT : h)) < (unsigned)GU_TILES; ++it)
        if (stack::poll_failed(it, P.poll_limit, abort_flag)) break;
  }
  __syncthreads();
  if (ndn > 0) {
    const int c0 = ctl.seg[0].count, all = c0 + (d1 != d0 ? ctl.seg[1].count : 0);
    for (int i = warp; i < all; i += CW) {
      const Seg& s = ctl.seg[i >= c0];
      const int p = i >= c0 ? i - c0 : i, pos = s.pos[p];
      const float4* ap = reinterpret_cast<const float4*>(P.act + (size_t)s.row[p] * I) + 4 * lane;
      float v[16], sum = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 a = __ldcg(ap + q);
        v[4 * q] = a.x, v[4 * q + 1] = a.y, v[4 * q + 2] = a.z, v[4 * q + 3] = a.w;
        sum += (a.x + a.y) + (a.z + a.w);
      }
      const float delta = digits16(v, planes + 3 * pos * DPITCH + 16 * lane, DPITCH);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if ((lane & 3) == 0) meta[pos * DMP + (lane >> 2)] = make_float2(delta, sum);
    }
  }
  __syncthreads();

  auto down = [&](auto tg_c, auto int8_c, const Seg& s, int tile) {
    constexpr int TG = decltype(tg_c)::value;
    constexpr bool INT8 = decltype(int8_c)::value;
    Cols<TG> c;
    cols_set<TG>(c, s, planes, DPITCH, meta, DMP, lane);
    Acc<TG> acc = {};
#pragma unroll 1
    for (int sub = 0; sub < (INT8 ? 4 : 2); ++sub) {
      step<TG, INT8>(acc, c, DPITCH, (INT8 ? 2 : 4) * sub, next_slot(), sub, lane);
      used(true);
    }
    const int g = lane >> 2, t = lane & 3;
    float* out = P.part + 16 * tile + g;
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
    // the last expert of these 16 columns to arrive adds them up
    __syncwarp();
    unsigned before = 0u;
    if (lane == 0) {
      __threadfence();
      before = atomicAdd(tile_done + tile, 1u);
      __threadfence();
    }
    if (__shfl_sync(0xffffffffu, before, 0) != (unsigned)nhit) return;  // nhit + 1 with the shared expert
    for (int i = lane; i < 16 * n; i += 32) {
      const int r = i >> 4, col = 16 * tile + (i & 15);
      if (!((live >> r) & 1u)) continue;
      float v[MAX_K];
#pragma unroll
      for (int k = 0; k < MAX_K; ++k) v[k] = k < topk ? __ldcg(P.part + (size_t)(r * topk + k) * H + col) : 0.f;
      float s = __ldcg(P.x + (size_t)r * H + col) + __ldcg(P.part + (size_t)(n * topk + r) * H + col);
      float rest = 0.f;
#pragma unroll
      for (int k = 0; k < MAX_K; ++k) rest += v[k];
      P.y[(size_t)r * H + col] = s + rest;
    }
  };
  auto down_any = [&](auto int8_c, const Seg& s, int tile) {
    if (s.count <= 2) down(integral_constant<int, 0>(), int8_c, s, tile);
    else if (TOK <= 8 || s.count <= 8) down(integral_constant<int, 1>(), int8_c, s, tile);
    else down(integral_constant<int, 2>(), int8_c, s, tile);
  };
  for (int j = 0; j < ndtile; ++j) {
    const int i = warp + CW * j;
    if (i < nshared) {
      down_any(integral_constant<bool, true>(), ctl.seg[0], dn_shared0 + i);
    } else {
      const int u = dn_first + i - nshared;
      down_any(integral_constant<bool, false>(), ctl.seg[u / DN_TILES == d0 ? 0 : 1], u % DN_TILES);
    }
  }
  cp_wait<0>();
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
