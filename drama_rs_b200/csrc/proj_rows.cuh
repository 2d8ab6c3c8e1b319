// The projection of drb_proj_q8_lora for many rows: tcgen05 with the int8 codes handed over in tensor memory.
//
//   y [rows, n] = x W^T (+ res) + B v      D[128, nc] = W_tile[128, K] . x[nc, K]^T,  nc = 16 .. 80 rows of x
//
// A code becomes a 16-bit number exactly, so the operand carries no scale: the multiplications of each 128 inputs have an
// accumulator of their own (two, in turns), and the epilogue warps sum scale * accumulator in fp32 as they complete. An adapter of the
// tile's rows is one more stretch of inputs: its rows of B as the A operand, v (zero in other adapters' rows) as B operand in
// three bf16 terms, 24 bits; the accumulator joins with a factor of one. 128 inputs of a tile take 0.49 us with nc = 16 and 0.55 with 80, some 1000 cycles. The conversion's
// instructions, two a weight (bf16; fp16 one and a quarter) beside its loads and stores, fill about 350 of them, the multiplications of nc = 80 160; no unit is
// near its limit (issue 0.44, integer pipe 0.37), and what the rest is has not been found. Queued, 4096 x 2048, 300 rows: 12.6 us, with 3 adapters of rank 64 17.8;
// 8192 x 2048, 2048 rows: 133 us (0.52 PFLOP/s), with three adapters of rank 16 162 (one tile a block: 168).
//
// Roles, one block of 16 warps per multiprocessor, meeting on mbarriers, every wait bounded: 8 convert warps (two sets that take turns; a
// thread the 128 codes of one weight row), 4 epilogue warps (a thread one weight row), one warp that issues the multiplications, one that issues the copies (tiled
// TMA, 128-byte swizzle), one that looks at the rows' adapters. A block keeps its rows of x (blockIdx.y) and walks weight tiles.
#pragma once

#include "moe_prefill_tc.cuh"
#include "proj_lora.cuh"

namespace pr {

using namespace tc;

constexpr int CONV = 8, SET = 4, SETS = CONV / SET, EPI = 4, MMA_WARP = CONV + EPI, LOAD_WARP = MMA_WARP + 1, WHO_WARP = LOAD_WARP + 1, THREADS = 512;
// Registers a thread: what the launch gets, and after the roles have parted (setmaxnreg works on groups of four warps; the sixteenth only gives
// its own). The shares are no more than the launch's.
constexpr int LAUNCH_REGS = 96, CONV_REGS = 88, EPI_REGS = 144, REST_REGS = 64;
static_assert(8 * CONV_REGS + 4 * EPI_REGS + 4 * REST_REGS <= THREADS / 32 * LAUNCH_REGS && CONV == 8 && EPI == 4, "registers");
constexpr int NRAW = 4, NA = 3;            // raw stages of 16 KB; stages of A (64 columns of tensor memory) with a tile of x
constexpr int MAX_C = 80;                  // rows of x a tile: their sums are an epilogue thread's registers
constexpr int RAW_BYTES = 128 * 128;
constexpr int TMEM_COLS = 512, A_COL0 = 2 * MAX_C;
static_assert(MAX_C == 80 && A_COL0 + NA * 64 <= TMEM_COLS, "tensor memory");

struct Ctl {
  uint64_t rawfull[NRAW], rawempty[NRAW];  // a raw stage has landed / has been read (one arrival per convert warp of a set)
  uint64_t full[NA], done[NA];             // a stage is complete (convert warps, and the tile of x) / its multiplications have completed
  uint64_t accfull[2], accfree[2];         // an accumulator is complete / has been drained (one arrival per epilogue warp)
  uint32_t tmem;
  int ndiff;
  __align__(16) int who[96];            // adapters of the tile's rows, -1: none
  int diff[MAX_C];                         // the different ones among them
};
constexpr int CTL_BYTES = 1024;
static_assert(sizeof(Ctl) <= CTL_BYTES, "control block");

// 1024 of slack for the alignment; a stage of x holds two boxes of 64 inputs, or three terms of v
static size_t smem_bytes(int nc) { return 1024 + CTL_BYTES + NRAW * RAW_BYTES + (size_t)NA * 3 * nc * 128; }

struct Maps {
  CUtensorMap w, x;
};

// After a wait that ran out: the copies and multiplications that this block has asked for end within the millisecond.
DRB_DEV void linger() {
  for (int i = 0; i < 64; ++i) __nanosleep(16384);
}

template <bool F16>
__global__ void __launch_bounds__(640, 1) k_proj_rows(const __grid_constant__ Maps maps, pl::Args p, int nc, int each, int tiles) {
  extern __shared__ unsigned char dyn_raw[];
  unsigned char* dyn = dyn_raw + (-smem_u32(dyn_raw) & 1023u);
  Ctl& ctl = *reinterpret_cast<Ctl*>(dyn);
  unsigned char* raw = dyn + CTL_BYTES;
  unsigned char* xst = raw + NRAW * RAW_BYTES;
  const int box = nc * 128, xstage = 3 * box;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.k >> 7, row0 = (int)blockIdx.y * each, cols = min(each, p.rows - row0);
  unsigned spent = 0;  // a wait of this thread ran out: none spins again
  const int first = (int)blockIdx.x, step = (int)gridDim.x, mine = first < tiles ? (tiles - first + step - 1) / step : 0;

  // ---------------- loader: weights are constants, so the first raw stages are requested at once
  int wi = 0, wtile = first, wg = 0;  // the next raw stage to request
  auto load_w = [&]() {
    const int r = wi % NRAW, use = wi / NRAW;
    if (use > 0) mbar_wait_ring<DRB_ERR_EMPTY_WAIT>(smem_u32(&ctl.rawempty[r]), (use - 1) & 1, spent);
    mbar_expect_tx(&ctl.rawfull[r], RAW_BYTES);
    tma_load_2d(raw + r * RAW_BYTES, &maps.w, wg * 128, wtile * 128, &ctl.rawfull[r]);
    ++wi;
    if (++wg == groups) wg = 0, wtile += step;
  };
  const int nw = mine * groups;
  if (warp == LOAD_WARP) {
    if (elect_one()) {
      for (int s = 0; s < NRAW; ++s) mbar_init(&ctl.rawfull[s], 1), mbar_init(&ctl.rawempty[s], SET);
      for (int s = 0; s < NA; ++s) mbar_init(&ctl.full[s], SET + 1), mbar_init(&ctl.done[s], 1);
      for (int s = 0; s < 2; ++s) mbar_init(&ctl.accfull[s], 1), mbar_init(&ctl.accfree[s], EPI);
      mbar_fence_init();
      while (wi < NRAW && wi < nw) load_w();
    }
    __syncwarp();
  }
  if (warp == MMA_WARP) tmem_alloc(&ctl.tmem, TMEM_COLS);
  pdl_launch_dependents();
  // The tile's adapters, a lane three of them, and the different ones among them. With adapters x and adapter_of are older than the launch before
  // (see proj_lora.cuh).
  if (warp == WHO_WARP && p.rank > 0) {
    int a[3], n = 0;
    bool is_first[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) a[i] = 32 * i + lane < cols ? pl::adapter(p, row0 + 32 * i + lane) : -1;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      ctl.who[32 * i + lane] = a[i];
      const unsigned same = __match_any_sync(0xffffffffu, a[i]);
      is_first[i] = a[i] >= 0 && __ffs(same) - 1 == lane;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const unsigned firsts = __ballot_sync(0xffffffffu, is_first[i]);
      if (is_first[i]) ctl.diff[n + __popc(firsts & ((1u << lane) - 1u))] = a[i];
      n += __popc(firsts);
      for (unsigned m = firsts; m; m &= m - 1u) {
        const int ad = __shfl_sync(0xffffffffu, a[i], __ffs(m) - 1);
#pragma unroll
        for (int k = i + 1; k < 3; ++k) is_first[k] = is_first[k] && a[k] != ad;
      }
    }
    if (lane == 0) ctl.ndiff = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  const int ndiff = p.rank > 0 ? ctl.ndiff : 0;
  const int seq = groups + ndiff, total = mine * seq;  // stretches of inputs: a tile's 128s, then its adapters

  if (warp < CONV) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONV_REGS));
  else if (warp < MMA_WARP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPI_REGS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REST_REGS));

  if (warp < CONV) {
    // ---------------- convert: two sets of four warps take turns at the stretches; a thread has one row of the tile
    const int q = warp & 3, row = 32 * q + lane;
    const uint32_t ta = tmem + ((uint32_t)(32 * q) << 16) + A_COL0;
    bool awaited = false;
    for (int c = warp >> 2, t = c / seq, g = c % seq; c < total; c += SETS) {
      const int s = c % NA, use = c / NA;
      uint32_t o[32];
      if (g < groups) {
        const int cw = t * groups + g, r = cw % NRAW;
        mbar_wait_ring<DRB_ERR_FULL_WAIT>(smem_u32(&ctl.rawfull[r]), (cw / NRAW) & 1, spent);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(raw + r * RAW_BYTES + swz_off(row, 4 * half + j));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pl::widen_codes<F16>(v[j].x, o[8 * j], o[8 * j + 1]);
            pl::widen_codes<F16>(v[j].y, o[8 * j + 2], o[8 * j + 3]);
            pl::widen_codes<F16>(v[j].z, o[8 * j + 4], o[8 * j + 5]);
            pl::widen_codes<F16>(v[j].w, o[8 * j + 6], o[8 * j + 7]);
          }
          if (half == 0) {
            if (use > 0) mbar_wait_ring<DRB_ERR_TMEM>(smem_u32(&ctl.done[s]), (use - 1) & 1, spent);
            tc_fence_after();
          }
          tmem_st32(ta + 64 * s + 32 * half, o);
        }
        // The stage goes back behind the stores that use its last codes: an arrival between the loads and their use let the stage's next codes in ahead of
        // loads that stood in the queue behind the other set's of an adapter's B (32 lines each; half of all calls of 280,000 x 8192 with adapters)
        reads_before_copies();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.rawempty[r]);
      } else {
        // an adapter: 64 ranks (zeros behind the last) of B's rows, and v
        const int ad = ctl.diff[g - groups], wr = (first + t * step) * 128 + row;
        const uint4* bp = reinterpret_cast<const uint4*>(p.b + ((size_t)ad * p.n + min(wr, p.n - 1)) * p.rank);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 b = 8 * j < p.rank ? __ldcg(bp + j) : make_uint4(0u, 0u, 0u, 0u);
          o[4 * j] = b.x, o[4 * j + 1] = b.y, o[4 * j + 2] = b.z, o[4 * j + 3] = b.w;
        }
        if (!awaited) pdl_wait(), awaited = true;
        // four ranks of a row a thread, five rows at once: thread i takes ranks 4 (i % 16) .. of rows i / 16, i / 16 + 8, ...
        const int k4 = threadIdx.x & 15;
        float4 f[5];
        auto load_v = [&](int r0) {
#pragma unroll
          for (int i = 0; i < 5; ++i) {
            const int r = r0 + 8 * i;
            f[i] = r < nc && ctl.who[r] == ad && 4 * k4 < p.rank ? __ldcg(reinterpret_cast<const float4*>(p.v + (size_t)(row0 + r) * p.rank) + k4)
                                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        };
        int r0 = (threadIdx.x & (SET * 32 - 1)) >> 4;
        load_v(r0);
        if (use > 0) mbar_wait_ring<DRB_ERR_TMEM>(smem_u32(&ctl.done[s]), (use - 1) & 1, spent);
        tc_fence_after();
        tmem_st32(ta + 64 * s, o);
        unsigned char* xs = xst + s * xstage;
        for (;;) {
#pragma unroll
          for (int i = 0; i < 5; ++i) {
            const int r = r0 + 8 * i;
            if (r >= nc) break;
            uint32_t b0[3], b1[3];
            pl::split3(f[i], b0, b1);
#pragma unroll
            for (int l = 0; l < 3; ++l) *reinterpret_cast<uint2*>(xs + l * box + swz_off(r, k4 >> 1) + 8 * (k4 & 1)) = make_uint2(b0[l], b1[l]);
          }
          if ((r0 += 40) >= nc) break;
          load_v(r0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the multiplications read v through the asynchronous proxy
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.full[s]);
      for (g += SETS; g >= seq; g -= seq) ++t;
    }
    if (!awaited) pdl_wait();  // this launch never ends before the one that it follows
  } else if (warp < MMA_WARP) {
    // ---------------- epilogue: a thread one weight row
    if (p.rank == 0) pdl_wait();  // res and y
    const int q = warp & 3, row = 32 * q + lane;
    const uint32_t td = tmem + ((uint32_t)(32 * q) << 16);
    float acc[MAX_C];
    int wr = first * 128 + row;
    auto scale = [&](int g) { return __ldg(p.s + (size_t)min(wr, p.n - 1) * groups + min(g, groups - 1)); };
    __half nxt = mine > 0 ? scale(0) : __half();
    for (int c = 0, g = 0; c < total; ++c) {
      const __half h = nxt;
      const int o = wr;
      if (g == 0)
#pragma unroll
        for (int j = 0; j < MAX_C; ++j) acc[j] = 0.f;
      if (g + 1 == seq) wr += step * 128;  // the next one's scale is on the way meanwhile
      nxt = c + 1 < total ? scale(g + 1 == seq ? 0 : g + 1) : h;
      mbar_wait_ring<DRB_ERR_TMEM>(smem_u32(&ctl.accfull[c & 1]), (c >> 1) & 1, spent);
      tc_fence_after();
      const float f = __half2float(h);
      // columns behind nc hold anything and are not stored
      const uint32_t at = td + (c & 1) * MAX_C;
      auto drained = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.accfree[c & 1]);
      };
      if (g < groups) {
#pragma unroll
        for (int j = 0; j < 64; j += 32)
          if (j < nc) {
            uint32_t d[32];
            tmem_ld32(at + j, d);
            if (j + 32 >= nc) drained();
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[j + e] = fmaf(f, __uint_as_float(d[e]), acc[j + e]);
          }
        if (nc > 64) {
          uint32_t d[16];
          tmem_ld16(at + 64, d);
          drained();
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[64 + e] = fmaf(f, __uint_as_float(d[e]), acc[64 + e]);
        }
      } else {
        // an adapter's sums join its own rows alone: zeros of v against a NaN or an infinity of B are NaNs in every other row
        const int ad = ctl.diff[g - groups];
#pragma unroll
        for (int j = 0; j < MAX_C; j += 16)
          if (j < nc) {
            const unsigned own = __ballot_sync(0xffffffffu, ctl.who[j + (lane & 15)] == ad);
            uint32_t d[16];
            tmem_ld16(at + j, d);
            if (j + 16 >= nc) drained();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if ((own >> e) & 1u) acc[j + e] += __uint_as_float(d[e]);
          }
      }
      if (++g == seq) {
        g = 0;
        if (o < p.n) {
          float* y = p.y + (size_t)row0 * p.n + o;
          const float* res = p.res ? p.res + (size_t)row0 * p.n + o : nullptr;
#pragma unroll
          for (int j = 0; j < MAX_C; j += 8) {
            if (j >= cols) break;
            float add[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              add[e] = res && j + e < cols ? __ldcg(res) : 0.f;
              if (res) res += p.n;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e, y += p.n)
              if (j + e < cols) *y = acc[j + e] + add[e];
          }
        }
      }
    }
  } else if (warp == MMA_WARP) {
    const uint32_t idesc = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(nc >> 3) << 17) | (128u >> 4 << 24);
    const uint32_t idesc_bf16 = idesc | (1u << 7) | (1u << 10);
    for (int c = 0, g = 0; c < total; ++c) {
      const int s = c % NA;
      mbar_wait_ring<DRB_ERR_FULL_WAIT>(smem_u32(&ctl.full[s]), (c / NA) & 1, spent);
      if (c > 1) mbar_wait_ring<DRB_ERR_TMEM>(smem_u32(&ctl.accfree[c & 1]), ((c >> 1) - 1) & 1, spent);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem + (c & 1) * MAX_C, ac = tmem + A_COL0 + 64 * s;
        const uint64_t bd = smem_desc(xst + s * xstage, 1024);
        if (g < groups) {
          for (int k = 0; k < 8; ++k) mma_f16_ts(d, ac + 8 * k, bd + (uint64_t)((k >> 2) * (box >> 4) + (k & 3) * 2), idesc, k > 0);
        } else {
          for (int l = 2; l >= 0; --l)  // the smallest term first
            for (int k = 0; k < 4; ++k) mma_f16_ts(d, ac + 8 * k, bd + (uint64_t)(l * (box >> 4) + k * 2), idesc_bf16, l < 2 || k > 0);
        }
        mma_commit(&ctl.done[s]);
        mma_commit(&ctl.accfull[c & 1]);
      }
      __syncwarp();
      if (++g == seq) g = 0;
    }
    if (spent) linger();
  } else if (warp == LOAD_WARP) {
    if (elect_one()) {
      if (p.rank == 0) pdl_wait();  // x
      for (int c = 0, g = 0; c < total; ++c) {
        const int s = c % NA, use = c / NA;
        if (use > 0) mbar_wait_ring<DRB_ERR_EMPTY_WAIT>(smem_u32(&ctl.done[s]), (use - 1) & 1, spent);
        if (g < groups) {
          unsigned char* xs = xst + s * xstage;
          mbar_expect_tx(&ctl.full[s], 2 * box);
          tma_load_2d(xs, &maps.x, g * 128, row0, &ctl.full[s]);
          tma_load_2d(xs + box, &maps.x, g * 128 + 64, row0, &ctl.full[s]);
        } else {
          mbar_arrive(&ctl.full[s]);
        }
        // x first: its stage was free two stretches ago, the raw stage in question only just
        while (wi < nw && wi < c / seq * groups + min(g, groups) + NRAW) load_w();
        if (++g == seq) g = 0;
      }
      if (spent) linger();
    }
    __syncwarp();
  } else if (warp == WHO_WARP) {  // the adapters' rows of B for the first tile come to L2 meanwhile
    for (int i = 0; i < ndiff; ++i)
      for (int r = lane; r < 128; r += 32) prefetch_line_l2(p.b + ((size_t)ctl.diff[i] * p.n + min(first * 128 + r, p.n - 1)) * p.rank);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

static int map_2d(CUtensorMap* m, CUtensorMapDataType type, const void* p, uint64_t inner, uint64_t rows, uint64_t stride, unsigned box0, unsigned box1) {
  const cuuint64_t dims[2] = {inner, rows}, strides[1] = {stride};
  const cuuint32_t box[2] = {box0, box1};
  return pft::encode(m, type, 2, p, dims, strides, box);
}

// As few passes over the weights as tiles of up to 80 rows of x allow, equally wide.
template <bool F16>
static int launch(const pl::Args& p, const DrbDevice& dev, cudaStream_t st) {
  const int ny = (p.rows + MAX_C - 1) / MAX_C, nc = ((p.rows + ny - 1) / ny + 15) / 16 * 16, passes = (p.rows + nc - 1) / nc;
  const int tiles = (p.n + 127) / 128;
  Maps maps;
  int e = map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, p.k, p.n, p.k, 128, 128);
  if (!e) e = map_2d(&maps.x, F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.x, p.k, p.rows, (uint64_t)p.k * 2, 64, nc);
  if (e) return e;
  if (p.rank > 0) pl::launch_shrink<F16>(p, dev, true, st);
  // A pass has its blocks for good, so the rows are shared out evenly, not nc a pass: 100 rows of 64 adapters were 64 and 36, with as many adapters
  const int blocks = dev.sms / passes, each = (p.rows + passes - 1) / passes;
  drb_launch(k_proj_rows<F16>, dim3(blocks < 1 ? 1 : blocks < tiles ? blocks : tiles, passes), dim3(THREADS), smem_bytes(nc), st, dev.pdl, maps, p, nc, each, tiles);
  return 0;
}

// Which form: both sides' times in ns, from measurements of 1 to 300 rows, 2048 to 65536 outputs and 2048 to 8192 inputs (within a tenth or two).
// The mma.sync form takes so many ns a million weights and pass, by its column tiles, and a launch's start for every 32 passes, whose
// clusters are about what is resident at once; a row's adapter costs it the row's outputs. The tcgen05 form takes
// 450 ns for 128 inputs of a tile (0.49 to 0.55 us where a block has several) and 1250 for each different adapter of the tile's rows, every wave of tiles. The host does not know how many
// meet in a tile: all that there are, up to 64 rows, which are likely to be as many requests; a quarter of them beyond, where neighbours are
// likely to be of one. Measured, mma.sync / tcgen05, us: 8192 x 2048 24 rows 9.0 / 10.1, 48 rows 16.2 / 11.1; 32768 x 2048 24 rows 27 / 19; 2048 x 4096 64
// rows 10.9 / 18.7; 8192 x 2048, 48 rows of 8 adapters 25.3 / 22.7, of 16 25.4 / 34.9.
static bool many(const pl::Args& p, const DrbDevice& dev, int nc, int row_tiles) {
  constexpr long long PER_PASS[4] = {210, 245, 355, 400};
  const int nt = p.rows > 24 ? 4 : (p.rows + 7) / 8, passes = (p.rows + 8 * nt - 1) / (8 * nt);
  const long long tiles = (p.n + 127) / 128, blocks = tiles * row_tiles, waves = (blocks + dev.sms - 1) / dev.sms;
  const int most = p.rank > 0 ? (p.adapters < nc ? p.adapters : nc) : 0, met = p.rows <= 64 ? (most < p.rows ? most : p.rows) : (most + 3) / 4;
  if (passes > 65535) return true;
  long long few = 3500 * (1 + (passes - 1) / 32) + PER_PASS[nt - 1] * passes * ((long long)p.n * p.k / 1000) / 1000, tc = 3000 + waves * (450 * (p.k / 128) + 1250 * met);
  if (p.rank > 0) few += 3000 + (long long)p.n * (p.rows > 8 ? p.rows : 8) / 100, tc += 2500;
  return tc < few;
}

// Whether k_proj_rows was compiled with the registers that its roles share out. Where it was not, the mma.sync form takes every call, up to as many rows as a grid
// has passes, and nothing else of the library is touched.
static bool g_fits[pl::MAX_DEVICES];

template <bool F16>
static int launch_any(const pl::Args& p, const DrbDevice& dev, cudaStream_t st) {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= pl::MAX_DEVICES) return -2;
  const int ny = (p.rows + MAX_C - 1) / MAX_C, nc = ((p.rows + ny - 1) / ny + 15) / 16 * 16;
  if (g_fits[d] && many(p, dev, nc, (p.rows + nc - 1) / nc)) return launch<F16>(p, dev, st);
  if (p.rows > 65535 * 32) return -1;
  return pl::launch_few<F16>(p, dev, st);
}

static cudaError_t configure_all() {
  cudaError_t e;
  if ((e = cudaFuncSetAttribute(k_proj_rows<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(MAX_C))) != cudaSuccess) return e;
  if ((e = cudaFuncSetAttribute(k_proj_rows<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(MAX_C))) != cudaSuccess) return e;
  cudaFuncAttributes a, b;  // with fewer registers at the launch than the shares add up to the warps would wait for the rest
  if ((e = cudaFuncGetAttributes(&a, k_proj_rows<true>)) != cudaSuccess || (e = cudaFuncGetAttributes(&b, k_proj_rows<false>)) != cudaSuccess) return e;
  int d = 0;
  if ((e = cudaGetDevice(&d)) != cudaSuccess) return e;
  if (d < 0 || d >= pl::MAX_DEVICES) return cudaErrorInvalidDevice;
  g_fits[d] = a.numRegs >= LAUNCH_REGS && b.numRegs >= LAUNCH_REGS;
  if ((e = drb_carveout(k_proj_rows<true>)) != cudaSuccess) return e;
  return drb_carveout(k_proj_rows<false>);
}

}  // namespace pr

extern "C" int drb_proj_q8_lora(const int8_t* w, const __half* s, const void* x, int x_type, const __nv_bfloat16* a, const __nv_bfloat16* b,
                                const float* scale, const int* adapter_of, int adapters, int rank, const float* res, float* y, float* v, int rows, int n,
                                int k, cudaStream_t st) {
  if ((x_type != 1 && x_type != 2) || rows < 0 || rows > 65535 * 64 || n < 1 || k < 128 || k > pl::MAX_K || k % 128 || rank < 0 || rank > pl::MAX_RANK || rank % 8 || adapters < 0)
    return -1;
  if (!w || !s || !x || !y || (rank > 0 && (!a || !b || !scale || !adapter_of || !v))) return -1;
  const auto off = [](const void* p, unsigned m) { return ((uintptr_t)p & (m - 1)) != 0; };
  if (off(w, 16) || off(s, 2) || off(x, 16) || off(y, 4) || off(res, 4)) return -3;
  if (rank > 0 && (off(a, 16) || off(b, 16) || off(v, 16) || off(scale, 4) || off(adapter_of, 4))) return -3;
  const DrbDevice& dev = drb_device(st);
  if (!dev.ready) return -2;
  if (rows == 0) return 0;
  const pl::Args p = {w, s, x, a, b, scale, res, adapter_of, y, v, adapters, adapters > 0 ? rank : 0, rows, n, k};
  return x_type == 2 ? pr::launch_any<true>(p, dev, st) : pr::launch_any<false>(p, dev, st);
}
