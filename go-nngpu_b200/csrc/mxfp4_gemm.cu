// C = act(A . B^T + bias) on packed MXFP4 operands (layout: Mxfp4Layout in kernels.h), on the
// block-scaled 4-bit form of the tensor cores (tcgen05.mma kind::mxf4): 64 of K an instruction,
// one scale byte for 32 of K, both scales applied by the tensor core, fp32 accumulators in TMEM.
//
// The rows of B (a layer's outputs) are the rows of the instruction's result and the rows of A
// (the batch) its columns: a warp that reads the accumulators holds 32 neighbouring outputs of
// one batch row in each register, so that every store covers 128 contiguous bytes of C whatever N
// and its alignment, and a batch of a few rows wastes columns of a narrow tile and not rows of a
// tall one.
//
// Shared memory holds stages of two k blocks of 256: 128 bytes of codes per row and block, fetched by
// TMA with the 128-byte swizzle (both blocks in one box where the rows are whole blocks: 256
// contiguous bytes a row), and the scales of 128 rows as four tiles of 512 bytes, which tcgen05.cp
// moves into TMEM right before the MMAs that read them.  Each stage has its own place for scales in
// TMEM: it is written again only after the stage's barrier has seen the MMAs retire.
#include <algorithm>
#include <cstring>

#include "activation.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "mxfp4.cuh"
#include "ptx.cuh"
#include "status.cuh"
#include "tmap.h"

namespace gonn {

namespace {

constexpr uint32_t ROWS = 128;                 // rows of B in a CTA's tile
constexpr uint32_t BLOCK_BYTES = 128;          // code bytes of a row in a k block: 256 of K
constexpr uint32_t SUB = 2;                    // k blocks a stage
constexpr uint32_t STEPS = 4;                  // MMAs (64 of K) a k block
constexpr uint32_t ROW_CODES = ROWS * BLOCK_BYTES;  // of one k block
constexpr uint32_t SCALE_TILE = 512;           // scales of 128 rows x 128 of K
constexpr uint32_t SCALES = 2 * SUB;           // scale tiles of 128 rows in a stage
constexpr uint32_t SMEM_LIMIT = 227 * 1024;
// The tensor core adds into its accumulators with truncation, so the error grows with the number
// of MMAs: on blocks whose scales differ by 2^4 (one standard deviation) 1.8e-7 relative at K =
// 4096, 6.0e-7 at 8192, 3.8e-6 at 16384, against 1.6e-7, 4.5e-7 and 1.2e-6 of float32 sums.  After
// this many stages (4096 of K) the accumulators are therefore added to sums in registers, with
// rounding to nearest, and start again.
constexpr uint32_t CHUNK = 8;

struct Params {
  uint32_t M, N;          // rows of A (columns of the tile), rows of B (rows of the tile)
  uint32_t tiles_n, tiles_m, num_tiles;
  uint32_t kblocks, ksteps, stages;  // k blocks, MMAs and stages along K
  uint32_t splits, per_split;        // single-CTA kernel: CTAs (of one cluster) that share a tile's K, stages each
  uint32_t rows_grouped, cols_grouped;  // both k blocks of a stage come in one box
  float* c;
  const float* bias;
  int act;
  float act_param;
  const float* x;         // the float32 matrix that a fused kernel quantises itself: [M, K]
  uint32_t K;
  uint32_t x_vec;         // its rows start on 16 bytes
  GemmStatus* status;
};

// The epilogues are unrolled over their registers.  With the choice of activation inside every
// copy the code outgrew the instruction cache: the 4096^3 product took 89 us, 59 us without its
// stores.  So the two common cases are compiled apart and the rest is one out-of-line call.
enum ActClass : int { IDENTITY = 0, RELU = 1, OTHER = 2 };
__device__ __noinline__ float other_activation(float v, int act, float param) { return apply_act(v, act, param); }
template <int CLASS>
__device__ __forceinline__ float finish(const Params& p, float sum, float bias) {
  const float v = sum + bias;
  return CLASS == IDENTITY ? v : CLASS == RELU ? fmaxf(v, 0.f) : other_activation(v, p.act, p.act_param);
}

// Adds 32 accumulator columns to (or, the first time, puts them into) a thread's sums.
__device__ __forceinline__ void take_columns(uint32_t taddr, float (&sum)[32], bool first) {
  uint32_t v[32];
  ptx::tmem_ld_32x32(taddr, v);
  ptx::tmem_ld_wait();
#pragma unroll
  for (uint32_t j = 0; j < 32; ++j) sum[j] = first ? __uint_as_float(v[j]) : sum[j] + __uint_as_float(v[j]);
}

// Scales: no swizzle, groups of 8 rows of 16 bytes 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return ptx::smem_desc(0, 0, 128) | uint64_t(addr >> 4);
}
// Codes: K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t code_desc(uint32_t addr) {
  return ptx::smem_desc(2, 16, 1024) | uint64_t(addr >> 4);
}

// The codes of one operand's tile for a stage.
template <bool PAIR>
__device__ __forceinline__ void load_codes(uint32_t dst, const CUtensorMap* m, uint32_t grouped, uint32_t stage,
                                           uint32_t row, uint32_t tile_bytes, uint32_t bar) {
  if (grouped) {
    if (PAIR) ptx::tma_load_3d_pair(dst, m, 0, int32_t(row), int32_t(stage * SUB), bar);
    else ptx::tma_load_3d(dst, m, 0, int32_t(row), int32_t(stage * SUB), bar);
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < SUB; ++j) {
    const int32_t k = int32_t((stage * SUB + j) * BLOCK_BYTES);
    if (PAIR) ptx::tma_load_2d_pair(dst + j * tile_bytes, m, k, int32_t(row), bar);
    else ptx::tma_load_2d(dst + j * tile_bytes, m, k, int32_t(row), bar);
  }
}

// ---- one CTA per tile of 128 outputs x BN batch rows, or a cluster that shares its K ------
// Warp 0 loads, warp 1 issues the MMAs, warps 2-5 read the accumulators out.  A product with few
// tiles gives each tile to a cluster of up to 4 CTAs: each multiplies its share of K, leaves its
// sums in its shared memory, and then adds up every `splits`-th column over all of them, in the
// order of the shares.
//
// FLOAT_A: A is still float32 and has at most 8 rows.  Warps 2-5, idle while the weights stream
// by, quantise it stage by stage into the place where the tensor core looks for its codes and
// scales: one launch instead of two.  (Every CTA does all of it, which is why it stops at 8 rows.)
constexpr uint32_t SINGLE_THREADS = 192;
constexpr uint32_t FLOAT_ROWS = kMxfp4FloatRows;
constexpr uint32_t MAX_SPLITS = 4;

template <int BN, int STAGES>
struct SingleShape {
  static constexpr uint32_t COL_CODES = BN * BLOCK_BYTES;
  static constexpr uint32_t COLS_AT = SUB * ROW_CODES, ROW_SCALES_AT = COLS_AT + SUB * COL_CODES,
                            COL_SCALES_AT = ROW_SCALES_AT + SCALES * SCALE_TILE,
                            STAGE = COL_SCALES_AT + SCALES * SCALE_TILE;
  static constexpr uint32_t SMEM = STAGES * STAGE + 1024 + 256;
  static constexpr uint32_t STAGE_COLS = 2 * SCALES * 4;  // of TMEM, for scales
  static constexpr uint32_t USED = BN + STAGES * STAGE_COLS;
  static constexpr uint32_t TMEM = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(STAGES * STAGE >= BN * ROWS * 4, "the stages hold the sums of a share");
};

// This lane's 8 floats of every row for the k block kb.
__device__ __forceinline__ void load_floats(const Params& p, uint32_t lane, uint32_t kb, float (&v)[FLOAT_ROWS][8]) {
  const uint32_t k = kb * 256u + lane * 8u;
#pragma unroll
  for (uint32_t m = 0; m < FLOAT_ROWS; ++m) {
    if (m >= p.M) break;
    const float* x = p.x + uint64_t(m) * p.K + k;
    if (p.x_vec && k + 8 <= p.K) {
      const float4 a = reinterpret_cast<const float4*>(x)[0], b = reinterpret_cast<const float4*>(x)[1];
      v[m][0] = a.x; v[m][1] = a.y; v[m][2] = a.z; v[m][3] = a.w;
      v[m][4] = b.x; v[m][5] = b.y; v[m][6] = b.z; v[m][7] = b.w;
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) v[m][j] = k + j < p.K ? x[j] : 0.f;
    }
  }
}
// Quantises them into a stage's k block: the same codes and scales as launch_mxfp4_quantize, the codes at
// their place in the 128-byte swizzle (16-byte chunks XOR-ed with the row).
__device__ __forceinline__ void quantize_block(const Params& p, uint32_t lane, const float (&v)[FLOAT_ROWS][8],
                                               uint8_t* codes, uint8_t* scales) {
#pragma unroll
  for (uint32_t m = 0; m < FLOAT_ROWS; ++m) {
    if (m >= p.M) break;  // the same for the whole warp
    uint32_t amax = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[m][j]) & 0x7fffffffu);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t byte = mxfp4::scale_byte(amax);
    const float f = mxfp4::inverse_scale(byte);
    uint32_t word = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) word |= mxfp4::encode2(v[m][2 * j] * f, v[m][2 * j + 1] * f) << (8 * j);
    if (byte == mxfp4::kScaleNan) word = 0;
    *reinterpret_cast<uint32_t*>(codes + m * BLOCK_BYTES + (((lane >> 2) ^ (m & 7u)) << 4) + (lane & 3u) * 4) = word;
    uint32_t four = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) four |= __shfl_sync(0xffffffffu, byte, (lane & 16u) + j * 4) << (8 * j);
    if ((lane & 15u) == 0) *reinterpret_cast<uint32_t*>(scales + (lane >> 4) * SCALE_TILE + m * 16) = four;
  }
}

template <int BN, int STAGES, int CLASS, bool FLOAT_A>
__global__ void __launch_bounds__(SINGLE_THREADS)
mxfp4_single_kernel(const __grid_constant__ CUtensorMap tm_rows, const __grid_constant__ CUtensorMap tm_row_scales,
                    const __grid_constant__ CUtensorMap tm_cols, const __grid_constant__ CUtensorMap tm_col_scales,
                    const __grid_constant__ Params p) {
  using S = SingleShape<BN, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  const uint32_t bar_base = base + STAGES * S::STAGE;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * STAGES), tempty_bar = tfull_bar + 8u;
  uint32_t* words = reinterpret_cast<uint32_t*>(smem_raw + pad + STAGES * S::STAGE + 8 * (2 * STAGES + 2));
  uint32_t* tmem_slot = words;
  volatile uint32_t* abort_flag = words + 1;

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tile = blockIdx.x / p.splits, split = blockIdx.x - tile * p.splits;
  const uint32_t tn = tile % p.tiles_n, tm = tile / p.tiles_n;
  const uint32_t st0 = split * p.per_split, st1 = min(st0 + p.per_split, p.stages);

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), FLOAT_A ? 1 + SUB : 1);  // the loader, and a quantising warp per k block
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(tfull_bar, 1);
    ptx::mbar_init(tempty_bar, 4);  // the reading warps
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tm_rows);
    ptx::prefetch_tmap(&tm_row_scales);
    if (!FLOAT_A) {
      ptx::prefetch_tmap(&tm_cols);
      ptx::prefetch_tmap(&tm_col_scales);
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), S::TMEM);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_release();
  ptx::grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      for (uint32_t st = st0; st < st1; ++st) {
        if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
          if (first_to_give_up(abort_flag)) report(p.status, 1, stage, tile, st);
          break;
        }
        const uint32_t fb = full_bar(stage), dst = base + stage * S::STAGE;
        ptx::mbar_arrive_expect_tx(fb, FLOAT_A ? SUB * ROW_CODES + SCALES * SCALE_TILE : S::STAGE);
        load_codes<false>(dst, &tm_rows, p.rows_grouped, st, tn * ROWS, ROW_CODES, fb);
        ptx::tma_load_3d(dst + S::ROW_SCALES_AT, &tm_row_scales, 0, int32_t(st * SCALES), int32_t(tn), fb);
        if (!FLOAT_A) {
          load_codes<false>(dst + S::COLS_AT, &tm_cols, p.cols_grouped, st, tm * BN, S::COL_CODES, fb);
          ptx::tma_load_3d(dst + S::COL_SCALES_AT, &tm_col_scales, 0, int32_t(st * SCALES), int32_t(tm * BN / 128), fb);
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp runs the loop and one lane issues: what the instructions take stays in
    // uniform registers.
    constexpr uint32_t idesc0 = ptx::make_idesc_mxf4(ROWS, BN, 0), idesc1 = ptx::make_idesc_mxf4(ROWS, BN, 1);
    // A column of TMEM holds the scales of 32 rows: where in its tile of 128 this tile's begin.  The
    // address has to be even, which is why tiles of 32 rows come alone along M.
    const uint32_t scale_column = tm * BN % 128 / 32;
    uint32_t stage = 0, phase = 0;
    for (uint32_t st = st0; st < st1; ++st) {
      const uint32_t in_chunk = (st - st0) % CHUNK;
      bool ok = true;
      if (in_chunk == 0) ok = ptx::mbar_wait(tempty_bar, ((st - st0) / CHUNK & 1u) ^ 1u, abort_flag);
      ok = ok && ptx::mbar_wait(full_bar(stage), phase, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0 && first_to_give_up(abort_flag)) report(p.status, 2, stage, tile, st);
        break;
      }
      ptx::tc_fence_after();
      const uint32_t src = base + stage * S::STAGE;
      const uint32_t ts = tmem + BN + stage * S::STAGE_COLS;
      const uint64_t da = code_desc(src), db = code_desc(src + S::COLS_AT), ds = scale_desc(src + S::ROW_SCALES_AT);
      const uint32_t steps = min(SUB * STEPS, p.ksteps - st * SUB * STEPS);
      if (ptx::elect_one()) {
#pragma unroll
        for (uint32_t j = 0; j < 2 * SCALES; ++j)  // the rows' tiles, then the columns'
          ptx::tmem_cp_scales<false>(ts + j * 4, ds + j * (SCALE_TILE >> 4));
#pragma unroll
        for (uint32_t k = 0; k < SUB * STEPS; ++k)
          if (k < steps)
            ptx::mma_mxf4<false>(tmem, da + (k / STEPS) * (ROW_CODES >> 4) + (k % STEPS) * 2,
                                 db + (k / STEPS) * (S::COL_CODES >> 4) + (k % STEPS) * 2, (k & 1) ? idesc1 : idesc0,
                                 ts + (k >> 1) * 4, ts + SCALES * 4 + (k >> 1) * 4 + scale_column,
                                 (in_chunk || k) ? 1u : 0u);
        ptx::mma_commit(empty_bar(stage));
        if (in_chunk + 1 == CHUNK || st + 1 == st1) ptx::mma_commit(tfull_bar);
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else {
    const uint32_t quarter = warp & 3u;
    const uint32_t r = quarter * 32u + lane;       // row of the tile
    const uint64_t n = uint64_t(tn) * ROWS + r;
    const uint32_t m0 = tm * BN, cols = min(uint32_t(BN), p.M - m0);
    const uint32_t taddr = tmem + ((quarter * 32u) << 16);
    const uint32_t chunks = (st1 - st0 + CHUNK - 1) / CHUNK;
    float sum[BN / 32][32];
    bool ok = true;
    // each of the four warps quantises every fourth k block; the floats of its next one are on
    // their way meanwhile
    static_assert(CHUNK * SUB % 4 == 0, "a chunk is whole rounds of the warps");
    const uint32_t turn = warp - 2;
    float v[FLOAT_ROWS][8];
    if (FLOAT_A) load_floats(p, lane, st0 * SUB + turn, v);
    for (uint32_t ch = 0; ch < chunks; ++ch) {
      if (FLOAT_A) {
        // a chunk's stages first, then its sums: the MMAs of a chunk wait for nothing else
        const uint32_t end = min(st0 + (ch + 1) * CHUNK, st1) * SUB;
        for (uint32_t kb = (st0 + ch * CHUNK) * SUB + turn; kb < end; kb += 4) {
          const uint32_t i = kb / SUB - st0, stage = i % STAGES;
          if (!__all_sync(0xffffffffu, ptx::mbar_wait(empty_bar(stage), (i / STAGES & 1u) ^ 1u, abort_flag))) {
            if (lane == 0 && first_to_give_up(abort_flag)) report(p.status, 1, 0x200u | stage, tile, kb);
          }
          uint8_t* at = smem_raw + pad + stage * S::STAGE;  // (past the end of K: zeros)
          quantize_block(p, lane, v, at + S::COLS_AT + kb % SUB * S::COL_CODES,
                         at + S::COL_SCALES_AT + kb % SUB * 2 * SCALE_TILE);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(full_bar(stage));
          load_floats(p, lane, kb + 4, v);
        }
      }
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(tfull_bar, ch & 1u, abort_flag));
      if (!ok) {
        if (lane == 0 && first_to_give_up(abort_flag)) report(p.status, 3, 0, tile, ch);
        break;
      }
      ptx::tc_fence_after();
#pragma unroll
      for (uint32_t c = 0; c < BN / 32; ++c)
        if (c * 32 < cols) take_columns(taddr + c * 32, sum[c], ch == 0);
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(tempty_bar);
    }
    if (ok && p.splits == 1 && n < p.N) {
      const float bias = p.bias ? p.bias[n] : 0.f;
      float* out = p.c + uint64_t(m0) * p.N + n;
#pragma unroll
      for (uint32_t c = 0; c < BN; ++c, out += p.N)
        if (c < cols) *out = finish<CLASS>(p, sum[c / 32][c % 32], bias);
    } else if (ok && p.splits > 1) {
      // every MMA of this CTA has retired and with it every read of the stages
      float* part = reinterpret_cast<float*>(smem_raw + pad) + r;
#pragma unroll
      for (uint32_t c = 0; c < BN; ++c)
        if (c < cols) part[c * ROWS] = sum[c / 32][c % 32];
    }
  }

  if (p.splits > 1) {
    __syncthreads();
    ptx::cluster_sync_all();  // the sums of every share are in place
    if (warp >= 2) {
      // A warp takes whole columns, four rows a lane.  All shares of a column are asked for
      // before the first is added (a read of another CTA's shared memory takes a good 200 ns:
      // one at a time, the 64 columns of a CTA cost 15 us), two columns in flight.
      const uint32_t r = lane * 4;
      const uint64_t n = uint64_t(tn) * ROWS + r;
      const uint32_t m0 = tm * BN, cols = min(uint32_t(BN), p.M - m0);
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (n + i < p.N) bias[i] = p.bias[n + i];
      }
      const uint32_t step = 4 * p.splits;
#pragma unroll 2
      for (uint32_t c = (warp & 3u) * p.splits + split; c < cols; c += step) {
        float4 part[MAX_SPLITS];
#pragma unroll
        for (uint32_t s = 0; s < MAX_SPLITS; ++s)
          if (s < p.splits) part[s] = ptx::ld_shared_cluster_16(ptx::mapa_shared(base + (c * ROWS + r) * 4, s));
        float4 sum = part[0];
#pragma unroll
        for (uint32_t s = 1; s < MAX_SPLITS; ++s)
          if (s < p.splits) {
            sum.x += part[s].x;
            sum.y += part[s].y;
            sum.z += part[s].z;
            sum.w += part[s].w;
          }
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        float* out = p.c + (uint64_t(m0) + c) * p.N + n;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (n + i < p.N) out[i] = finish<CLASS>(p, v[i], bias[i]);
      }
    }
    ptx::cluster_sync_all();  // no CTA leaves while another still reads its sums
  }

  ptx::tc_fence_before();
  __syncthreads();
  wait_out(abort_flag);
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, S::TMEM);
  }
}

// ---- CTA pairs: 256 outputs x 256 batch rows, persistent ---------------------------------
// Two CTAs share one MMA (M = 256): CTA r holds the codes of rows r*128.. of the tile's B and of
// r*128.. of its A, the scales of its own rows of B and those of all 256 rows of A.  The single
// 256-column accumulator leaves room in TMEM for every stage's scales; the eight warps that read
// it out take it into registers at once and hand TMEM back before they store, so the next tile's
// MMAs wait only for the read, while its loads have been running all the time.
constexpr uint32_t PAIR_THREADS = 320;
constexpr uint32_t PAIR_COLS = 256;
constexpr uint32_t PAIR_COLS_AT = SUB * ROW_CODES, PAIR_ROW_SCALES_AT = 2 * SUB * ROW_CODES,
                   PAIR_COL_SCALES_AT = PAIR_ROW_SCALES_AT + SCALES * SCALE_TILE,
                   PAIR_STAGE = PAIR_COL_SCALES_AT + 2 * SCALES * SCALE_TILE;
constexpr uint32_t PAIR_STAGES = 3;
constexpr uint32_t PAIR_STAGE_COLS = 3 * SCALES * 4;  // of TMEM, for scales
constexpr uint32_t PAIR_SMEM = PAIR_STAGES * PAIR_STAGE + 1024 + 256;
static_assert(PAIR_SMEM <= SMEM_LIMIT && PAIR_COLS + PAIR_STAGES * PAIR_STAGE_COLS <= 512, "pair kernel resources");

__device__ __forceinline__ void pair_tile(const Params& p, uint32_t t, uint32_t& tn, uint32_t& tm) {
  // groups of 8 tiles of B sweep A together
  const uint32_t per = 8 * p.tiles_m, g = t / per, first = g * 8;
  const uint32_t wide = min(8u, p.tiles_n - first), r = t - g * per;
  tn = first + r % wide;
  tm = r / wide;
}

template <int CLASS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tm_rows, const __grid_constant__ CUtensorMap tm_row_scales,
                  const __grid_constant__ CUtensorMap tm_cols, const __grid_constant__ CUtensorMap tm_col_scales,
                  const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  const uint32_t bar_base = base + PAIR_STAGES * PAIR_STAGE;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (PAIR_STAGES + s); };
  const uint32_t tfull_bar = bar_base + 8u * (2 * PAIR_STAGES), tempty_bar = tfull_bar + 8u;
  uint32_t* words = reinterpret_cast<uint32_t*>(smem_raw + pad + PAIR_STAGES * PAIR_STAGE + 8 * (2 * PAIR_STAGES + 2));
  uint32_t* tmem_slot = words;
  volatile uint32_t* abort_flag = words + 1;

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < PAIR_STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(tfull_bar, 1);
    ptx::mbar_init(tempty_bar, 16);  // the eight reading warps of both CTAs
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tm_rows);
    ptx::prefetch_tmap(&tm_row_scales);
    ptx::prefetch_tmap(&tm_cols);
    ptx::prefetch_tmap(&tm_col_scales);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_release();
  ptx::grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool alive = true;
      for (uint32_t t = pair; alive && t < p.num_tiles; t += pairs) {
        uint32_t tn, tm;
        pair_tile(p, t, tn, tm);
        for (uint32_t st = 0; st < p.stages; ++st) {
          if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
            if (first_to_give_up(abort_flag)) report(p.status, 1, stage, t, st);
            alive = false;
            break;
          }
          if (leader) ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * PAIR_STAGE);
          const uint32_t fb = ptx::mapa_shared(full_bar(stage), 0), dst = base + stage * PAIR_STAGE;
          load_codes<true>(dst, &tm_rows, p.rows_grouped, st, (tn * 2 + rank) * ROWS, ROW_CODES, fb);
          load_codes<true>(dst + PAIR_COLS_AT, &tm_cols, p.cols_grouped, st, (tm * 2 + rank) * ROWS, ROW_CODES, fb);
          ptx::tma_load_3d_pair(dst + PAIR_ROW_SCALES_AT, &tm_row_scales, 0, int32_t(st * SCALES),
                                int32_t(tn * 2 + rank), fb);
          ptx::tma_load_3d_pair(dst + PAIR_COL_SCALES_AT, &tm_col_scales, 0, int32_t(st * SCALES), int32_t(tm * 2), fb);
          if (++stage == PAIR_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp runs the loop and one lane issues: what the instructions take stays in
    // uniform registers.
    if (leader) {
      constexpr uint32_t idesc0 = ptx::make_idesc_mxf4(256, PAIR_COLS, 0), idesc1 = ptx::make_idesc_mxf4(256, PAIR_COLS, 1);
      uint32_t stage = 0, phase = 0, drained = 1;
      bool alive = true;
      for (uint32_t t = pair; alive && t < p.num_tiles; t += pairs) {
        uint32_t in_chunk = 0;
        for (uint32_t st = 0; st < p.stages; ++st) {
          bool ok = true;
          if (in_chunk == 0) {
            ok = ptx::mbar_wait(tempty_bar, drained, abort_flag);
            drained ^= 1u;
          }
          ok = ok && ptx::mbar_wait(full_bar(stage), phase, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            if (lane == 0 && first_to_give_up(abort_flag)) report(p.status, 2, stage, t, st);
            alive = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t src = base + stage * PAIR_STAGE;
          // per stage: 4 columns for each of the rows' four scale tiles, 8 (128 + 128 rows) for each
          // of the columns' four
          const uint32_t ts = tmem + PAIR_COLS + stage * PAIR_STAGE_COLS, tc = ts + SCALES * 4;
          const uint64_t da = code_desc(src), db = code_desc(src + PAIR_COLS_AT),
                         ds = scale_desc(src + PAIR_ROW_SCALES_AT), dc = scale_desc(src + PAIR_COL_SCALES_AT);
          const uint32_t steps = min(SUB * STEPS, p.ksteps - st * SUB * STEPS);
          if (ptx::elect_one()) {
#pragma unroll
            for (uint32_t k = 0; k < SCALES; ++k) {
              ptx::tmem_cp_scales<true>(ts + k * 4, ds + k * (SCALE_TILE >> 4));
#pragma unroll
              for (uint32_t h = 0; h < 2; ++h)
                ptx::tmem_cp_scales<true>(tc + k * 8 + h * 4, dc + (h * SCALES + k) * (SCALE_TILE >> 4));
            }
#pragma unroll
            for (uint32_t k = 0; k < SUB * STEPS; ++k)
              if (k < steps)
                ptx::mma_mxf4<true>(tmem, da + (k / STEPS) * (ROW_CODES >> 4) + (k % STEPS) * 2,
                                    db + (k / STEPS) * (ROW_CODES >> 4) + (k % STEPS) * 2, (k & 1) ? idesc1 : idesc0,
                                    ts + (k >> 1) * 4, tc + (k >> 1) * 8, (in_chunk || k) ? 1u : 0u);
            ptx::mma_commit_pair(empty_bar(stage), 3);
            if (in_chunk + 1 == CHUNK || st + 1 == p.stages) ptx::mma_commit_pair(tfull_bar, 3);
          }
          __syncwarp();
          if (++in_chunk == CHUNK) in_chunk = 0;
          if (++stage == PAIR_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else {
    const uint32_t quarter = warp & 3u, half = (warp - 2u) >> 2;
    const uint32_t taddr = tmem + ((quarter * 32u) << 16) + half * 128u;
    const uint32_t chunks = (p.stages + CHUNK - 1) / CHUNK;
    uint32_t filled = 0;
    for (uint32_t t = pair; t < p.num_tiles; t += pairs) {
      uint32_t tn, tm;
      pair_tile(p, t, tn, tm);
      float sum[4][32];
      bool ok = true;
      for (uint32_t ch = 0; ch < chunks; ++ch) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(tfull_bar, filled, abort_flag));
        filled ^= 1u;
        if (!ok) break;
        ptx::tc_fence_after();
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) take_columns(taddr + c * 32u, sum[c], ch == 0);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(tempty_bar, 0));
      }
      if (!ok) {
        if (lane == 0 && first_to_give_up(abort_flag)) report(p.status, 3, 0, t, 0);
        break;
      }
      const uint64_t n = uint64_t(tn * 2 + rank) * ROWS + quarter * 32u + lane;
      const uint32_t m0 = tm * PAIR_COLS + half * 128u;
      float* out = p.c + uint64_t(m0) * p.N + n;
      if (n < p.N) {
        const float bias = p.bias ? p.bias[n] : 0.f;
        if (m0 + 128 <= p.M) {
#pragma unroll
          for (uint32_t j = 0; j < 128; ++j, out += p.N) *out = finish<CLASS>(p, sum[j / 32][j % 32], bias);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 128; ++j, out += p.N)
            if (m0 + j < p.M) *out = finish<CLASS>(p, sum[j / 32][j % 32], bias);
        }
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  wait_out(abort_flag);
  __syncthreads();
  ptx::cluster_sync_all();  // neither CTA leaves while the other can still signal or read it
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
}

// ---- host side -----------------------------------------------------------------------
// Codes as a byte matrix: boxes of 128 bytes x `box_rows` rows; or, for rows of whole k blocks, as
// [k block, row, 128 bytes] with both k blocks of a stage in one box (*grouped).
bool code_map(CUtensorMap* map, const void* packed, const Mxfp4Layout& l, uint32_t box_rows, uint32_t* grouped) {
  *grouped = 0;
  if (l.row_bytes % BLOCK_BYTES == 0) {
    const uint64_t dims[3] = {BLOCK_BYTES, l.rows, l.row_bytes / BLOCK_BYTES}, strides[2] = {l.row_bytes, BLOCK_BYTES};
    const uint32_t box[3] = {BLOCK_BYTES, box_rows, SUB};
    // (the driver may refuse strides in this order)
    *grouped = encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, packed, dims, strides, box,
                                 CU_TENSOR_MAP_SWIZZLE_128B);
    if (*grouped) return true;
  }
  const uint64_t dims[2] = {l.row_bytes, l.rows}, strides[1] = {l.row_bytes};
  const uint32_t box[2] = {BLOCK_BYTES, box_rows};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, packed, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}
// Scale tiles of 512 bytes: boxes of a stage's four along K x `tall` along the rows.
bool scale_map(CUtensorMap* map, const void* packed, const Mxfp4Layout& l, uint32_t tall) {
  const uint64_t dims[3] = {SCALE_TILE / 4, l.groups, (l.rows + 127) / 128};
  const uint64_t strides[2] = {SCALE_TILE, l.groups * SCALE_TILE};
  const uint32_t box[3] = {SCALE_TILE / 4, SCALES, tall};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3,
                           static_cast<const uint8_t*>(packed) + l.scale_offset, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <auto KERN>
bool allow_smem(uint32_t bytes) {
  static bool done[64] = {};  // per kernel and device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63]) done[dev & 63] = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) == cudaSuccess;
  return done[dev & 63];
}

template <int BN, int STAGES, int CLASS, bool FLOAT_A = false>
const char* launch_single(const Mxfp4Product& q, const Mxfp4Layout& la, const Mxfp4Layout& lb, Params p,
                          cudaStream_t stream) {
  CUtensorMap rows, row_scales, cols{}, col_scales{};
  if (!code_map(&rows, q.b, lb, ROWS, &p.rows_grouped) || !scale_map(&row_scales, q.b, lb, 1) ||
      (!FLOAT_A && (!code_map(&cols, q.a, la, BN, &p.cols_grouped) || !scale_map(&col_scales, q.a, la, 1))))
    return "cuTensorMapEncodeTiled failed";
  constexpr auto kern = mxfp4_single_kernel<BN, STAGES, CLASS, FLOAT_A>;
  constexpr uint32_t smem = SingleShape<BN, STAGES>::SMEM;
  static_assert(smem <= SMEM_LIMIT, "shared memory");
  if (!allow_smem<kern>(smem)) return "cudaFuncSetAttribute(max dynamic shared memory) failed";
  if (launch_kernel_cluster(kern, p.splits, dim3(p.num_tiles * p.splits), dim3(SINGLE_THREADS), smem, stream, rows,
                            row_scales, cols, col_scales, p) != cudaSuccess)
    return "product launch failed";
  return nullptr;
}

template <int CLASS>
const char* launch_pair(const Mxfp4Product& q, const Mxfp4Layout& la, const Mxfp4Layout& lb, Params p,
                        int sm_count, cudaStream_t stream) {
  CUtensorMap rows, row_scales, cols, col_scales;
  if (!code_map(&rows, q.b, lb, ROWS, &p.rows_grouped) || !scale_map(&row_scales, q.b, lb, 1) ||
      !code_map(&cols, q.a, la, ROWS, &p.cols_grouped) ||
      !scale_map(&col_scales, q.a, la, 2))
    return "cuTensorMapEncodeTiled failed";
  constexpr auto kern = mxfp4_pair_kernel<CLASS>;
  if (!allow_smem<kern>(PAIR_SMEM)) return "cudaFuncSetAttribute(max dynamic shared memory) failed";
  const uint32_t pairs = std::min(uint32_t(sm_count) / 2, p.num_tiles);
  if (launch_kernel(kern, dim3(2 * pairs), dim3(PAIR_THREADS), PAIR_SMEM, stream, rows, row_scales, cols, col_scales,
                    p) != cudaSuccess)
    return "product launch failed";
  return nullptr;
}

template <int CLASS>
const char* launch_class(const Mxfp4Product& q, GemmStatus* status, int sm_count, cudaStream_t stream) {
  const Mxfp4Layout la(q.M, q.K), lb(q.N, q.K);
  Params p{};
  p.M = uint32_t(q.M);
  p.N = uint32_t(q.N);
  p.kblocks = uint32_t((lb.row_bytes + BLOCK_BYTES - 1) / BLOCK_BYTES);
  p.ksteps = uint32_t((lb.blocks + 1) / 2);
  p.stages = (p.kblocks + SUB - 1) / SUB;
  p.splits = 1;
  p.per_split = p.stages;
  p.c = q.c;
  p.bias = q.bias;
  p.act = q.act;
  p.act_param = q.act_param;
  p.status = status;
  const uint64_t pair_tiles = ((q.N + 255) / 256) * ((q.M + 255) / 256);
  if (pair_tiles >= (1ull << 30)) return "too many tiles";
  // Few pair tiles leave SMs idle: 1024^3 (16 tiles) takes 8.0 us on pairs and 4.3 us on single CTAs,
  // 512 x 4096 x 4096 (32) 11.9 and 9.5, 2048^3 (64) 9.8 and 12.5, 1024 x 4096 x 4096 (64) 12.2 and
  // 17.7.  And up to 128 rows half of each pair tile would be empty.
  if (q.M > 128 && pair_tiles >= 48) {
    p.tiles_n = uint32_t((q.N + 255) / 256);
    p.tiles_m = uint32_t((q.M + 255) / 256);
    p.num_tiles = uint32_t(pair_tiles);
    return launch_pair<CLASS>(q, la, lb, p, sm_count, stream);
  }
  // (tiles of 128 rows were slower than those of 64 at every size that comes here)
  const uint32_t bn = q.M <= 32 ? 32 : 64;
  p.tiles_n = uint32_t((q.N + ROWS - 1) / ROWS);
  p.tiles_m = uint32_t((q.M + bn - 1) / bn);
  p.num_tiles = p.tiles_n * p.tiles_m;
  // Few tiles: share each one's K among the CTAs of a cluster, where that saves more than the 2 us
  // (32 columns) or 4 us (64) that the exchange of the sums costs; a stage takes about 0.3 us.  1 x 4096
  // x 4096: 7.4 us whole, 5.5 us in 4 shares, 12.3 us in 8; 256 x 4096 x 4096: 8.9 us whole, 10.4 us in 2.
  const uint32_t least = bn == 32 ? 4 : 16;
  const uint32_t splits = std::max(1u, std::min({uint32_t(sm_count) / p.num_tiles, p.kblocks / least, MAX_SPLITS}));
  p.per_split = (p.stages + splits - 1) / splits;
  p.splits = (p.stages + p.per_split - 1) / p.per_split;
  if (q.a_float) {
    p.x = q.a_float;
    p.K = uint32_t(q.K);
    p.x_vec = (q.K & 3) == 0 && (reinterpret_cast<uintptr_t>(q.a_float) & 15u) == 0;
    return launch_single<32, 4, CLASS, true>(q, la, lb, p, stream);
  }
  return bn == 32 ? launch_single<32, 4, CLASS>(q, la, lb, p, stream)
                  : launch_single<64, 2, CLASS>(q, la, lb, p, stream);
}

}  // namespace

const char* launch_mxfp4_product(const Mxfp4Product& q, GemmStatus* status, int sm_count, cudaStream_t stream) {
  if (q.act == ACT_RELU) return launch_class<RELU>(q, status, sm_count, stream);
  if (q.act >= ACT_RELU && q.act <= ACT_GELU) return launch_class<OTHER>(q, status, sm_count, stream);
  return launch_class<IDENTITY>(q, status, sm_count, stream);
}

}  // namespace gonn
