// bf16 products grouped by ragged rows, fp32 accumulation in tensor memory: group e (an expert) owns rows off[e] .. off[e+1]
// of the token operands, any number of them, and a weight matrix W_e.
//   rows kernel    y[t, :] = x[t, :] * W_e^T  (forward)   or   dx[t, :] = dy[t, :] * W_e  (input gradient)
//   wgrad kernel   dW_e = sum over the group's rows t of dy[t, :]^T x[t, :]
// The offsets are read on the device: no synchronisation, and the host sizes the grid by an upper bound.  Each CTA makes the
// table of tiles per group from them.
//
// Rows kernel: the WEIGHTS are the M operand (128 rows a CTA, 256 a pair), the tokens the N operand.  N is a field of the
// instruction, so that a group's rows are cut into equal blocks of any multiple of 16 (32 for pairs): what a ragged end costs
// is a part of a 16-row step and not of a 128- or 256-row tile, and one token costs a pass over W_e alone.
// Wgrad kernel: the reduction runs over a group's rows, 64 at a time from off[e] on; the last block also holds rows of the
// next group.  Steps of 16 rows behind the end are not issued, and a warp zeroes the rest of the last step in both operands
// (a product with zero in one alone would still be NaN where the other holds an infinity) before the product may read it.
// Roles, ring, double-buffered accumulators and bounded waits are those of the plain GEMM.
#include "common.cuh"
#include "launch.cuh"

#include <type_traits>

namespace jpb {
namespace ragged {

constexpr int BK = 64, UMMA_K = 16;
constexpr int W_BYTES = 128 * BK * 2;          // 128 rows of the M operand per CTA and stage
constexpr int SMEM_MAX = 227 * 1024;
constexpr int BAR_BYTES = 256;
constexpr int MAX_GROUPS = 1024;
constexpr int MAX_ROWS = 0x7fffffff - (1 << 16);      // a step past the last row, by a block at most, stays within 32 bits
constexpr int TABLE_BYTES = 2 * (MAX_GROUPS + 1) * 4 + 8;
constexpr int GROUP_BLOCKS = 2048;             // token rows that are walked together: they stay in L2 while W streams

// The groups' row bounds (clamped to 0 .. rows and to be non-decreasing) in shared memory, by one warp.
__device__ __forceinline__ void make_bounds(const int* __restrict__ offsets, int groups, int rows, int* off) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int i0 = 0; i0 <= groups; i0 += 32) {
    const int i = i0 + lane;
    int v = i <= groups ? min(max(__ldg(offsets + i), 0), rows) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, u);
    }
    v = max(v, carry);
    if (i <= groups) off[i] = v;
    carry = __shfl_sync(0xffffffffu, v, 31);
  }
}
// The same, and the running numbers of tiles.
template <typename Tiles>
__device__ __forceinline__ void make_table(const int* __restrict__ offsets, int groups, int rows, int* off, int* first, Tiles tiles_of) {
  const int lane = threadIdx.x & 31;
  make_bounds(offsets, groups, rows, off);
  __syncwarp();
  int base = 0;
  for (int i0 = 0; i0 < groups; i0 += 32) {
    const int i = i0 + lane;
    const int n = i < groups ? tiles_of(off[i + 1] - off[i]) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (i < groups) first[i] = base + sum - n;
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) first[groups] = base;
}

// -------------------------------------------------------------------------------------------------------------
// rows kernel
// -------------------------------------------------------------------------------------------------------------
template <int CG, int BT>
struct RowsCfg {
  static constexpr int T_ROWS = BT / CG;       // token rows per CTA and stage
  static constexpr int T_BYTES = T_ROWS * BK * 2;
  static constexpr int BOX = T_ROWS < 64 ? T_ROWS : 64;   // token rows per copy: a short block takes as many as it needs
  static constexpr int STAGE_BYTES = W_BYTES + T_BYTES;
  static constexpr int FIT = (SMEM_MAX - 1024 - BAR_BYTES - TABLE_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = FIT < 12 ? FIT : 12;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + BAR_BYTES + TABLE_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * BT;
  static constexpr int GRAIN = 16 * CG;        // rows of a block: a multiple of this
  static_assert(STAGES >= 4 && TMEM_COLS >= 32 && TMEM_COLS <= 512 && T_BYTES % 1024 == 0, "");
};

struct RowsParams {
  const int* offsets;
  int groups, rows;
  int M, K;              // columns of the result (rows of the M operand), reduction length
  int w_blocked;         // MN-major weights through a 4-D map {64, K, M / 64, groups}: one copy per stage
  int tiles_m;
  __nv_bfloat16* D;      // [rows, M]
  int* head;             // single CTAs, or null: number of parts of the reduction, first row of a group, end of the last
  float* parts;          // [parts][rows, M]
  int* status;
};
// Parts of a long reduction where its tiles are fewer than half the SMs (SPLIT_MIN blocks of 64 at least in each).
constexpr int SPLIT_MAX = 8, SPLIT_MIN = 8;

// A group of n rows is cut into blocks of at most BT rows, as even as the grain allows: a stage of the ring carries 128 rows of
// weights whatever the block's size, so that a short block costs at least half of a whole one.
template <int BT>
__device__ __forceinline__ int blocks_of(int n) { return (n + BT - 1) / BT; }

struct RowsTile {
  int group, m_blk, t0, n;   // rows t0 .. t0 + n of the tokens
};
template <int BT, int GRAIN>
__device__ __forceinline__ RowsTile rows_tile(int tiles_m, const int* off, const int* first, int tile, int& e) {   // first: in blocks
  while (tile >= first[e + 1] * tiles_m) ++e;
  const int n = off[e + 1] - off[e], blocks = blocks_of<BT>(n), grains = (n + GRAIN - 1) / GRAIN;
  constexpr int GB = GROUP_BLOCKS / BT;
  const int i = tile - first[e] * tiles_m, per = GB * tiles_m, g = i / per, in = i - g * per;
  const int gb = min(GB, blocks - g * GB);
  const int m_blk = in / gb, b = g * GB + in - m_blk * gb;
  const int lo = int((long long)grains * b / blocks) * GRAIN, hi = int((long long)grains * (b + 1) / blocks) * GRAIN;
  return {e, m_blk, off[e] + lo, min(hi, n) - lo};
}

// SPLIT: tiles may be cut along the reduction (a kernel of its own: the tests for it cost 8 x 2048 x 512 with 2000 rows 1.8 us of 14).
template <int CG, int BT, bool W_MN, bool SPLIT>
__global__ void __launch_bounds__(192, 1)
ragged_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t, const __grid_constant__ RowsParams p) {
  using C = RowsCfg<CG, BT>;
  constexpr int STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES, GRAIN = C::GRAIN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* acc_full = bars + 2 * STAGES;
  uint64_t* acc_empty = bars + 2 * STAGES + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* off = reinterpret_cast<int*>(smem + STAGES * STAGE_BYTES + BAR_BYTES);
  int* first = off + p.groups + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? int(cluster_ctarank()) : 0;
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;
  const int k_blocks = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * CG);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_t);
  }
  if (warp == 1) {
    tmem_alloc_cg<CG>(tmem_slot, C::TMEM_COLS);
    tmem_relinquish_cg<CG>();
  }
  if (warp == 2)
    make_table(p.offsets, p.groups, p.rows, off, first, [&](int n) { return n > 0 ? blocks_of<BT>(n) : 0; });
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int blocks = first[p.groups];
  // Weight rows of a tile.  Blocks of few tokens are a pass over the weights, at 6.8 TB/s while all SMs read and 70 GB/s of an SM
  // alone: a last round of a few tiles takes as long as a quarter of a round does otherwise.  Lower tiles, whose copies overlap (in
  // L2), give that round more of them.  One token of two experts of 28672 x 4096, 448 tiles of 128 rows on 148 SMs: 86 us with
  // these, 83 with the 552 of 104 that this finds; a token of each of eight 280 and 268 (7.0 TB/s).  (Tiles of 32 rows in that round
  // alone took 90: an SM's rate falls with the size of its copies.)
  int height = 128 * CG, tiles_m = p.tiles_m;
  if constexpr (BT == 32 && !W_MN) {
    long long best = 0x7fffffffffffffffll;
    for (int h = 128; h >= 96; h -= 8) {
      const int per = (p.M + h - 1) / h, tiles = blocks * per, last = tiles % tile_step;
      const long long cost = (long long)(tiles - last) * h + (last ? max(last * h, 128 * 96) : 0);     // rows at the common rate
      if (cost < best) { best = cost; height = h; tiles_m = per; }
    }
  }
  // few tiles: their reductions in parts, which a second kernel adds up
  int splits = 1;
  if constexpr (SPLIT) splits = max(1, min(min(SPLIT_MAX, k_blocks / SPLIT_MIN), tile_step / max(1, blocks * tiles_m)));
  const int num_items = blocks * tiles_m * splits;
  auto k_from = [&](int item) { return SPLIT ? k_blocks * (item % splits) / splits : 0; };
  auto k_to = [&](int item) { return SPLIT ? k_blocks * (item % splits + 1) / splits : k_blocks; };
  auto tile_of = [&](int item) { return SPLIT ? item / splits : item; };
  if (SPLIT && blockIdx.x == 0 && threadIdx.x == 64) {
    p.head[0] = splits;
    p.head[1] = off[0];
    p.head[2] = off[p.groups];
  }

  if (warp == 0) {
    // ------------------------------- TMA producer --------------------------------------------
    uint32_t it = 0, armed = 0, armed_phase = 0;
    bool ok = true;
    int e = 0;
    for (int item = first_tile; item < num_items && ok; item += tile_step) {
      const RowsTile t = rows_tile<BT, GRAIN>(tiles_m, off, first, tile_of(item), e);
      const int kb1 = k_to(item);
      const int n_mma = (t.n + GRAIN - 1) / GRAIN * GRAIN;
      const int m0 = t.m_blk * height + rank * 128, t_rows = n_mma / CG, t0 = t.t0 + rank * t_rows;
      const uint32_t bytes = W_BYTES + (t_rows + C::BOX - 1) / C::BOX * (C::BOX * BK * 2);
      for (int kb = k_from(item); kb < kb1; ++kb) {
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1;
        if (!mbar_wait_bounded_warp(&empty[s], ph ^ 1, abort_flag, p.status)) { ok = false; break; }
        uint8_t* sw = smem + s * STAGE_BYTES;
        uint8_t* st = sw + W_BYTES;
        armed |= 1u << s;
        armed_phase = (armed_phase & ~(1u << s)) | (ph << s);
        const int k0 = kb * BK;
        if (elect_one()) {
          // (pair: all copies report to the leader's barrier, which announces both CTAs' bytes; the peer's may land first)
          if (CG == 1 || rank == 0) mbar_expect_tx(&full[s], bytes * CG);
          const uint32_t bar = CG == 2 ? mapa_u32(&full[s], 0) : smem_u32(&full[s]);
          if constexpr (CG == 2) {
            if (!W_MN) tma_load_3d_pair(sw, &map_w, bar, k0, m0, t.group);                       // box {64 k, 128 rows}
            else if (p.w_blocked) tma_load_4d_pair(sw, &map_w, bar, 0, k0, m0 >> 6, t.group);    // box {64 m, 64 k, 2 blocks}
            else {
              tma_load_3d_pair(sw, &map_w, bar, m0, k0, t.group);
              tma_load_3d_pair(sw + 8192, &map_w, bar, m0 + 64, k0, t.group);
            }
#pragma unroll
            for (int j = 0; j < C::T_ROWS; j += C::BOX)
              if (j < t_rows) tma_load_2d_pair(st + j * 128, &map_t, bar, k0, t0 + j);
          } else {
            if (!W_MN) tma_load_3d(sw, &map_w, &full[s], k0, m0, t.group);
            else if (p.w_blocked) tma_load_4d(sw, &map_w, &full[s], 0, k0, m0 >> 6, t.group);
            else {
              tma_load_3d(sw, &map_w, &full[s], m0, k0, t.group);
              tma_load_3d(sw + 8192, &map_w, &full[s], m0 + 64, k0, t.group);
            }
#pragma unroll
            for (int j = 0; j < C::T_ROWS; j += C::BOX)
              if (j < t_rows) tma_load_2d(st + j * 128, &map_t, &full[s], k0, t0 + j);
          }
        }
        __syncwarp();
        ++it;
      }
    }
    if (!ok) {
      // wait (bounded) for the copies in flight before the shared memory is released
      const uint64_t begin = globaltimer_ns();
      if (CG == 2 && rank != 0) {
        while (globaltimer_ns() - begin < 2000000) {   // they report to the leader's barriers: many times a copy's time
        }
      } else {
        for (int s = 0; s < STAGES; ++s) {
          if (!(armed & (1u << s))) continue;
          const uint32_t ph = (armed_phase >> s) & 1;
          while (!mbar_try_wait(&full[s], ph) && globaltimer_ns() - begin < wait_budget_ns()) {
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (the leader's, in a pair) ------------------------
    if (CG == 1 || rank == 0) {
      constexpr uint32_t idesc0 = make_idesc_bf16(128 * CG, 0, W_MN, 0);
      constexpr uint32_t W_STEP = (W_MN ? 2048 : 32) >> 4, T_STEP = 32 >> 4;
      const SmemDesc w_desc = W_MN ? make_smem_desc2(smem_u32(smem), 8192, 1024) : make_smem_desc2(smem_u32(smem), 16, 1024);
      const SmemDesc t_desc = make_smem_desc2(smem_u32(smem) + W_BYTES, 16, 1024);
      uint32_t it = 0, tile_i = 0;
      bool ok = true;
      int e = 0;
      for (int item = first_tile; item < num_items && ok; item += tile_step, ++tile_i) {
        const RowsTile t = rows_tile<BT, GRAIN>(tiles_m, off, first, tile_of(item), e);
        const int kb0 = k_from(item), kb1 = k_to(item);
        const uint32_t idesc = idesc0 | (uint32_t((t.n + GRAIN - 1) / GRAIN * GRAIN >> 3) << 17);
        const uint32_t acc = tile_i & 1, acc_ph = (tile_i >> 1) & 1;
        if (!mbar_wait_bounded_warp(&acc_empty[acc], acc_ph ^ 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BT;
        for (int kb = kb0; kb < kb1; ++kb) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait_bounded_warp(&full[s], ph, abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = uint32_t(s * STAGE_BYTES) >> 4;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k)
              umma_bf16_ss2_cg<CG>(d_tmem, w_desc.lo + at + k * W_STEP, w_desc.hi, t_desc.lo + at + k * T_STEP, t_desc.hi, idesc,
                                   kb > kb0 || k > 0);
            umma_commit_cg<CG>(&empty[s], 3);
          }
          __syncwarp();
          ++it;
        }
        if (ok && elect_one()) umma_commit_cg<CG>(&acc_full[acc], 3);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------- epilogue (warps 2..5) ------------------------------------------
    const int quarter = warp & 3;
    // rows of no group: zeros
    {
      const int head = off[0], tail = off[p.groups], loose = head + p.rows - tail, pieces = p.M >> 3;
      for (long long i = (long long)blockIdx.x * 128 + (threadIdx.x - 64); i < (long long)loose * pieces; i += (long long)gridDim.x * 128) {
        const int r = int(i / pieces), row = r < head ? r : tail + r - head;
        *reinterpret_cast<uint4*>(p.D + size_t(row) * p.M + (i - (long long)r * pieces) * 8) = make_uint4(0, 0, 0, 0);
      }
    }
    uint32_t tile_i = 0;
    bool ok = true;
    int e = 0;
    for (int item = first_tile; item < num_items && ok; item += tile_step, ++tile_i) {
      const RowsTile t = rows_tile<BT, GRAIN>(tiles_m, off, first, tile_of(item), e);
      const uint32_t acc = tile_i & 1, acc_ph = (tile_i >> 1) & 1;
      if (!mbar_wait_bounded_warp(&acc_full[acc], acc_ph, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      const uint32_t t_acc = tmem_base + (uint32_t(quarter * 32) << 16) + acc * BT;
      // A thread holds one column of the result, the tokens one after the other.  Neighbours trade every second value, so
      // that a lane has two columns of one token: 4 bytes a lane, two rows of 64 bytes a warp and store.
      const int at = rank * 128 + quarter * 32 + (lane & ~1), col = t.m_blk * height + at;
      const bool odd = lane & 1, in = at < height && col < p.M;
      __nv_bfloat16* d = p.D + size_t(t.t0) * p.M + col;
#pragma unroll 1
      for (int c = 0; c < t.n; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32(t_acc + c, v);
        tc_wait_ld();
        if (SPLIT && splits > 1) {
          const int own = at + odd;
          float* to = p.parts + (size_t(item % splits) * p.rows + t.t0 + c) * p.M + t.m_blk * height + own;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (in && c + j < t.n) to[size_t(j) * p.M] = __uint_as_float(v[j]);
          continue;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
          const int row = c + j + odd;
          if (in && row < t.n)
            *reinterpret_cast<uint32_t*>(d + size_t(row) * p.M) = odd ? pack_bf16(__uint_as_float(got), __uint_as_float(v[j + 1]))
                                                                       : pack_bf16(__uint_as_float(v[j]), __uint_as_float(got));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2 && rank != 0) mbar_arrive_cluster(mapa_u32(&acc_empty[acc], 0));
        else mbar_arrive(&acc_empty[acc]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem_base, C::TMEM_COLS);
  }
}

// The parts of a reduction added up, eight columns a thread; rows of no group have their zeros.
__global__ void __launch_bounds__(256) ragged_parts_kernel(const int* __restrict__ head, const float* __restrict__ parts,
                                                           __nv_bfloat16* __restrict__ D, int rows, int M) {
  const int splits = head[0], lo = head[1], hi = head[2], pieces = M >> 3;
  if (splits < 2) return;
  const long long n = (long long)(hi - lo) * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const size_t at = size_t(lo) * M + i * 8;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int k = 0; k < splits; ++k) {
      const float4* q = reinterpret_cast<const float4*>(parts + size_t(k) * rows * M + at);
      const float4 u = __ldcg(q), v = __ldcg(q + 1);
      a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
      b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w;
    }
    *reinterpret_cast<uint4*>(D + at) = make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
  }
}

// -------------------------------------------------------------------------------------------------------------
// wgrad kernel: D_e [N, K] = dy^T x over the group's rows
// -------------------------------------------------------------------------------------------------------------
constexpr int EPI_BUF = 32 * 128;              // one store of an epilogue warp: 32 rows of 128 bytes
constexpr int EPI_BYTES = 4 * 2 * EPI_BUF;

template <int CG, int BN>
struct WgradCfg {
  static constexpr int X_COLS = BN / CG;       // columns of x per CTA
  static constexpr int X_BYTES = X_COLS * BK * 2;
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
  static constexpr int MAX_STAGES = 6;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int smem_bytes(int stages, int groups) {
    return stages * STAGE_BYTES + EPI_BYTES + BAR_BYTES + ((groups + 1) * 4 + 15) / 16 * 16 + 1024;
  }
  static int stages(int groups) {              // 6 for up to 400 groups (pairs)
    int n = MAX_STAGES;
    while (smem_bytes(n, groups) > SMEM_MAX) --n;
    return n;
  }
  static_assert(smem_bytes(4, MAX_GROUPS) <= SMEM_MAX && TMEM_COLS <= 512 && (4 * MAX_STAGES + 5) * 8 <= BAR_BYTES, "");
};

struct WgradParams {
  const int* offsets;
  int groups, rows;
  int N, K;                  // rows and columns of a group's result
  int dy_blocked, x_blocked; // operand through a 3-D map {64, rows, columns / 64}: one copy per stage
  int tiles_n, tiles_k, stages;
  int out_fp32, accumulate;
  int* status;
};

// A stage of the ring and its phase.  The barriers of blocks that end a group (`tail`) are used only there, so that their
// phases have a bit for each stage.
struct RingPos {
  int s = 0;
  uint32_t ph = 0, tail_ph = 0;
  __device__ __forceinline__ uint32_t tail() const { return (tail_ph >> s) & 1u; }
  __device__ __forceinline__ void next(int stages, bool tail) {
    if (tail) tail_ph ^= 1u << s;
    if (++s == stages) { s = 0; ph ^= 1; }
  }
};

template <int CG, int BN>
__global__ void __launch_bounds__(224, 1)
ragged_wgrad_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ CUtensorMap map_d, const __grid_constant__ WgradParams p) {
  using C = WgradCfg<CG, BN>;
  constexpr int STAGE_BYTES = C::STAGE_BYTES, MS = C::MAX_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + p.stages * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + EPI_BYTES);
  uint64_t* full = bars;                    // [stages] TMA -> MMA (pair: the leader's counts both CTAs' bytes)
  uint64_t* empty = bars + MS;              // [stages] MMA -> TMA
  uint64_t* tail_full = bars + 2 * MS;      // [stages] a block with masked rows: TMA -> this CTA's masking warp
  uint64_t* tail_ready = bars + 3 * MS;     // [stages] and the masking warps of both CTAs -> MMA (the leader's)
  uint64_t* acc_full = bars + 4 * MS;
  uint64_t* acc_empty = bars + 4 * MS + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * MS + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* off = reinterpret_cast<int*>(epi + EPI_BYTES + BAR_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? int(cluster_ctarank()) : 0;
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;
  const int per_group = p.tiles_n * p.tiles_k, num_tiles = per_group * p.groups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail_full[s], 1);
      mbar_init(&tail_ready[s], CG);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * CG);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_dy);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_d);
  }
  if (warp == 1) {
    tmem_alloc_cg<CG>(tmem_slot, C::TMEM_COLS);
    tmem_relinquish_cg<CG>();
  }
  if (warp == 2) make_bounds(p.offsets, p.groups, p.rows, off);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // tile -> group, block of result rows, block of result columns: rows of blocks 2048 columns wide, so that the tiles in
  // flight share their panels of dy and x in L2
  auto place = [&](int tile, int& e, int& nb, int& kb) {
    constexpr int WIDE = 2048 / BN;
    e = tile / per_group;
    const int i = tile - e * per_group, per = WIDE * p.tiles_n, g = i / per, in = i - g * per;
    const int w = min(WIDE, p.tiles_k - g * WIDE);
    nb = in / w;
    kb = g * WIDE + in - nb * w;
  };

  if (warp == 0) {
    // ------------------------------- TMA producer --------------------------------------------
    RingPos at;
    uint32_t armed = 0, armed_phase = 0, tail_armed = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      int e, nb, kb;
      place(tile, e, nb, kb);
      const int n0 = (nb * CG + rank) * 128, c0 = kb * BN + rank * C::X_COLS;
      const int end = off[e + 1];
      for (int r = off[e]; r < end; r += BK) {
        const int s = at.s;
        if (!mbar_wait_bounded_warp(&empty[s], at.ph ^ 1, abort_flag, p.status)) { ok = false; break; }
        const bool tail = (end - r) < BK && (end - r) % UMMA_K != 0;   // rows to be masked
        uint8_t* sa = smem + s * STAGE_BYTES;
        uint8_t* sb = sa + W_BYTES;
        armed |= 1u << s;
        armed_phase = (armed_phase & ~(1u << s)) | ((tail ? at.tail() : at.ph) << s);
        tail_armed = (tail_armed & ~(1u << s)) | (uint32_t(tail) << s);
        if (elect_one()) {
          // Blocks without masked rows report to the leader's `full`, which announces both CTAs' bytes.  The others report to
          // `tail_full` of their own CTA, and `full` takes a plain arrival, to keep its phase.
          if (tail) {
            mbar_expect_tx(&tail_full[s], STAGE_BYTES);
            if (CG == 1 || rank == 0) mbar_arrive(&full[s]);
          } else if (CG == 1 || rank == 0) {
            mbar_expect_tx(&full[s], STAGE_BYTES * CG);
          }
          const uint32_t bar = tail ? smem_u32(&tail_full[s]) : CG == 2 ? mapa_u32(&full[s], 0) : smem_u32(&full[s]);
          auto load2 = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
            if constexpr (CG == 2) tma_load_2d_pair(dst, map, bar, x, y);
            else tma_load_2d(dst, map, tail ? &tail_full[s] : &full[s], x, y);
          };
          auto load3 = [&](uint8_t* dst, const CUtensorMap* map, int y, int z) {
            if constexpr (CG == 2) tma_load_3d_pair(dst, map, bar, 0, y, z);
            else tma_load_3d(dst, map, tail ? &tail_full[s] : &full[s], 0, y, z);
          };
          if (p.dy_blocked) load3(sa, &map_dy, r, n0 >> 6);
          else {
            load2(sa, &map_dy, n0, r);
            load2(sa + 8192, &map_dy, n0 + 64, r);
          }
          if (p.x_blocked) load3(sb, &map_x, r, c0 >> 6);
          else {
#pragma unroll
            for (int j = 0; j < C::X_COLS / 64; ++j) load2(sb + j * 8192, &map_x, c0 + j * 64, r);
          }
        }
        __syncwarp();
        at.next(p.stages, tail);
      }
    }
    if (!ok) {
      // wait (bounded) for the copies in flight before the shared memory is released
      const uint64_t begin = globaltimer_ns();
      if (CG == 2 && rank != 0) {
        while (globaltimer_ns() - begin < 2000000) {   // most report to the leader's barriers: many times a copy's time
        }
      } else {
        for (int s = 0; s < p.stages; ++s) {
          if (!(armed & (1u << s))) continue;
          const uint32_t ph = (armed_phase >> s) & 1;
          uint64_t* bar = (tail_armed >> s) & 1 ? &tail_full[s] : &full[s];
          while (!mbar_try_wait(bar, ph) && globaltimer_ns() - begin < wait_budget_ns()) {
          }
        }
      }
    }
  } else if (warp == 6) {
    // ------------------------------- masking warp: one block per tile at most ---------------------
    RingPos at;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      const int e = tile / per_group, end = off[e + 1];
      for (int r = off[e]; r < end; r += BK) {
        const int live = end - r;
        const bool tail = live < BK && live % UMMA_K != 0;
        if (tail) {
          const int s = at.s;
          if (!mbar_wait_bounded_warp(&tail_full[s], at.tail(), abort_flag, p.status)) { ok = false; break; }
          // rows live .. of the last step of 16.  A token is a 128-byte row of each 64-column block; the swizzle moves pieces
          // within the row only
          constexpr int BLOCKS = STAGE_BYTES / 8192;
          uint8_t* at_row = smem + s * STAGE_BYTES + live * 128 + lane * 16;      // four rows a step
          for (int dead = UMMA_K - live % UMMA_K - (lane >> 3); dead > 0; dead -= 4, at_row += 512) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) *reinterpret_cast<uint4*>(at_row + b * 8192) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) mbar_arrive_cluster(mapa_u32(&tail_ready[s], 0));
            else mbar_arrive(&tail_ready[s]);
          }
        }
        at.next(p.stages, tail);
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (the leader's, in a pair) ------------------------
    if (CG == 1 || rank == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(128 * CG, BN, 1, 1);
      constexpr uint32_t STEP = 2048 >> 4;
      const SmemDesc a_desc = make_smem_desc2(smem_u32(smem), 8192, 1024);
      const SmemDesc b_desc = make_smem_desc2(smem_u32(smem) + W_BYTES, 8192, 1024);
      RingPos at;
      uint32_t tile_i = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
        const int e = tile / per_group, begin = off[e], end = off[e + 1];
        if (begin >= end) continue;
        const uint32_t acc = tile_i & 1, acc_ph = (tile_i >> 1) & 1;
        if (!mbar_wait_bounded_warp(&acc_empty[acc], acc_ph ^ 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        bool fresh = true;
        for (int r = begin; r < end; r += BK) {
          const int s = at.s;
          const bool tail = (end - r) < BK && (end - r) % UMMA_K != 0;
          if (!mbar_wait_bounded_warp(&full[s], at.ph, abort_flag, p.status)) { ok = false; break; }
          if (tail && !mbar_wait_bounded_warp(&tail_ready[s], at.tail(), abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t word = uint32_t(s * STAGE_BYTES) >> 4;
          if (elect_one()) {
            if (end - r > BK - UMMA_K) {       // (no test between the products of a whole block: they are issued one by one)
#pragma unroll
              for (int k = 0; k < BK / UMMA_K; ++k)
                umma_bf16_ss2_cg<CG>(d_tmem, a_desc.lo + word + k * STEP, a_desc.hi, b_desc.lo + word + k * STEP, b_desc.hi, idesc,
                                     !(fresh && k == 0));
            } else {
              for (int k = 0; r + k * UMMA_K < end; ++k)
                umma_bf16_ss2_cg<CG>(d_tmem, a_desc.lo + word + k * STEP, a_desc.hi, b_desc.lo + word + k * STEP, b_desc.hi, idesc,
                                     !(fresh && k == 0));
            }
            umma_commit_cg<CG>(&empty[s], 3);
          }
          fresh = false;
          __syncwarp();
          at.next(p.stages, tail);
        }
        if (ok && elect_one()) umma_commit_cg<CG>(&acc_full[acc], 3);
        __syncwarp();
        ++tile_i;
      }
    }
  } else {
    // ------------------------------- epilogue (warps 2..5) ------------------------------------------
    const int quarter = warp & 3;
    uint8_t* buf = epi + quarter * 2 * EPI_BUF;
    uint32_t tile_i = 0, stores = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      int e, nb, kb;
      place(tile, e, nb, kb);
      const bool none = off[e] >= off[e + 1];           // a group without rows: zeros, or nothing to add
      if (none && p.accumulate) continue;
      const uint32_t acc = tile_i & 1, acc_ph = (tile_i >> 1) & 1;
      if (!none) {
        if (!mbar_wait_bounded_warp(&acc_full[acc], acc_ph, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
      }
      const uint32_t t_acc = tmem_base + (uint32_t(quarter * 32) << 16) + acc * BN;
      const int row_w = (nb * CG + rank) * 128 + quarter * 32, c0 = kb * BN;
      // (a warp whose rows lie behind the last one stores nothing and leaves its buffers alone)
      const int c_end = row_w < p.N ? min(BN, p.K - c0) : 0;
      const int cols = p.out_fp32 ? 32 : 64;            // 128 bytes of a row per step
#pragma unroll 1
      for (int c = 0; c < c_end; c += cols) {
        uint32_t r[32];
        uint8_t* b = buf + (stores & 1) * EPI_BUF;
        if (lane == 0) bulk_wait_read<1>();             // the store before last has read this buffer
        __syncwarp();
        uint8_t* row = b + lane * 128;
        const int sw = lane & 7;                        // 128-byte swizzle: piece i of row r sits at i ^ (r & 7)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && p.out_fp32) break;
          if (none) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0;
          } else {
            tmem_ld_32x32(t_acc + c + h * 32, r);
            tc_wait_ld();
          }
          if (p.out_fp32) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(row + ((j ^ sw) << 4)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              auto two = [&](int i) { return pack_bf16(__uint_as_float(r[8 * j + i]), __uint_as_float(r[8 * j + i + 1])); };
              *reinterpret_cast<uint4*>(row + (((j + 4 * h) ^ sw) << 4)) = make_uint4(two(0), two(2), two(4), two(6));
            }
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          if (p.accumulate) tma_reduce_add_3d(&map_d, b, c0 + c, row_w, e);
          else tma_store_3d(&map_d, b, c0 + c, row_w, e);
          bulk_commit();
        }
        ++stores;
      }
      if (none) continue;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2 && rank != 0) mbar_arrive_cluster(mapa_u32(&acc_empty[acc], 0));
        else mbar_arrive(&acc_empty[acc]);
      }
      ++tile_i;
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem_base, C::TMEM_COLS);
  }
}

// -------------------------------------------------------------------------------------------------------------
// host side
// -------------------------------------------------------------------------------------------------------------
template <typename Kernel, typename... Args>
static int launch(SmemLimit& limit, Kernel kernel, int cg, int smem, int threads, long long tiles, cudaStream_t stream, const Args&... args) {
  if (const int rc = limit.allow(kernel, smem)) return rc;
  const int slots = sm_count_of_device() / cg;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(int(tiles < slots ? tiles : slots) * cg);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cg;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cg > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return launch_result(e);
}

template <int CG, int BT>
static int launch_rows(const void* w, const void* tokens, RowsParams& p, int w_mn, cudaStream_t stream) {
  using C = RowsCfg<CG, BT>;
  CUtensorMap mw, mt;
  const uint64_t M = p.M, K = p.K, E = p.groups;
  int rc;
  if (!w_mn) {             // W_e [M, K]
    const uint64_t dims[3] = {K, M, E}, strides[2] = {K * 2, M * K * 2};
    const uint32_t box[3] = {BK, 128, 1};
    rc = jpb_make_tensor_map(&mw, w, 2, 3, dims, strides, box, 1);
  } else if (p.w_blocked) {  // W_e [K, M]
    const uint64_t dims[4] = {64, K, M / 64, E}, strides[3] = {M * 2, 128, M * K * 2};
    const uint32_t box[4] = {64, BK, 2, 1};
    rc = jpb_make_tensor_map(&mw, w, 2, 4, dims, strides, box, 1);
  } else {
    const uint64_t dims[3] = {M, K, E}, strides[2] = {M * 2, M * K * 2};
    const uint32_t box[3] = {64, BK, 1};
    rc = jpb_make_tensor_map(&mw, w, 2, 3, dims, strides, box, 1);
  }
  if (rc) return rc;
  const uint64_t dims[2] = {K, uint64_t(p.rows)}, strides[1] = {K * 2};
  // (the token rows of a stage come in copies of 64; 16-row copies for the remainder made 14336 x 4096 dgrad 10 % slower)
  const uint32_t box[2] = {BK, uint32_t(C::BOX)};
  if ((rc = jpb_make_tensor_map(&mt, tokens, 2, 2, dims, strides, box, 1))) return rc;
  p.tiles_m = (p.M + 128 * CG - 1) / (128 * CG);
  const long long tiles = ((long long)(p.rows + BT - 1) / BT + p.groups) * (p.M / (96 * CG) + 1) * (p.parts ? SPLIT_MAX : 1);   // at most
  if (tiles > 0x7fffffffll) return -JPB_ERR_BAD_ARGUMENT;
  auto run = [&](auto mn, auto split) {
    static SmemLimit limit;
    return launch(limit, ragged_rows_kernel<CG, BT, decltype(mn)::value, decltype(split)::value>, CG, C::SMEM_BYTES, 192, tiles, stream, mw, mt, p);
  };
  if constexpr (CG == 1)
    if (p.parts) return w_mn ? run(std::true_type(), std::true_type()) : run(std::false_type(), std::true_type());
  return w_mn ? run(std::true_type(), std::false_type()) : run(std::false_type(), std::false_type());
}

static int columns_map(CUtensorMap* out, const void* t, uint64_t rows, uint64_t cols, uint32_t box_cols, int blocked) {
  if (blocked) {
    const uint64_t dims[3] = {64, rows, cols / 64}, strides[2] = {cols * 2, 128};
    const uint32_t box[3] = {64, BK, box_cols / 64};
    return jpb_make_tensor_map(out, t, 2, 3, dims, strides, box, 1);
  }
  const uint64_t dims[2] = {cols, rows}, strides[1] = {cols * 2};
  const uint32_t box[2] = {64, BK};
  return jpb_make_tensor_map(out, t, 2, 2, dims, strides, box, 1);
}

template <int CG, int BN>
static int launch_wgrad(const void* dy, const void* x, void* D, WgradParams& p, cudaStream_t stream) {
  using C = WgradCfg<CG, BN>;
  CUtensorMap ma, mb, md;
  int rc;
  if ((rc = columns_map(&ma, dy, p.rows, p.N, 128, p.dy_blocked))) return rc;
  if ((rc = columns_map(&mb, x, p.rows, p.K, C::X_COLS, p.x_blocked))) return rc;
  const uint64_t es = p.out_fp32 ? 4 : 2, N = p.N, K = p.K;
  const uint64_t dims[3] = {K, N, uint64_t(p.groups)}, strides[2] = {K * es, N * K * es};
  const uint32_t box[3] = {uint32_t(128 / es), 32, 1};
  if ((rc = jpb_make_tensor_map(&md, D, int(es), 3, dims, strides, box, 1))) return rc;
  p.tiles_n = (p.N + 128 * CG - 1) / (128 * CG);
  p.tiles_k = (p.K + BN - 1) / BN;
  const long long tiles = (long long)p.tiles_n * p.tiles_k * p.groups;
  if (tiles > 0x7fffffffll) return -JPB_ERR_BAD_ARGUMENT;
  p.stages = C::stages(p.groups);
  static SmemLimit limit;
  return launch(limit, ragged_wgrad_kernel<CG, BN>, CG, C::smem_bytes(p.stages, p.groups), 224, tiles, stream, ma, mb, md, p);
}

// Which blocks of token rows (the host knows the mean of the groups' rows, not the rows).  Measured with ragged groups, us, as 1 x 32
// rows / 1 x 128 / a pair's 256, L2 flushed:
//   8 x 14336 x 4096    mean 1: 115 / 141 / 115    24: 170 / 180 / 182    32: 195 / 182 / 182    96: - / 186 / 186   128: - / 209 / 190
//   64 x 1408 x 2048    mean 1: 55 / 55 / 61       24: 86 / 82 / 86       48: 100 / 82 / 88      96: - / 88 / 90     192: - / 115 / 94
// Small products are short of tiles, or of steps in a tile to hide its start and its store behind:
//   8 x 2048 x 512      mean 250: - / 18 / 20      512 (8.6 GFLOP): - / 23 / 27      1024 (17 GFLOP): - / 35 / 33
//   8 x 1024 x 4096     mean 128 (8.6 GFLOP): - / 33 / 35    192 (13 GFLOP): - / 33 / 37    250 (17 GFLOP): - / 49 / 39
static int block_rows(int rows, int groups, int M, int K, int sms) {
  const int mean = (rows + groups - 1) / groups;
  if (mean <= 24) return 32;
  const long long pairs = ((long long)rows / 256 + groups) * ((M + 255) / 256);
  const bool small = pairs < sms / 4 || 2.0 * rows * M * K < 14e9;
  return mean <= 96 || small ? 128 : 256;
}
// Parts that the reduction of a single CTA's tiles may have: none where the tiles may be more than half the SMs, or for reductions
// of less than 2048, where their sum costs more than they save.  One token of two experts, us, whole / in parts: 4096 x 14336 59 / 45,
// 4096 x 4096 21 / 16, 2048 x 8192 36 / 17, 1024 x 2048 13.1 / 10.4, 4096 x 2048 12.9 / 11.9, 4096 x 1024 9.4 / 10.9;
// 300 rows of four, 256 x 4096, 22 / 14; 400 rows of eight, 512 x 4096, 21 / 14.5.
static int most_parts(int rows, int groups, int M, int K, int slots) {
  const int block = block_rows(rows, groups, M, K, slots);
  const long long tiles_m = (M + 127) / 128, blocks = rows / block + (rows < groups ? rows : groups);
  if (block == 256 || K < 2048 || 2 * blocks * tiles_m > slots) return 1;
  const long long most = slots / tiles_m;
  return int(most < SPLIT_MAX ? most : SPLIT_MAX);
}
// Tiles of 128 x 128 where pairs' 256 x 256 would leave most SMs without one, and for short groups, whose time is that of the
// stores.  Measured, us, single / pairs: 8 x 512 x 512 (32 pairs) 8.2 / 10.2 with 16 rows a group, 16.4 / 18.4 with 1024, 32.8 / 36.9
// with 4096; 4 x 1024 x 1024 (64 pairs) 20.5 / 18.4 with 1024, 53.2 / 34.8 with 4096; 64 x 2896 x 1864 194 / 304 with 4; 64 x 1408 x
// 2048 102 / 108 with 16, 103 / 115 with 128, 156 / 145 with 256.
static int wgrad_tile(int rows, int groups, int N, int K, int sms) {
  const long long pairs = (long long)groups * ((N + 255) / 256) * ((K + 255) / 256);
  return pairs < sms / 3 || (rows + groups - 1) / groups <= 128 ? 128 : 256;
}
static bool bad(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace ragged
}  // namespace jpb

// y [rows, N] = x [rows, K] * w[e]^T (w [groups, N, K]; transposed = 0) or dx [rows, K] = dy [rows, N] * w[e] (transposed = 1),
// row t in group e where offsets[e] <= t < offsets[e + 1] (int32 on the device); rows of no group give zeros.  bf16,
// contiguous, on 16-byte boundaries, N and K multiples of 8.
// scratch: as many fp32 elements as jpb_linear_ragged_scratch_elems says (none: null), on a 16-byte boundary.
JPB_API int jpb_linear_ragged(const void* tokens, const void* w, const int* offsets, void* out, int rows, int groups, int N, int K,
                              int transposed, float* scratch, void* stream) {
  using namespace jpb;
  using namespace jpb::ragged;
  if (rows < 0 || rows > MAX_ROWS || groups < 1 || groups > MAX_GROUPS || N <= 0 || K <= 0 || (N & 7) || (K & 7) || bad(tokens) || bad(w) || bad(out))
    return -JPB_ERR_BAD_ARGUMENT;
  if (rows == 0) return 0;
  RowsParams p = {};
  p.offsets = offsets; p.groups = groups; p.rows = rows; p.M = transposed ? K : N; p.K = transposed ? N : K;
  p.w_blocked = transposed && p.M % 64 == 0; p.D = static_cast<__nv_bfloat16*>(out); p.status = jpb_status_device_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count_of_device(), parts = most_parts(rows, groups, p.M, p.K, sms);
  if (parts > 1) {
    if (!scratch || bad(scratch)) return -JPB_ERR_BAD_ARGUMENT;
    p.head = reinterpret_cast<int*>(scratch);
    p.parts = scratch + 4;
  }
  const int block = block_rows(rows, groups, p.M, p.K, sms);
  const int rc = block == 32    ? launch_rows<1, 32>(w, tokens, p, transposed, s)
                 : block == 128 ? launch_rows<1, 128>(w, tokens, p, transposed, s)
                                : launch_rows<2, 256>(w, tokens, p, transposed, s);
  if (rc || parts < 2) return rc;
  const long long pieces = (long long)rows * (p.M >> 3);
  ragged_parts_kernel<<<int((pieces + 255) / 256), 256, 0, s>>>(p.head, p.parts, p.D, rows, p.M);
  return launch_result(cudaSuccess);
}

JPB_API long long jpb_linear_ragged_scratch_elems(int rows, int groups, int N, int K, int transposed) {
  if (rows <= 0 || groups <= 0) return 0;
  const int M = transposed ? K : N, parts = jpb::ragged::most_parts(rows, groups, M, transposed ? N : K, jpb::sm_count_of_device());
  return parts > 1 ? 4 + (long long)parts * rows * M : 0;
}

// dw [groups, N, K] (fp32 or bf16), written or (fp32 only) added to = sum over each group's rows of dy [rows, N]^T x [rows, K].
// A group without rows gives zeros.  Otherwise as above.
JPB_API int jpb_linear_ragged_wgrad(const void* dy, const void* x, const int* offsets, void* dw, int rows, int groups, int N, int K,
                                    int out_fp32, int accumulate, void* stream) {
  using namespace jpb;
  using namespace jpb::ragged;
  if (rows < 0 || rows > MAX_ROWS || groups < 1 || groups > MAX_GROUPS || N <= 0 || K <= 0 || (N & 7) || (K & 7) || bad(dy) || bad(x) || bad(dw) ||
      (accumulate && !out_fp32))
    return -JPB_ERR_BAD_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) return accumulate ? 0 : int(cudaMemsetAsync(dw, 0, size_t(groups) * N * K * (out_fp32 ? 4 : 2), s));
  WgradParams p = {};
  p.offsets = offsets; p.groups = groups; p.rows = rows; p.N = N; p.K = K; p.dy_blocked = N % 64 == 0; p.x_blocked = K % 64 == 0;
  p.out_fp32 = out_fp32; p.accumulate = accumulate; p.status = jpb_status_device_ptr();
  if (wgrad_tile(rows, groups, N, K, sm_count_of_device()) == 128) return launch_wgrad<1, 128>(dy, x, dw, p, s);
  return launch_wgrad<2, 256>(dy, x, dw, p, s);
}

// What a product of these sizes runs as on a device of `sms` SMs (for tests; rows and groups above zero): rows of the token operand in
// a block (32 and 128 of single CTAs, 256 of a pair), plus 1024 times the most parts that a reduction may have; and the edge of the
// weight gradient's tiles (128 single CTAs, 256 pairs).
JPB_API int jpb_linear_ragged_form(int rows, int groups, int N, int K, int transposed, int sms) {
  using namespace jpb::ragged;
  const int M = transposed ? K : N, R = transposed ? N : K;
  return block_rows(rows, groups, M, R, sms) + 1024 * most_parts(rows, groups, M, R, sms);
}
JPB_API int jpb_linear_ragged_wgrad_form(int rows, int groups, int N, int K, int sms) { return jpb::ragged::wgrad_tile(rows, groups, N, K, sms); }
