// The residual connection of a block whose output is normalised as well as its input, forward and backward:
//   p = y * rstd1,  n = p * w_post            (w_post absent: p = n = y)
//   r = scale * x + gate * n                  (gate absent: 1)
//   h = r * rstd2 * w_pre                     (w_pre absent: no h)
// with rstd = 1 / sqrt(mean of the squares + eps) of y and of r.  Gradients, for those of r and h (dr, dh; either may be
// absent), with u = dh * w_pre, hat = r * rstd2, v = gate * dR * w_post:
//   dR = dr + rstd2 * (u - hat * mean(u * hat))      dx = scale * dR       dw_pre  = sum over rows of dh * hat
//   dy = rstd1 * (v - p * mean(v * p))               dgate = sum of dR * n        dw_post = sum over rows of gate * dR * p
// All arithmetic is fp32; r is kept unrounded between the two norms, and the backward computes it again from x and y, so that
// its gradients are those of the forward's function and not of the rounded stream.
//
// What bounds it: HBM, four rows moved per row forward (x, y, r, h) and six backward (dr, dh, x, y, dx, dy).  8192 x 4096 bf16 forward
// takes 51 us (5.3 TB/s), a launch and the first row's way through included, which are 5 of them.  Backward of 8192 x 8192 with a gate
// for each of four sequences 153 us (5.3 TB/s), of 4096 rows 88: 78 and 7 for the sums of the partial rows (the copies without
// arithmetic take 67): every operand is widened from bf16 twice, for the sums and for the results, since there is no room in the
// registers for a row and the three running sums of its columns.
#include "launch.cuh"
#include "vec.cuh"

#include <initializer_list>
#include <type_traits>

namespace jpb {

struct ResNormParams {
  const void *x, *y, *w_post, *gate, *w_pre;
  void *r, *h;
  float *rstd_post, *rstd_pre;
  const void *dr, *dh;
  void *dx, *dy;
  float* scratch;
  long long rows;
  int d, stages;
  long long group_rows;   // rows of x for each row of the gate
  int groups, chunks;     // backward: every group's rows are cut into `chunks` parts, a CTA each (or a CTA has whole groups)
  int stream_gate;        // the gate's row comes with every row of x, else it is loaded when it changes
  void* dgate;            // written by the main kernel where chunks == 1
  int wide;
  float scale, eps;
  int* status;
};

constexpr int RN_THREADS = 512;     // threads of an SM: as many rows at a time as there are CTAs of them
constexpr int RN_MAX_STAGES = 4;
constexpr int RN_HEAD = 512;        // shared memory in front of the ring: barriers, sums of a CTA

// Rows stream through a ring in shared memory, copied whole by the bulk-copy unit (one thread asks for them): what is in
// flight does not depend on registers or on how many threads wait for a sum.  A stage holds one row of each operand that there
// is, in the order y, x, dh, dr, gate.
struct RowRing {
  uint64_t* full;
  uint8_t* ring;
  uint32_t row_bytes, stage_bytes;
  const void *y, *x, *dh, *dr, *gate;
  long long group_rows;
  volatile int* abort_flag;
  int* status;

  __device__ __forceinline__ int operands() const { return int(stage_bytes / row_bytes); }
  // The k-th operand's row on its way to stage s (one thread; the barrier counts the operands).  The operands of a stage are
  // asked for by different warps: asking takes 100 cycles each.
  __device__ __forceinline__ void ask(int k, int s, long long row) const {
    const void* src = k == 0 ? y : gate;
    if (gate == nullptr || k + 1 < operands()) {
      if (k == 1) src = x ? x : dr;
      else if (k == 2) src = dh ? dh : dr;
      else if (k == 3) src = dr;
    }
    if (gate != nullptr && k + 1 == operands()) row /= group_rows;
    mbar_expect_tx(&full[s], row_bytes);
    bulk_load(ring + size_t(s) * stage_bytes + k * row_bytes, static_cast<const uint8_t*>(src) + size_t(row) * row_bytes, row_bytes, &full[s]);
  }
  __device__ __forceinline__ void ask_all(int s, long long row) const {   // every thread of the CTA
    const int nwarps = blockDim.x >> 5, n = operands();
    for (int k = threadIdx.x >> 5; k < n; k += nwarps)
      if ((threadIdx.x & 31) == 0) ask(k, s, row);
  }
  // (a time-out is reported and the kernel goes on, over rows that nothing will use)
  __device__ __forceinline__ void wait(int s, uint32_t phase) const { mbar_wait_bounded(&full[s], phase, abort_flag, status); }
};

template <typename T>
__device__ __forceinline__ Vec<T> ones() {
  Vec<T> v;
  float f[Vec<T>::N];
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) f[j] = 1.f;
  v.from_float(f);
  return v;
}

// Sums over a CTA with one barrier.  Shuffles are what a sum costs (an SM does one a cycle, for all its warps): lanes trade values
// so that each ends up with one of the sums, and after the barrier a lane picks up one warp's part and as many steps follow as
// there are warps, not as there are lanes; `span` is the number of warps rounded up to a power of two, the parts behind it are
// zeros.  `slot` alternates between two halves of the scratch.
// Two sums (parts as [warp][2]):
__device__ __forceinline__ void cta_sum2(float& a, float& b, float* scratch, int& slot, int span) {
  float* s = scratch + slot * 32;
  slot ^= 1;
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1;
  float x = odd ? b : a;
  x += __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
#pragma unroll
  for (int o = 2; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (lane < 2) s[(threadIdx.x >> 5) * 2 + lane] = x;
  __syncthreads();
  x = s[lane & (2 * span - 1)];
  for (int o = 2; o < 2 * span; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  const float other = __shfl_xor_sync(0xffffffffu, x, 1);
  a = odd ? other : x;
  b = odd ? x : other;
}
// Four (parts as [warp][4]), in two halves with the caller's barrier between them:
__device__ __forceinline__ void sum4_begin(const float (&v)[4], float* s) {
  const int lane = threadIdx.x & 31;
  const bool b0 = lane & 1, b1 = lane & 2;
  float a = b0 ? v[2] : v[0], c = b0 ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, b0 ? v[0] : v[2], 1);
  c += __shfl_xor_sync(0xffffffffu, b0 ? v[1] : v[3], 1);
  float x = b1 ? c : a;
  x += __shfl_xor_sync(0xffffffffu, b1 ? a : c, 2);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  // lane & 3 = 0, 1, 2, 3 has the sums of v[0], v[2], v[1], v[3]
  if (lane < 4) s[(threadIdx.x >> 5) * 4 + lane] = x;
}
__device__ __forceinline__ void sum4_end(float (&v)[4], const float* s, int span) {
  const int lane = threadIdx.x & 31;
  float x = 0.f;
  for (int i = lane; i < span * 4; i += 32) x += s[i];
  for (int o = 4; o < 32 && o < span * 4; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  v[0] = __shfl_sync(0xffffffffu, x, 0);
  v[2] = __shfl_sync(0xffffffffu, x, 1);
  v[1] = __shfl_sync(0xffffffffu, x, 2);
  v[3] = __shfl_sync(0xffffffffu, x, 3);
}
__device__ __forceinline__ int warps_span() {
  int n = 1;
  while (n * 32 < int(blockDim.x)) n <<= 1;
  return n;
}

// gate * w_post, either of which may be null, at this thread's places.
template <typename T, int VECS, bool EXACT>
__device__ __forceinline__ void gate_weights(F2 (&gw)[VECS][Vec<T>::N / 2], const void* w_post, const T* gate, int nvec) {
  constexpr int VN = Vec<T>::N, NP = VN / 2;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (!EXACT && v >= nvec) continue;
    Vec<T> w = ones<T>(), g = ones<T>();
    if (w_post) w.load(static_cast<const T*>(w_post) + size_t(v) * VN);
    if (gate) g.load(gate + size_t(v) * VN);
    F2 f[NP];
    to_pairs(w, f);
    to_pairs(g, gw[i]);
#pragma unroll
    for (int j = 0; j < NP; ++j) gw[i][j] = gw[i][j] * f[j];
  }
}

// KIND and EXACT, of both kernels: which norms there are (and then the gate does not come through the ring, and the backward has dr
// and, with the second norm, dh), and whether rows are VECS pieces for every thread, so that the loop does not ask.  A third of the
// backward's instructions were such tests and the moves around them: 4096 x 8192 88 us instead of 108, 16384 x 1024 55 instead of 69,
// 15804 x 744 (not exact) 50 instead of 66; forward of 4096 x 4096 26 instead of 29; without the second norm, 8192 x 4096, 38 and 59 us
// instead of 46 and 87; without the first, 75 backward instead of 105.
enum RnKind { RN_ANY, RN_BOTH, RN_POST, RN_PRE };
template <typename T, int VECS, int KIND, bool EXACT>
__global__ void __launch_bounds__(RN_THREADS, 1) residual_norm_fwd_kernel(const __grid_constant__ ResNormParams p) {
  constexpr int VN = Vec<T>::N, NP = VN / 2;
  constexpr bool KNOWN = KIND != RN_ANY;
  const bool post = KNOWN ? KIND != RN_PRE : p.w_post != nullptr;
  const bool pre = KNOWN ? KIND != RN_POST : p.w_pre != nullptr;
  const bool stream_gate = !KNOWN && p.stream_gate;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int abort_flag;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  float* scratch = reinterpret_cast<float*>(smem + 128);    // [2][32]
  const int tid = threadIdx.x, nvec = p.d / VN, span = warps_span();
  for (int i = tid; i < 64; i += blockDim.x) scratch[i] = 0.f;
  const long long lo = p.rows * blockIdx.x / gridDim.x, hi = p.rows * (blockIdx.x + 1) / gridDim.x;
  const uint32_t row_bytes = uint32_t(p.d) * sizeof(T);
  const RowRing ring = {full, smem + RN_HEAD, row_bytes, row_bytes * (stream_gate ? 3 : 2), p.y, p.x, nullptr, nullptr,
                        stream_gate ? p.gate : nullptr, p.group_rows, &abort_flag, p.status};
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], ring.operands());
    fence_barrier_init();
  }
  __syncthreads();
  for (int s = 0; s < p.stages && lo + s < hi; ++s) ring.ask_all(s, lo + s);
  // (while the first rows come)
  Vec<T> w_pre[VECS];
  F2 gw[VECS][NP];      // gate * w_post
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = tid + i * blockDim.x;
    w_pre[i] = ones<T>();
    if (pre && (EXACT || v < nvec)) w_pre[i].load(static_cast<const T*>(p.w_pre) + size_t(v) * VN);
  }
  const T* const gate = static_cast<const T*>(p.gate);
  const bool now_and_then = p.gate && !stream_gate;
  long long gate_end = hi;             // row from which on another row of the gate counts
  if (now_and_then) gate_end = (lo / p.group_rows + 1) * p.group_rows;
  else if (p.gate) gate_end = lo;
  if (!stream_gate && lo < hi) gate_weights<T, VECS, EXACT>(gw, p.w_post, now_and_then ? gate + size_t(lo / p.group_rows) * p.d : nullptr, nvec);
  const uint32_t ring0 = smem_u32(ring.ring) + tid * 16, step = blockDim.x * 16;
  const float inv_d = 1.f / p.d;
  const F2 scale = f2(p.scale);
  // this thread's part of the sum of y^2 over the row in stage s
  auto squares = [&](int s) {
    F2 sum = f2(0.f);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      if (!EXACT && tid + i * blockDim.x >= nvec) continue;
      Vec<T> raw;
      F2 y[NP];
      lds_vec(raw, ring0 + s * ring.stage_bytes + i * step);
      to_pairs(raw, y);
#pragma unroll
      for (int j = 0; j < NP; ++j) sum = fma2(y[j], y[j], sum);
    }
    return sum.lo() + sum.hi();
  };
  int slot = 0, s = 0, s_next = 1;
  uint32_t phase = 0;                                // of the stage of row + 1
  float rstd1 = 1.f;
  auto post_stat = [&](float sum, long long row) {
    if (!post) return;
    rstd1 = rsqrtf(sum * inv_d + p.eps);
    if (tid == 0) p.rstd_post[row] = rstd1;
  };
  if (lo < hi) {
    ring.wait(0, 0);
    float sum = squares(0), none = 0.f;
    cta_sum2(none, sum, scratch, slot, span);
    post_stat(sum, lo);
  }
  // One barrier a row: the second norm's sum goes with the first norm's of the next row.
  for (long long row = lo; row < hi; ++row) {
    const uint32_t sy = ring0 + s * ring.stage_bytes, sx = sy + row_bytes;
    if (row == gate_end) {
      const long long g = row / p.group_rows;
      gate_end = (g + 1) * p.group_rows;
      gate_weights<T, VECS, EXACT>(gw, p.w_post, stream_gate ? reinterpret_cast<const T*>(ring.ring + size_t(s) * ring.stage_bytes + 2 * row_bytes)
                                                        : gate + size_t(g) * p.d, nvec);
    }
    F2 r[VECS][NP], squares_r = f2(0.f);
    const F2 r1 = f2(rstd1);
    T* const out_r = static_cast<T*>(p.r) + size_t(row) * p.d + size_t(tid) * VN;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      if (!EXACT && tid + i * blockDim.x >= nvec) continue;
      Vec<T> raw;
      F2 y[NP];
      lds_vec(raw, sy + i * step);
      to_pairs(raw, y);
      lds_vec(raw, sx + i * step);
      to_pairs(raw, r[i]);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        r[i][j] = fma2(r1, y[j] * gw[i][j], scale * r[i][j]);
        if (pre) squares_r = fma2(r[i][j], r[i][j], squares_r);
      }
      from_pairs(raw, r[i]);
      raw.store(out_r + i * step / int(sizeof(T)));
    }
    const bool more = row + 1 < hi;
    float sum = squares_r.lo() + squares_r.hi(), sum_next = 0.f;
    if (more) {
      ring.wait(s_next, phase);
      if (post) sum_next = squares(s_next);
    }
    cta_sum2(sum, sum_next, scratch, slot, span);
    // every thread is done with the row's stage: it takes another row
    if (row + p.stages < hi) ring.ask_all(s, row + p.stages);
    if (more) post_stat(sum_next, row + 1);
    if (pre) {
      const float rstd2 = rsqrtf(sum * inv_d + p.eps);
      if (tid == 0) p.rstd_pre[row] = rstd2;
      const F2 r2 = f2(rstd2);
      T* const out_h = static_cast<T*>(p.h) + size_t(row) * p.d + size_t(tid) * VN;
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        if (!EXACT && tid + i * blockDim.x >= nvec) continue;
        F2 w[NP];
        to_pairs(w_pre[i], w);
#pragma unroll
        for (int j = 0; j < NP; ++j) w[j] = w[j] * (r[i][j] * r2);
        Vec<T> raw;
        from_pairs(raw, w);
        raw.store(out_h + i * step / int(sizeof(T)));
      }
    }
    s = s_next;
    if (++s_next >= p.stages) { s_next = 0; phase ^= 1; }
  }
  if (abort_flag) {     // copies may still be in flight: many times their time
    const uint64_t begin = globaltimer_ns();
    while (globaltimer_ns() - begin < 2000000) {
    }
  }
}

// Backward.  With c = gate * w_post * y (so that r = scale * x + rstd1 * c) the two means need one round of sums, and one
// barrier, over the row:
//   dR = A - k1 * r  with  A = dr + rstd2 * u,  k1 = rstd2^2 * sum(rstd2 * u * r) / d
//   mean(v * p) = rstd1 * (sum(c A) - k1 * sum(c r)) / d
// and the sums over the rows of dR * p alone, S, give both dgate = w_post * S and dw_post = gate * S.  A CTA has consecutive
// rows: a part of one group of rows that share a gate row, or whole groups.  The sums for the gate leave at the end of a group
// (as the result, where the CTA has all of it), those for the weights when the CTA is done.
// (Two rounds of sums and scalar arithmetic took three times as long; with the operands kept in registers from the sums on, their
// spills made it 161 us for 4096 x 8192.)
template <typename T, int VECS, int KIND, bool EXACT>
__global__ void __launch_bounds__(RN_THREADS, 1) residual_norm_bwd_kernel(const __grid_constant__ ResNormParams p) {
  constexpr int VN = Vec<T>::N, NP = VN / 2;
  constexpr bool KNOWN = KIND != RN_ANY;
  const bool post = KNOWN ? KIND != RN_PRE : p.w_post != nullptr;
  const bool stream_gate = !KNOWN && p.stream_gate;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int abort_flag;
  __shared__ __align__(16) float scratch[2 * 32 * 4];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  const int tid = threadIdx.x, nvec = p.d / VN, span = warps_span();
  for (int i = tid; i < 2 * 32 * 4; i += blockDim.x) scratch[i] = 0.f;
  const bool pre = KNOWN ? KIND != RN_POST : p.w_pre && p.dh, has_dr = KNOWN || p.dr;
  float* part_post = p.scratch + size_t(blockIdx.x) * p.d;
  float* part_pre = p.scratch + size_t(gridDim.x + blockIdx.x) * p.d;
  float* part_gate = p.scratch + size_t(2 * gridDim.x + blockIdx.x) * p.d;
  long long lo, hi;
  if (p.chunks > 1) {
    const long long g = blockIdx.x / p.chunks, c = blockIdx.x - g * p.chunks;
    lo = g * p.group_rows + p.group_rows * c / p.chunks;
    hi = g * p.group_rows + p.group_rows * (c + 1) / p.chunks;
  } else {
    lo = (long long)p.groups * blockIdx.x / gridDim.x * p.group_rows;
    hi = (long long)p.groups * (blockIdx.x + 1) / gridDim.x * p.group_rows;
  }
  const uint32_t row_bytes = uint32_t(p.d) * sizeof(T);
  const int operands = KNOWN ? (pre ? 4 : 2) : 1 + 2 * pre + has_dr + stream_gate;
  const RowRing ring = {full, smem + RN_HEAD, row_bytes, row_bytes * operands, p.y, pre ? p.x : nullptr, pre ? p.dh : nullptr, p.dr,
                        stream_gate ? p.gate : nullptr, p.group_rows, &abort_flag, p.status};
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], ring.operands());
    fence_barrier_init();
  }
  __syncthreads();
  for (int s = 0; s < p.stages && lo + s < hi; ++s) ring.ask_all(s, lo + s);
  const F2 zero = f2(0.f);
  Vec<T> w_pre[VECS];
  F2 gw[VECS][NP], S[VECS][NP], a_pre[VECS][NP];    // gate * w_post; sums of dR * p (of the group) and dh * hat
  auto load_gate = [&](const T* gate) { gate_weights<T, VECS, EXACT>(gw, p.w_post, gate, nvec); };   // gate: this row's, or null
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = tid + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < NP; ++j) S[i][j] = a_pre[i][j] = gw[i][j] = zero;
    w_pre[i] = ones<T>();
    if (pre && (EXACT || v < nvec)) w_pre[i].load(static_cast<const T*>(p.w_pre) + size_t(v) * VN);
  }
  long long group = lo < hi ? lo / p.group_rows : 0;
  bool first_group = true;
  // end of a group: S goes to dgate (or its partial sum) and, times the gate, to the partial sum of dw_post
  auto flush = [&](const T* gate) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = tid + i * blockDim.x;
      if (!EXACT && v >= nvec) continue;
      Vec<T> w = ones<T>(), g = ones<T>();
      if (p.w_post) w.load(static_cast<const T*>(p.w_post) + size_t(v) * VN);
      if (gate) g.load(gate + size_t(v) * VN);
      F2 f[NP], o[NP];
      if (gate) {
        to_pairs(w, f);
#pragma unroll
        for (int j = 0; j < NP; ++j) o[j] = f[j] * S[i][j];
        if (p.chunks == 1 && !p.wide) {
          from_pairs(w, o);
          w.store(static_cast<T*>(p.dgate) + size_t(group) * p.d + size_t(v) * VN);
        } else {
          float2* to = reinterpret_cast<float2*>(p.chunks > 1 ? part_gate : static_cast<float*>(p.dgate) + size_t(group) * p.d) + v * NP;
#pragma unroll
          for (int j = 0; j < NP; ++j) to[j] = make_float2(o[j].lo(), o[j].hi());
        }
      }
      if (p.w_post) {
        float2* to = reinterpret_cast<float2*>(part_post) + v * NP;
        to_pairs(g, f);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          F2 sum = f[j] * S[i][j];
          if (!first_group) { const float2 old = to[j]; sum = sum + f2(old.x, old.y); }
          to[j] = make_float2(sum.lo(), sum.hi());
        }
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) S[i][j] = zero;
    }
    first_group = false;
  };
  // A row's sums are finished while the next row's are made: one barrier per row, between the sums of row + 1 and the results of
  // row + 1, with the results of row in front of it.  (At the end of a group the next row waits for its gate.)
  const float inv_d = 1.f / p.d;
  const F2 scale = f2(p.scale);
  struct Stats {
    float rstd1, rstd2;
  };
  auto stats_of = [&](long long row) {
    Stats t = {1.f, 0.f};
    if (row < hi) {
      if (post) t.rstd1 = p.rstd_post[row];
      if (pre) t.rstd2 = p.rstd_pre[row];
    }
    return t;
  };
  // shared-memory address of this thread's first piece of operand k in stage s; the next ones are `step` bytes further
  const uint32_t ring0 = smem_u32(ring.ring) + tid * 16, step = blockDim.x * 16;
  auto operand = [&](int s, int k) { return ring0 + s * ring.stage_bytes + k * row_bytes; };
  const int at_dr = pre ? 3 : 1, at_gate = operands - 1;
  int slot = 0;
  // this thread's part of sum(u r), sum(c A), sum(c r) with A = dr + rstd2 * u; adds to the sum for w_pre
  auto row_sums = [&](int s, const Stats& t) {
    const uint32_t sy = operand(s, 0), sx = operand(s, 1), sdh = operand(s, 2), sdr = operand(s, at_dr);
    const F2 r1 = f2(t.rstd1), r2 = f2(t.rstd2);
    F2 ur = zero, ca = zero, cr = zero;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = tid + i * blockDim.x;
      if (!EXACT && v >= nvec) continue;
      Vec<T> raw;
      F2 c[NP], A[NP];
      lds_vec(raw, sy + i * step);
      to_pairs(raw, c);
#pragma unroll
      for (int j = 0; j < NP; ++j) c[j] = c[j] * gw[i][j];
      if (has_dr) {
        lds_vec(raw, sdr + i * step);
        to_pairs(raw, A);
      } else {
#pragma unroll
        for (int j = 0; j < NP; ++j) A[j] = zero;
      }
      if (pre) {
        F2 x[NP], u[NP], w[NP];
        lds_vec(raw, sx + i * step);
        to_pairs(raw, x);
        lds_vec(raw, sdh + i * step);
        to_pairs(raw, u);
        to_pairs(w_pre[i], w);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const F2 r = fma2(r1, c[j], scale * x[j]);
          u[j] = u[j] * r2;
          a_pre[i][j] = fma2(u[j], r, a_pre[i][j]);
          u[j] = u[j] * w[j];
          A[j] = A[j] + u[j];
          ur = fma2(u[j], r, ur);
          if (post) cr = fma2(c[j], r, cr);
        }
      }
#pragma unroll
      for (int j = 0; j < NP; ++j)
        if (post) ca = fma2(c[j], A[j], ca);
    }
    float sums[4] = {ur.lo() + ur.hi(), ca.lo() + ca.hi(), cr.lo() + cr.hi(), 0.f};
    sum4_begin(sums, scratch + slot * 128);
  };
  // dx and dy of a row from its sums
  auto row_results = [&](int s, long long row, const Stats& t, const float (&sums)[4]) {
    const uint32_t sy = operand(s, 0), sx = operand(s, 1), sdh = operand(s, 2), sdr = operand(s, at_dr);
    // dR = A - k1 * r = dr + rstd2 * u - k1 * rstd1 * c - k1 * scale * x;   dy = rstd1 * gate * w_post * dR - k2 * y
    const float k1 = t.rstd2 * t.rstd2 * sums[0] * inv_d;
    // (the sums are of the size of y: one factor at a time keeps the products within fp32 wherever the mean of y^2 is)
    const float k2 = post ? t.rstd1 * (t.rstd1 * (t.rstd1 * ((sums[1] - k1 * sums[2]) * inv_d))) : 0.f;
    const F2 r1 = f2(t.rstd1), r2 = f2(t.rstd2), mc = f2(-k1 * t.rstd1), mx = f2(-k1 * p.scale), my = f2(-k2);
    T* const dx = static_cast<T*>(p.dx) + size_t(row) * p.d + size_t(tid) * VN;
    T* const dy = static_cast<T*>(p.dy) + size_t(row) * p.d + size_t(tid) * VN;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = tid + i * blockDim.x;
      if (!EXACT && v >= nvec) continue;
      Vec<T> raw;
      F2 y[NP], dR[NP], o[NP];
      lds_vec(raw, sy + i * step);
      to_pairs(raw, y);
      if (has_dr) {
        lds_vec(raw, sdr + i * step);
        to_pairs(raw, dR);
      } else {
#pragma unroll
        for (int j = 0; j < NP; ++j) dR[j] = zero;
      }
      if (pre) {
        F2 x[NP], u[NP], w[NP];
        lds_vec(raw, sx + i * step);
        to_pairs(raw, x);
        lds_vec(raw, sdh + i * step);
        to_pairs(raw, u);
        to_pairs(w_pre[i], w);
#pragma unroll
        for (int j = 0; j < NP; ++j)
          dR[j] = fma2(mx, x[j], fma2(mc, y[j] * gw[i][j], fma2(r2, u[j] * w[j], dR[j])));
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const F2 dRp = dR[j] * r1;
        o[j] = scale * dR[j];
        S[i][j] = fma2(dRp, y[j], S[i][j]);
        y[j] = fma2(dRp, gw[i][j], my * y[j]);
      }
      from_pairs(raw, o);
      raw.store(dx + i * step / int(sizeof(T)));
      from_pairs(raw, y);
      raw.store(dy + i * step / int(sizeof(T)));
    }
  };
  auto gate_of = [&](int s) {
    return stream_gate ? reinterpret_cast<const T*>(ring.ring + size_t(s) * ring.stage_bytes + at_gate * row_bytes)
                         : static_cast<const T*>(p.gate) + size_t(group) * p.d;
  };
  int s = 0;
  uint32_t phase = 0;             // of the stage of row + 1
  long long left = p.gate ? p.group_rows : 0;        // rows of the current group from row on (a part of a group ends with the CTA's rows)
  Stats now = stats_of(lo), next = stats_of(lo + 1);
  if (lo < hi) {
    if (!p.gate) load_gate(nullptr);
    else if (!stream_gate) load_gate(gate_of(0));
    ring.wait(0, 0);
    if (stream_gate) load_gate(gate_of(0));
    row_sums(0, now);
  }
  __syncthreads();
  int s_next = p.stages > 1 ? 1 : 0;
  phase = p.stages > 1 ? 0 : 1;
  for (long long row = lo; row < hi; ++row) {
    float sums[4];
    sum4_end(sums, scratch + slot * 128, span);
    slot ^= 1;
    const bool more = row + 1 < hi, group_end = p.gate && (left == 1 || !more);
    const Stats after = stats_of(row + 2);
    // (with one stage the next row comes only when this one is done with)
    const bool early = more && !group_end && p.stages > 1;
    if (early) {
      ring.wait(s_next, phase);
      row_sums(s_next, next);
    }
    row_results(s, row, now, sums);
    if (group_end) {
      flush(gate_of(s));
      ++group;
      left = p.group_rows + 1;
    }
    --left;
    if (more && !early) {
      if (p.stages == 1) {
        __syncthreads();
        ring.ask_all(0, row + 1);
      }
      ring.wait(s_next, phase);
      if (group_end) load_gate(gate_of(s_next));
      row_sums(s_next, next);
    }
    __syncthreads();              // the sums of row + 1 are there, and the stage of this row is done with
    if (p.stages > 1 && row + p.stages < hi) ring.ask_all(s, row + p.stages);
    s = s_next;
    if (++s_next >= p.stages) { s_next = 0; phase ^= 1; }
    now = next;
    next = after;
  }
  if (!p.gate) flush(nullptr);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = tid + i * blockDim.x;
    if (!EXACT && v >= nvec) continue;
    float2* to = reinterpret_cast<float2*>(part_pre) + v * NP;
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (p.w_pre) to[j] = make_float2(a_pre[i][j].lo(), a_pre[i][j].hi());
  }
  if (p.gate && lo >= hi && p.w_post)     // a CTA without rows (none at all, or a gate of more groups than rows)
    for (int c = tid; c < p.d; c += blockDim.x) part_post[c] = 0.f;
  if (abort_flag) {
    const uint64_t begin = globaltimer_ns();
    while (globaltimer_ns() - begin < 2000000) {
    }
  }
}

// Sums of partial rows: blockIdx.y 0 and 1 the weights' (`parts` rows each), 2 + g the gate's group g (`chunks` rows).  A CTA
// owns 128 columns, four a lane; its warps (8, or 32 for many rows) take a row each in turn, up to six loads in flight, and meet in
// shared memory.
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) residual_norm_sums_kernel(const float* __restrict__ scratch, void* dw_post, void* dw_pre, void* dgate,
                                                                 int parts, int chunks, int d, int wide) {
  __shared__ float4 red[WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 128 + lane * 4;
  const int which = blockIdx.y;
  void* out = which == 0 ? dw_post : which == 1 ? dw_pre : dgate;
  if (out == nullptr) return;      // the same for the whole CTA
  const int n = which < 2 ? parts : chunks;
  const size_t at = which < 2 ? size_t(which) * parts * d : (size_t(2) * parts + size_t(which - 2) * chunks) * d;
  const size_t out_at = which < 2 ? 0 : size_t(which - 2) * d;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < d) {                     // (d is a multiple of 4)
    const float* s = scratch + at + c;
#pragma unroll 6
    for (int i = warp; i < n; i += WARPS) {
      const float4 v = *reinterpret_cast<const float4*>(s + size_t(i) * d);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
  }
  red[warp][lane] = a;
  __syncthreads();
  if (threadIdx.x < 128 && blockIdx.x * 128 + int(threadIdx.x) < d) {
    const float* r = reinterpret_cast<const float*>(red) + threadIdx.x;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < WARPS; ++k) v[k & 3] += r[k * 128];
    const float sum = (v[0] + v[1]) + (v[2] + v[3]);
    const size_t o = out_at + blockIdx.x * 128 + threadIdx.x;
    if (wide) static_cast<float*>(out)[o] = sum;
    else static_cast<T*>(out)[o] = from_f<T>(sum);
  }
}

// Threads of a CTA, 16-byte pieces of a row per thread, CTAs per SM, stages of the ring and bytes of shared memory.  Two pieces a
// thread, four where 512 threads need them (rows of more than 16 KB): with tests in the loops, four took 183 us instead of 112 for
// the backward of 8192 x 4096 and 59 instead of 55 forward.  The forward needs two stages and has them: three operands of 32 KB are its most.
struct RnShape {
  int threads, vecs, per_sm, stages, smem;
};
static RnShape rn_shape(int d, int elem, int operands) {
  RnShape s;
  const int nvec = d * elem / 16;
  s.vecs = nvec > 1024 ? 4 : 2;
  s.threads = ((nvec + s.vecs - 1) / s.vecs + 31) / 32 * 32;
  s.per_sm = RN_THREADS / s.threads;
  const int stage = operands * d * elem;
  s.stages = (226 * 1024 / s.per_sm - 2560 - RN_HEAD) / stage;   // (2560: static and reserved shared memory of a CTA)
  if (s.stages > RN_MAX_STAGES) s.stages = RN_MAX_STAGES;
  if (s.stages < 1) s.stages = 1;
  s.smem = RN_HEAD + s.stages * stage;
  return s;
}
struct RnPlan {
  int grid, chunks;
};
// CTAs of the backward, and the parts that a group's rows are cut into: one CTA each, or whole groups to a CTA.
static RnPlan rn_bwd_plan(long long rows, int groups, int per_sm) {
  const long long want = (long long)sm_count_of_device() * per_sm, group_rows = rows / groups;
  long long chunks = want / groups;
  if (chunks > group_rows) chunks = group_rows;
  if (chunks < 1) chunks = 1;
  const long long units = groups * chunks;
  return {int(units < want ? units : want), int(chunks)};
}
// A gate whose rows change after one to three rows of x comes with them through the ring; one that changes seldomer is loaded
// then.  Backward of 8192 x 4096 bf16, streamed / loaded, us: 168 / 199 with a gate of its own for every row, 145 / 152 for every
// two, 135 / 131 for every four, 137 / 121 for every 32.
static bool rn_short_groups(long long rows, int groups) { return groups > 1 && rows / groups < 4; }
static int rn_stream_gate(const void* gate, long long rows, int groups) { return gate && rn_short_groups(rows, groups); }
// (as many operands as the backward can have: the plan must not depend on which are absent, since the scratch goes by it)
static int rn_bwd_operands(long long rows, int groups) { return 4 + rn_short_groups(rows, groups); }
template <typename T, int VECS, bool BWD, int KIND, bool EXACT>
static int rn_launch_as(int grid, const RnShape& shape, const ResNormParams& p, cudaStream_t stream) {
  static SmemLimit limit;
  auto kernel = BWD ? residual_norm_bwd_kernel<T, VECS, KIND, EXACT> : residual_norm_fwd_kernel<T, VECS, KIND, EXACT>;
  if (const int rc = limit.allow(kernel, shape.smem)) return rc;
  kernel<<<grid, shape.threads, shape.smem, stream>>>(p);
  return launch_result(cudaSuccess);
}
template <typename T, bool BWD>
static int rn_launch(int grid, const RnShape& shape, const ResNormParams& p, cudaStream_t s) {
  int kind = RN_ANY;
  if (!p.stream_gate && (!BWD || (p.dr && (p.dh || !p.w_pre))))
    kind = p.w_post && p.w_pre ? RN_BOTH : p.w_post ? RN_POST : p.w_pre ? RN_PRE : RN_ANY;
  const bool exact = p.d == shape.vecs * shape.threads * Vec<T>::N;
  auto with = [&](auto vecs, auto whole) {
    constexpr int VECS = decltype(vecs)::value;
    constexpr bool EXACT = decltype(whole)::value;
    switch (kind) {
      case RN_BOTH: return rn_launch_as<T, VECS, BWD, RN_BOTH, EXACT>(grid, shape, p, s);
      case RN_POST: return rn_launch_as<T, VECS, BWD, RN_POST, EXACT>(grid, shape, p, s);
      case RN_PRE: return rn_launch_as<T, VECS, BWD, RN_PRE, EXACT>(grid, shape, p, s);
    }
    return rn_launch_as<T, VECS, BWD, RN_ANY, false>(grid, shape, p, s);
  };
  const std::integral_constant<int, 2> two;
  const std::integral_constant<int, 4> four;
  if (exact) return shape.vecs == 2 ? with(two, std::true_type()) : with(four, std::true_type());
  return shape.vecs == 2 ? with(two, std::false_type()) : with(four, std::false_type());
}
template <typename F>
static int rn_dtype(int dt, F&& f) {
  if (dt == 0) return f(float{});
  if (dt == 1) return f(__nv_bfloat16{});
  return -JPB_ERR_BAD_ARGUMENT;
}
static bool rn_aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (reinterpret_cast<uintptr_t>(q) & 15) return false;
  return true;
}

}  // namespace jpb

// dtype 0 = fp32, 1 = bf16.  x, y, r, h [rows, d] contiguous, w_post, w_pre [d], gate [groups, d] with rows / groups
// consecutive rows of x to each of its rows; w_post, gate and w_pre (with h) may be null.  rstd_post, rstd_pre [rows].
// Pointers on 16-byte boundaries, d a multiple of 16 bytes.
JPB_API int jpb_residual_norm_fwd(int dt, const void* x, const void* y, const void* w_post, const void* gate, const void* w_pre, void* r,
                                  void* h, float* rstd_post, float* rstd_pre, long long rows, int d, int groups, float scale, float eps,
                                  void* stream) {
  using namespace jpb;
  if (rows <= 0) return 0;
  return rn_dtype(dt, [&](auto tag) {
    using T = decltype(tag);
    constexpr int VN = Vec<T>::N;
    if (d <= 0 || d % VN || d / VN > 2 * 1024 || groups < 1 || rows % groups || !rn_aligned({x, y, w_post, gate, w_pre, r, h}))
      return -int(JPB_ERR_BAD_ARGUMENT);
    ResNormParams p = {};
    p.x = x; p.y = y; p.w_post = w_post; p.gate = gate; p.w_pre = w_pre; p.r = r; p.h = h;
    p.rstd_post = rstd_post; p.rstd_pre = rstd_pre; p.rows = rows; p.d = d; p.group_rows = rows / groups;
    p.scale = scale; p.eps = eps; p.status = jpb_status_device_ptr();
    p.stream_gate = rn_stream_gate(gate, rows, groups);
    const RnShape shape = rn_shape(d, sizeof(T), 2 + p.stream_gate);
    p.stages = shape.stages;
    const long long most = (long long)sm_count_of_device() * shape.per_sm;
    const int grid = int(rows < most ? rows : most);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return rn_launch<T, false>(grid, shape, p, s);
  });
}

// fp32 elements of scratch for jpb_residual_norm_bwd.
JPB_API long long jpb_residual_norm_bwd_scratch_elems(int dt, long long rows, int d, int groups) {
  const jpb::RnShape shape = jpb::rn_shape(d, dt == 0 ? 4 : 2, jpb::rn_bwd_operands(rows, groups));
  const jpb::RnPlan plan = jpb::rn_bwd_plan(rows, groups, shape.per_sm);
  return (2ll * plan.grid + (plan.chunks > 1 ? (long long)groups * plan.chunks : 0)) * d;
}

// dr and dh may be null; dw_post, dgate and dw_pre go with w_post, gate and w_pre and are of the type of x or, with `wide`, fp32.
JPB_API int jpb_residual_norm_bwd(int dt, const void* dr, const void* dh, const void* x, const void* y, const void* w_post,
                                  const void* gate, const void* w_pre, const float* rstd_post, const float* rstd_pre, void* dx, void* dy,
                                  void* dw_post, void* dgate, void* dw_pre, float* scratch, long long rows, int d, int groups, float scale,
                                  int wide, void* stream) {
  using namespace jpb;
  return rn_dtype(dt, [&](auto tag) {
    using T = decltype(tag);
    constexpr int VN = Vec<T>::N;
    if (rows < 0 || d <= 0 || d % VN || d / VN > 2 * 1024 || groups < 1 || rows % groups ||
        !rn_aligned({dr, dh, x, y, w_post, gate, w_pre, dx, dy, dgate}))
      return -int(JPB_ERR_BAD_ARGUMENT);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const RnShape shape = rn_shape(d, sizeof(T), rn_bwd_operands(rows, groups));
    const RnPlan plan = rn_bwd_plan(rows, groups, shape.per_sm);
    ResNormParams p = {};
    p.x = x; p.y = y; p.w_post = w_post; p.gate = gate; p.w_pre = w_pre;
    p.rstd_post = const_cast<float*>(rstd_post); p.rstd_pre = const_cast<float*>(rstd_pre);
    p.dr = dr; p.dh = dh; p.dx = dx; p.dy = dy; p.scratch = scratch; p.rows = rows; p.d = d; p.group_rows = rows / groups;
    p.groups = groups; p.chunks = plan.chunks; p.dgate = dgate; p.wide = wide; p.scale = scale;
    p.stages = shape.stages; p.stream_gate = rn_stream_gate(gate, rows, groups); p.status = jpb_status_device_ptr();
    if (rows == 0 && gate) cudaMemsetAsync(dgate, 0, size_t(groups) * d * (wide ? 4 : sizeof(T)), s);
    const int rc = rn_launch<T, true>(plan.grid, shape, p, s);
    if (rc) return rc;
    const bool gate_sums = gate && plan.chunks > 1;
    if (w_post || w_pre || gate_sums) {
      const dim3 sums((d + 127) / 128, gate_sums ? 2 + groups : 2);
      auto run = [&](auto kernel, int threads) {
        kernel<<<sums, threads, 0, s>>>(scratch, w_post ? dw_post : nullptr, w_pre ? dw_pre : nullptr, gate_sums ? dgate : nullptr,
                                        plan.grid, plan.chunks, d, wide);
      };
      // (148 partial rows of 4096: the whole call 19.5 us with 32 warps, 21.5 with 8; 64: 17.4 with either)
      if (plan.grid > 64) run(residual_norm_sums_kernel<T, 32>, 1024);
      else run(residual_norm_sums_kernel<T, 8>, 256);
    }
    return launch_result(cudaSuccess);
  });
}
