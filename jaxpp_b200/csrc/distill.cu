// Distillation loss of a row of logits z against a teacher's top entries, with cross entropy mixed in, and its gradient.
//
// With t the temperature, p = softmax(z / t), q_j the teacher's probability of entry j (id i_j), S the set of the listed ids,
// Q = sum of q_j, and (where the teacher's whole log-sum-exp is known) q_o = 1 - Q and p_o = 1 - sum over S of p:
//   soft = sum_j q_j (log q_j - log p_{i_j})  [+ q_o (log q_o - log p_o)]        loss = alpha t^2 soft + (1 - alpha) nll
//   d soft / d z_v = ((Q + q_o) p_v - (sum of q_j with i_j = v)) / t      for v in S
//                    ((Q + q_o) - q_o / p_o) p_v / t                      for the others
// p_o is summed over the entries outside of S, never as a difference: a student that agrees with the teacher leaves almost
// nothing there.
//
// A row is copied into shared memory once (bulk copy), by one CTA or, where it is long or there are few rows, a cluster whose
// CTAs have a part each and trade eight sums.  The elements of S are taken out of it first (-inf in their place), so that the
// passes over the row, its maximum, the sums and the gradient, have no special cases; S is added by itself and its gradients
// are written last.
// What bounds it: HBM (a row read, and one written), then the exponentials, of which an SM does 16 a cycle: one per element for
// the sums and one for the gradient.  With both temperatures in play the plain exponential is a power of the softened one where
// t is 2 or 4, else it is taken too.  4096 x 32000 bf16, 64 entries: the loss 60 us (4.4 TB/s; its bytes take 40, one exponential an
// element 29), with the gradient 106 us (4.9 TB/s; a copy would take 80, both exponentials 58): the rest are the barriers between a
// row's phases, which the two or three other CTAs of the SM do not quite cover.  Many entries cost their scattered reads and writes:
// 512 of them 98 and 198 us.
#include "launch.cuh"
#include "vec.cuh"

#include <type_traits>

namespace jpb {

struct DistillParams {
  const void* logits;
  const void *ids, *top;
  const float* lse;            // null: q is renormalised over the entries
  const long long* labels;     // null: no cross entropy
  const float* dloss;          // gradient kernel: weight of each row
  float* loss;
  void* dlogits;
  long long rows;
  int V, K;
  int ids64, top_fp32;
  float temperature, alpha;
  int log_cluster;             // CTAs of a row: 1, 2, 4 or 8
  int buffer;                  // bytes of a CTA's part of a row
  int* status;
};

constexpr int DISTILL_MAX_K = 1024;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// log(x) for x > 0 to half a unit in the last place or so: x = 2^e m with m in [0.75, 1.5), log m = 2 atanh(s) with s = (m - 1) /
// (m + 1), |s| <= 0.2, by its series up to s^13 / 13.  (The approximate logarithm is off by 4e-7 near 1, as much as a small loss
// may be; the 64-bit one takes a microsecond, a tenth of a row's time.)
__device__ __forceinline__ float log_exact(float x) {
  if (!(x > 0.f) || x == INFINITY) return x == 0.f ? -INFINITY : x;
  int e = 0;
  if (x < 1.2e-38f) { x *= 16777216.f; e = -24; }
  const int bits = __float_as_int(x), shift = (bits - 0x3f400000) >> 23;      // 0x3f400000 = 0.75
  const float m = __int_as_float(bits - (shift << 23));
  e += shift;
  const float s = __fdiv_rn(m - 1.f, m + 1.f), q = s * s;
  float r = 1.f / 13.f;
  r = fmaf(r, q, 1.f / 11.f);
  r = fmaf(r, q, 1.f / 9.f);
  r = fmaf(r, q, 1.f / 7.f);
  r = fmaf(r, q, 1.f / 5.f);
  r = fmaf(r, q, 1.f / 3.f);
  r = fmaf(2.f * s * q, r, 2.f * s);
  return fmaf(float(e), 0.693359375f, fmaf(float(e), -2.12194440e-4f, r));    // log 2 in two parts, the first of 10 bits
}

// Sums and maxima over a CTA of WARPS warps (4 or 8), one barrier each; two halves of the scratch take turns.
template <int WARPS>
struct CtaReduce {
  float* scratch;   // [2][WARPS][8]
  int slot;
  template <bool MAX>
  __device__ __forceinline__ float one(float v) {
    float* s = scratch + slot * WARPS * 8;
    slot ^= 1;
    v = MAX ? warp_max(v) : warp_sum(v);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[threadIdx.x & (WARPS - 1)];
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? fmaxf(v, u) : v + u;
    }
    return v;
  }
  __device__ __forceinline__ void max2(float& a, float& b) {
    float* s = scratch + slot * WARPS * 8;
    slot ^= 1;
    a = warp_max(a);
    b = warp_max(b);
    if ((threadIdx.x & 31) == 0) { s[threadIdx.x >> 5] = a; s[WARPS + (threadIdx.x >> 5)] = b; }
    __syncthreads();
    a = s[threadIdx.x & (WARPS - 1)];
    b = s[WARPS + (threadIdx.x & (WARPS - 1))];
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
      b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
  }
  // Eight sums: lanes trade values until each has one of the eight, 9 shuffles instead of 40, and 10 after the barrier.
  __device__ __forceinline__ void eight(float (&v)[8]) {
    const int lane = threadIdx.x & 31;
    float* s = scratch + slot * WARPS * 8;
    slot ^= 1;
    float a[4], b[2];
    const bool h = lane & 16, q = lane & 8, e = lane & 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (h ? v[i + 4] : v[i]) + __shfl_xor_sync(0xffffffffu, h ? v[i] : v[i + 4], 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (q ? a[i + 2] : a[i]) + __shfl_xor_sync(0xffffffffu, q ? a[i] : a[i + 2], 8);
    float x = (e ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, e ? b[0] : b[1], 4);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    if ((lane & 3) == 0) s[(threadIdx.x >> 5) * 8 + (lane >> 2)] = x;     // value number: bits 4, 3, 2 of the lane
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS / 4; ++k) x += s[k * 32 + lane];            // value lane & 7, every fourth warp
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    x += __shfl_xor_sync(0xffffffffu, x, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __shfl_sync(0xffffffffu, x, i);
  }
};

__device__ __forceinline__ float piece_max(const Vec<float>& v) { return fmaxf(fmaxf(v.raw.x, v.raw.y), fmaxf(v.raw.z, v.raw.w)); }
__device__ __forceinline__ float piece_max(const Vec<__nv_bfloat16>& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v.raw);
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(f.x, f.y);
}

// What a CTA tells the others about its part of a row; the sums of exponentials are relative to m, out_t to m_out.
struct PartSums {
  float m, m_out, out_t, in_t, s_1, cross, mass, label;
};
// Below this share of the largest exponential the sum over the elements outside of S is taken relative to its own maximum: it then
// keeps its digits down to the smallest p_o that counts, and 1 / p_o stays out of the gradient's coefficients (below it, a weight of
// 1e22 still fits).  One pass more over such a row.
constexpr float THIN = 9.094947017729282e-13f;       // 2^-40

// MODE: exponentials of a gradient and a loss in which 0 only one temperature counts, 1 / 2 both and t = 2 / 4, 3 both, any t
template <int MODE>
__device__ __forceinline__ float plain_exp(float e, float f, float k1, float m1) {   // exp(f - m) from e = exp((f - m) / t)
  if (MODE == 0) return e;
  if (MODE == 1) return e * e;
  if (MODE == 2) { const float s = e * e; return s * s; }
  return exp2_fast(fmaf(f, k1, -m1));
}
// The factor k (log2(e) / t or log2(e)) of exponents relative to m, or 1 where m * k could leave fp32's range (a part of a row that is
// masked with the type's lowest value has no other maximum): logits of that size are equal or so far apart that any factor does.
__device__ __forceinline__ float factor(float m, float k) { return fabsf(m) > 1.2676506e30f ? 1.f : k; }    // 2^100
__device__ __forceinline__ F2 exp2_pair(F2 x) { return f2(exp2_fast(x.lo()), exp2_fast(x.hi())); }
template <typename T, bool GRAD, int MODE, int THREADS>
__global__ void __launch_bounds__(THREADS, 768 / THREADS) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int VN = Vec<T>::N, ES = sizeof(T);
  using Bits = typename std::conditional<ES == 2, uint16_t, uint32_t>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float scratch[2 * THREADS / 32 * 8];
  __shared__ __align__(16) PartSums parts[2];
  __shared__ uint64_t full;
  __shared__ int abort_flag, repeated[2];
  const int tid = threadIdx.x, V = p.V, K = p.K;
  const int rank = p.log_cluster ? int(cluster_ctarank()) : 0, C = 1 << p.log_cluster;
  const long long row0 = blockIdx.x >> p.log_cluster, row_step = gridDim.x >> p.log_cluster;
  const long long row_bytes = (long long)V * ES, step_bytes = row_step * row_bytes;
  const float it = 1.f / p.temperature, it2 = it * LOG2E;
  CtaReduce<THREADS / 32> reduce{scratch, 0};

  // This CTA's part of the row that begins at byte `begin`: 16-byte pieces lo .. of the whole tensor, and the byte of the row's
  // first element from lo on.
  struct Part {
    long long lo;
    int pieces, lead;
  };
  auto part_of = [&](long long begin) {
    const int lead = int(begin & 15), n = (lead + int(row_bytes) + 15) >> 4, a = (n * rank) >> p.log_cluster;
    return Part{(begin >> 4) + a, ((n * (rank + 1)) >> p.log_cluster) - a, lead - a * 16};
  };
  // pieces that are wholly in the row: copied at once; the one or two others hold elements of the next rows
  auto first_whole = [&](const Part& q) { return q.lead > 0 ? 1 : 0; };
  auto last_whole = [&](const Part& q) { return min(q.pieces, (q.lead + int(row_bytes)) >> 4); };
  auto fetch = [&](long long begin) {                // one thread
    const Part q = part_of(begin);
    const int a = first_whole(q), b = last_whole(q);
    if (b > a) {
      mbar_expect_tx(&full, uint32_t(b - a) * 16);
      bulk_load(smem + a * 16, static_cast<const uint8_t*>(p.logits) + (q.lo + a) * 16, uint32_t(b - a) * 16, &full);
    } else {
      mbar_arrive(&full);
    }
  };
  // What a row needs beside its logits is asked for a row ahead: first the entries (one a thread; further ones when their turn
  // comes), the label and the row's numbers, and when these are there the logits that they name.  All of it is kept as it comes:
  // a conversion would wait for the load.
  struct Ahead {
    uint32_t id_lo, id_hi, top, z, z_label;
    uint32_t edge;         // an element of the pieces at the ends of the part (16 threads have one each)
    float lse, g;
    long long label;
  };
  auto raw_entry = [&](long long r, int j, Ahead& h) {
    const size_t at = size_t(r) * K + j;
    if (p.ids64) {
      const uint2 w = static_cast<const uint2*>(p.ids)[at];
      h.id_lo = w.x; h.id_hi = w.y;
    } else {
      h.id_lo = static_cast<const uint32_t*>(p.ids)[at];
    }
    h.top = p.top_fp32 ? static_cast<const uint32_t*>(p.top)[at] : static_cast<const uint16_t*>(p.top)[at];
  };
  auto id_of = [&](const Ahead& h) { return p.ids64 ? (long long)(uint64_t(h.id_hi) << 32 | h.id_lo) : (long long)int(h.id_lo); };
  auto raw_logit = [&](long long r, long long v) { return uint32_t(static_cast<const Bits*>(p.logits)[size_t(r) * V + v]); };
  auto logit_of = [&](uint32_t raw) { return __uint_as_float(ES == 2 ? raw << 16 : raw); };
  // Element of the part that thread i has of the pieces at its ends (the others are copied whole), or -1.
  auto edge_of = [&](const Part& q, int i) {
    const int a = first_whole(q) * VN, b = max(a, last_whole(q) * VN);
    return i < a ? i : b + i - a < q.pieces * VN ? b + i - a : -1;
  };
  auto ahead_ids = [&](long long r, long long begin) {
    Ahead h;
    const Part q = part_of(begin);
    const int v = edge_of(q, tid) - q.lead / ES;       // of the row
    h.edge = 0;
    if (tid < 2 * VN && edge_of(q, tid) >= 0 && v >= 0 && v < V) h.edge = raw_logit(r, v);
    h.id_lo = h.id_hi = 0xffffffffu;        // no entry
    h.top = h.z = h.z_label = 0;
    if (tid < K) raw_entry(r, tid, h);
    h.label = p.labels ? p.labels[r] : -1;
    h.lse = p.lse ? p.lse[r] : 0.f;
    h.g = GRAD ? p.dloss[r] : 0.f;
    return h;
  };
  auto ahead_logits = [&](long long r, Ahead& h) {
    const long long id = id_of(h);
    if (id >= 0 && id < V) h.z = raw_logit(r, id);
    if (h.label >= 0 && h.label < V) h.z_label = raw_logit(r, h.label);
  };
  long long begin = row0 * row_bytes;
  if (tid == 0) {
    abort_flag = 0;
    repeated[0] = repeated[1] = 0;
    mbar_init(&full, 1);
    fence_barrier_init();
    if (row0 < p.rows) fetch(begin);
  }
  // The exponentials relative to m are 2^(z * it2 - fl(m * it2)): all of them too large by 2^off, off being what the rounding of
  // m * it2 leaves (and likewise for the plain ones).  Ratios do not see it; the logarithm of a sum takes it off.
  auto off_by = [&](float m, float k) { return fmaf(m, factor(m, k), -(m * factor(m, k))); };
  auto off_t = [&](float m) { return off_by(m, it2); };
  auto off_1 = [&](float m) { return MODE == 1 ? 2.f * off_t(m) : MODE == 2 ? 4.f * off_t(m) : MODE == 3 ? off_by(m, LOG2E) : off_t(m); };
  Ahead next;
  if (row0 < p.rows) {
    next = ahead_ids(row0, begin);
    ahead_logits(row0, next);
  }
  __syncthreads();
  int turn = 0;
  for (long long row = row0; row < p.rows; row += row_step, begin += step_bytes, turn ^= 1) {
    const Part q = part_of(begin);
    uint8_t* buf = smem;                             // this CTA's part of the row
    // [K] elements of the part where the entries' ids are (-2: no entry, -1: in another part), their logits and probabilities;
    // two sets take turns, so that the last gradients of a row need not be waited for
    int* s_id = reinterpret_cast<int*>(smem + p.buffer) + turn * 3 * K;
    float* s_q = reinterpret_cast<float*>(s_id + K);
    float* s_z = s_q + K;
    T* elem = reinterpret_cast<T*>(buf);
    const int lead = q.lead / ES;                    // element of the part that the row's first one would be (or is)
    const int n = q.pieces * VN;
    const int v_lo = max(lead, 0), v_hi = min(n, lead + V);        // elements that are of the row
    const T* z = reinterpret_cast<const T*>(static_cast<const uint8_t*>(p.logits) + begin);
    // ---- the teacher's entries, and the row's logits there ----
    const Ahead now = next;
    const long long label = now.label;
    const bool label_here = label >= 0 && label < V && label + lead >= v_lo && label + lead < v_hi;
    const int label_at = label_here ? int(label + lead) : -1;
    const float z_own = logit_of(now.z_label);
    float z_label = z_own;
    const bool more = row + row_step < p.rows;
    if (more) next = ahead_ids(row + row_step, begin + step_bytes);
    // the largest of the teacher's values, and of the row's logits at the same places
    float top_max = -INFINITY, ref = -INFINITY;
    for (int j = tid; j < K; j += THREADS) {
      Ahead h = now;
      if (j != tid) raw_entry(row, j, h);
      const long long id = id_of(h);
      const float top = it * __uint_as_float(p.top_fp32 ? h.top : h.top << 16);
      const bool valid = id >= 0 && id < V && top != -INFINITY;
      if (valid) {
        const float zj = logit_of(j == tid ? h.z : raw_logit(row, id));
        s_z[j] = zj;
        top_max = fmaxf(top_max, top == top ? top : INFINITY);      // (a NaN is an entry too)
        ref = fmaxf(ref, zj);
      }
      const long long e = id + lead;
      s_id[j] = !valid ? -2 : e >= v_lo && e < v_hi ? int(e) : -1;
      s_q[j] = top;
    }
    if (tid < 2 * VN) {      // pieces at the ends of the part: the row's elements, and -inf around them
      const int v = edge_of(q, tid);
      if (v >= 0) reinterpret_cast<Bits*>(buf)[v] = v >= v_lo && v < v_hi ? Bits(now.edge) : ES == 2 ? Bits(0xff80u) : Bits(0xff800000u);
    }
    reduce.max2(top_max, ref);
    const bool some = top_max != -INFINITY;
    // The exponentials are taken relative to the largest logit among the entries (the label's, or 0, where there are none): the
    // row's maximum is no further above it than fp32 has room for, or is looked up after all (below).
    if (ref == -INFINITY) ref = label >= 0 && label < V && z_own != -INFINITY ? z_own : 0.f;
    float q_sum = 1.f;                                 // log q = top - lse, or top - top_max - log of this sum
    if (p.lse == nullptr && some) {
      float sum = 0.f;
      for (int j = tid; j < K; j += THREADS)
        if (s_id[j] != -2) sum += exp2_fast((s_q[j] - top_max) * LOG2E);
      q_sum = reduce.template one<false>(sum);
    }
    // out_t, out_1: sums over the others; in_t, in_1: over S; cross = sum of q (log q - (z - ref) / t) without the logarithm of
    // q_sum; mass = sum of q
    float out_t, out_1, in_t = 0.f, in_1 = 0.f, cross = 0.f, mass_in = 0.f;
    {
      const float q_sub = p.lse ? now.lse : top_max, q_inv = 1.f / q_sum;
      for (int j = tid; j < K; j += THREADS) {
        const int at = s_id[j];
        if (at == -2) continue;
        const float logq = s_q[j] - q_sub, qj = exp2_fast(logq * LOG2E) * q_inv;
        s_q[j] = qj;
        if (at < 0) continue;
        if (qj != 0.f) cross += qj * (logq - (s_z[j] - ref) * it);
        mass_in += qj;
      }
    }
    // ---- the row ----
    mbar_wait_bounded(&full, turn, &abort_flag, p.status);
    // S is taken out of the row: every entry leaves its number in its place, and the one whose number is found there stands for
    // the id and leaves -inf (whose bits are no entry's number)
    volatile Bits* place = reinterpret_cast<volatile Bits*>(buf);
    for (int j = tid; j < K; j += THREADS)
      if (s_id[j] >= 0) place[s_id[j]] = Bits(j);
    if (tid == 0) repeated[turn ^ 1] = 0;
    __syncthreads();
    unsigned owner = 0;                                // bit i: this thread's i-th entry stands for its id (K <= 1024)
    for (int j = tid, i = 0; j < K; j += THREADS, ++i)
      if (s_id[j] >= 0) {
        if (place[s_id[j]] == Bits(j)) {
          owner |= 1u << i;
          place[s_id[j]] = ES == 2 ? Bits(0xff80u) : Bits(0xff800000u);
        } else {
          repeated[turn] = 1;
        }
      }
    __syncthreads();
    const bool twice = repeated[turn] != 0;
    if (twice) {                                       // the first of its kind, whichever write came last
      owner = 0;
      for (int j = tid, i = 0; j < K; j += THREADS, ++i) {
        bool first = s_id[j] >= 0;
        for (int k = 0; k < j && first; ++k) first = s_id[k] != s_id[j];
        if (first) owner |= 1u << i;
      }
    }
    if (more) ahead_logits(row + row_step, next);
    const Vec<T>* piece = reinterpret_cast<const Vec<T>*>(buf);
    float m = ref;
    for (int attempt = 0;; ++attempt) {
      const float km = factor(m, it2), k1m = factor(m, LOG2E), mt = m * km, m1 = m * k1m;
      F2 sum_t = f2(0.f), sum_1 = f2(0.f);
      const F2 k = f2(km), k1 = f2(k1m), at = f2(-mt), at1 = f2(-m1);
#pragma unroll 2
      for (int i = tid; i < q.pieces; i += THREADS) {
        F2 f[VN / 2];
        to_pairs(piece[i], f);
#pragma unroll
        for (int j = 0; j < VN / 2; ++j) {
          const F2 e = exp2_pair(fma2(f[j], k, at));
          sum_t = sum_t + e;
          if (MODE == 1) sum_1 = fma2(e, e, sum_1);
          if (MODE == 2) { const F2 h = e * e; sum_1 = fma2(h, h, sum_1); }
          if (MODE == 3) sum_1 = sum_1 + exp2_pair(fma2(f[j], k1, at1));
        }
      }
      in_t = in_1 = 0.f;
      for (int j = tid, i = 0; j < K; j += THREADS, ++i)
        if (owner >> i & 1) {
          const float e = exp2_fast(fmaf(s_z[j], km, -mt));
          in_t += e;
          if (MODE != 0) in_1 += plain_exp<MODE>(e, s_z[j], k1m, m1);
        }
      float acc[8] = {sum_t.lo() + sum_t.hi(), sum_1.lo() + sum_1.hi(), in_t, in_1, attempt ? 0.f : cross, attempt ? 0.f : mass_in, 0.f, 0.f};
      if (!GRAD) fence_proxy_async();   // elements of the row were written here, the next row comes by the bulk-copy unit
      reduce.eight(acc);
      out_t = acc[0]; out_1 = acc[1]; in_t = acc[2]; in_1 = acc[3];
      if (attempt == 0) { cross = acc[4]; mass_in = acc[5]; }
      const float s_t = out_t + in_t, s_1 = MODE == 0 ? s_t : out_1 + in_1;
      if (attempt || (s_t > 1e-30f && s_t < 1e30f && s_1 > 1e-30f && s_1 < 1e30f)) break;
      // out of range: relative to this part's own maximum (the same in all threads: the sums are)
      float mx = -INFINITY;
      for (int i = tid; i < q.pieces; i += THREADS) mx = fmaxf(mx, piece_max(piece[i]));
      for (int j = tid; j < K; j += THREADS)
        if (s_id[j] >= 0) mx = fmaxf(mx, s_z[j]);
      mx = reduce.template one<true>(mx);
      if (mx == -INFINITY) break;       // nothing here but -inf: sums of zero, relative to anything
      m = mx;
    }
    float m_out = m;
    if (p.lse != nullptr && out_t < THIN) {
      float mx = -INFINITY;
#pragma unroll 1
      for (int i = tid; i < q.pieces; i += THREADS) mx = fmaxf(mx, piece_max(piece[i]));
      mx = reduce.template one<true>(mx);
      if (mx != -INFINITY) {            // (else there is nothing outside)
        const float km = factor(mx, it2), mt = mx * km;
        float sum = 0.f;
#pragma unroll 1
        for (int i = tid; i < q.pieces; i += THREADS) {
          F2 f[VN / 2];
          to_pairs(piece[i], f);
#pragma unroll
          for (int j = 0; j < VN / 2; ++j) sum += exp2_fast(fmaf(f[j].lo(), km, -mt)) + exp2_fast(fmaf(f[j].hi(), km, -mt));
        }
        out_t = reduce.template one<false>(sum);
        m_out = mx;
      }
    }
    if (!GRAD && tid == THREADS - 32 && more) fetch(begin + step_bytes);   // (all have read it)
    // ---- together with the other parts ----
    float M = m, M_out = m_out, s_1 = out_1 + in_1;
    if (C > 1) {
      PartSums* mine = &parts[turn];
      if (tid == 0) *mine = {m, m_out, out_t, in_t, s_1, cross, mass_in, label_here ? z_own : -INFINITY};
      __syncwarp();
      cluster_sync();
      // lane c reads part c (lanes go round), and the parts are added up across lanes: one trip to the other SMs
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(tid & (C - 1)));
      PartSums o;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.m), "=f"(o.m_out), "=f"(o.out_t), "=f"(o.in_t) : "r"(at) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.s_1), "=f"(o.cross), "=f"(o.mass), "=f"(o.label) : "r"(at + 16) : "memory");
      M = o.m;
      M_out = o.out_t > 0.f ? o.m_out : -INFINITY;     // (a part with nothing outside has no say)
      for (int x = 1; x < C; x <<= 1) {
        M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        M_out = fmaxf(M_out, __shfl_xor_sync(0xffffffffu, M_out, x));
      }
      if (M_out == -INFINITY) M_out = M;
      const float et = exp2_fast((o.m - M) * it2 + (off_t(M) - off_t(o.m))), e1 = exp2_fast((o.m - M) * LOG2E + (off_1(M) - off_1(o.m)));
      const float eo = o.m_out == o.m && M_out == M ? et : exp2_fast((o.m_out - M_out) * it2 + (off_t(M_out) - off_t(o.m_out)));
      out_t = o.out_t == 0.f ? 0.f : o.out_t * eo; in_t = o.in_t * et; s_1 = o.s_1 * e1;
      cross = o.cross; mass_in = o.mass; z_label = o.label;
      for (int x = 1; x < C; x <<= 1) {
        out_t += __shfl_xor_sync(0xffffffffu, out_t, x);
        in_t += __shfl_xor_sync(0xffffffffu, in_t, x);
        if (MODE != 0) s_1 += __shfl_xor_sync(0xffffffffu, s_1, x);
        cross += __shfl_xor_sync(0xffffffffu, cross, x);
        mass_in += __shfl_xor_sync(0xffffffffu, mass_in, x);
        z_label = fmaxf(z_label, __shfl_xor_sync(0xffffffffu, z_label, x));
      }
    }
    const bool thin = M_out != M;                      // out_t has a reference of its own
    float s_t = out_t + in_t, p_o = out_t / s_t, shift = 0.f;
    if (thin) {
      shift = (M_out - M) * it2 + (off_t(M) - off_t(M_out));
      s_t = fmaf(out_t, exp2_fast(shift), in_t);
      const float l = shift + __log2f(out_t) - __log2f(s_t);
      p_o = l >= -126.f ? exp2_fast(l) : l == l ? 0.f : l;
    }
    if (MODE == 0) s_1 = s_t;
    // (comparisons that keep a NaN of the teacher's: fmaxf(0, NaN) would be 0)
    const float q_o = p.lse == nullptr || mass_in >= 1.f ? 0.f : 1.f - mass_in;
    const bool rest = q_o > 0.f && p_o > 0.f;
    const float ratio = rest ? q_o / p_o : 0.f, mass = rest ? mass_in + q_o : mass_in;
    const bool hard = label >= 0 && label < V && p.alpha < 1.f;
    T* dz = reinterpret_cast<T*>(static_cast<uint8_t*>(p.dlogits) + begin);
    const float gs = some ? now.g * p.alpha * p.temperature : 0.f;   // alpha t^2 / t
    const float gh = hard ? now.g * (1.f - p.alpha) : 0.f;
    // gradient = ct * exp((z - M) / t) + c1 * exp(z - M); a row of weight zero has none, whatever it holds
    const bool zero = now.g == 0.f || (gs == 0.f && gh == 0.f);
    float ct = gs != 0.f ? gs * (mass - ratio) / s_t : 0.f, ct_in = gs != 0.f ? gs * mass / s_t : 0.f, c1 = gh != 0.f ? gh / s_1 : 0.f;
    if (MODE == 0) { ct += c1; ct_in += c1; }
    // Outside of S: relative to M_out, where the plain exponential is a power of the softened one too.
    float c1_out = MODE == 0 ? 0.f : c1;
    if (thin) {
      ct = gs != 0.f ? gs * ((mass * p_o - (rest ? q_o : 0.f)) / out_t) : 0.f;
      if (MODE == 0) ct = fmaf(c1, exp2_fast(shift), ct);
      if (MODE == 1) c1_out *= exp2_fast(2.f * shift);
      if (MODE == 2) c1_out *= exp2_fast(4.f * shift);
    }
    const float kM = factor(M, it2), k1M = factor(M, LOG2E), Mt = M * kM, M1 = M * k1M;
    const float kM_out = factor(M_out, it2), Mt_out = M_out * kM_out;
    auto grad_of = [&](float f, float c, float c1, float k, float Mt) {
      const float e = exp2_fast(fmaf(f, k, -Mt));
      return MODE == 0 ? c * e : fmaf(c, e, c1 * plain_exp<MODE>(e, f, k1M, M1));
    };
    auto grad_out = [&](float f) { return grad_of(f, ct, c1_out, kM_out, Mt_out); };
    if constexpr (GRAD) {
      uint8_t* out = static_cast<uint8_t*>(p.dlogits) + q.lo * 16;
      const int a = first_whole(q), b = last_whole(q);
      if (zero) {
        for (int i = a + tid; i < b; i += THREADS) *reinterpret_cast<uint4*>(out + size_t(i) * 16) = make_uint4(0, 0, 0, 0);
      } else {
        const F2 k = f2(kM_out), k1 = f2(k1M), at = f2(-Mt_out), at1 = f2(-M1), wt = f2(ct), w1 = f2(c1_out);
#pragma unroll 2
        for (int i = a + tid; i < b; i += THREADS) {
          F2 f[VN / 2];
          to_pairs(piece[i], f);
#pragma unroll
          for (int j = 0; j < VN / 2; ++j) {
            const F2 e = exp2_pair(fma2(f[j], k, at));
            if (MODE == 0) f[j] = wt * e;
            if (MODE == 1) f[j] = e * fma2(w1, e, wt);
            if (MODE == 2) { const F2 h = e * e; f[j] = e * fma2(w1 * h, e, wt); }
            if (MODE == 3) f[j] = fma2(wt, e, w1 * exp2_pair(fma2(f[j], k1, at1)));
          }
          Vec<T> o;
          from_pairs(o, f);
          o.store(reinterpret_cast<T*>(out + size_t(i) * 16));
        }
      }
      const int ae = a * VN, be = max(ae, b * VN);
      for (int i = tid; i < ae + n - be; i += THREADS) {
        const int v = i < ae ? i : be + i - ae;
        if (v >= v_lo && v < v_hi) dz[v - lead] = from_f<T>(zero ? 0.f : grad_out(to_f(elem[v])));
      }
      fence_proxy_async();
      __syncthreads();            // the row is done with; the elements of S and the label's are written again
      if (tid == THREADS - 32 && more) fetch(begin + step_bytes);
      if (!zero) {
        for (int j = tid, i = 0; j < K; j += THREADS, ++i) {
          if (!(owner >> i & 1)) continue;
          const int e = s_id[j];
          float qj = s_q[j];
          if (twice)
            for (int k = j + 1; k < K; ++k)
              if (s_id[k] == e) qj += s_q[k];
          float d = grad_of(s_z[j], ct_in, c1, kM, Mt) - (gs != 0.f ? gs * qj : 0.f);
          if (e == label_at) d -= gh;
          dz[e - lead] = from_f<T>(d);
        }
        if (tid == THREADS - 1 && label_here && gh != 0.f) {
          bool listed = false;
          for (int k = 0; k < K; ++k) listed |= s_id[k] == label_at;
          if (!listed) dz[label_at - lead] = from_f<T>(grad_out(z_own) - gh);
        }
      }
    }
    // the loss: its logarithms in four lanes of a warp that has neither the first entries nor the next row to see to
    if (tid >> 5 == THREADS / 32 - 2 && rank == 0) {
      const int lane = tid & 31;
      const float l4 = log_exact(lane == 1 ? q_sum : lane == 2 ? (rest ? ratio : 1.f) : lane == 3 ? s_1 : s_t);
      constexpr float LN2 = 0.6931471805599453f;
      const float log_t = __shfl_sync(0xffffffffu, l4, 0) - off_t(M) * LN2, log_1 = __shfl_sync(0xffffffffu, l4, 3) - off_1(M) * LN2;
      const float log_q = __shfl_sync(0xffffffffu, l4, 1), log_r = __shfl_sync(0xffffffffu, l4, 2);
      float l = 0.f;
      if (some && p.alpha > 0.f) {
        float soft = cross + q_o * log_r;
        if (mass_in != 0.f) soft += mass_in * (log_t + (M - ref) * it - log_q);
        l = p.alpha * p.temperature * p.temperature * soft;
      }
      if (hard) l += (1.f - p.alpha) * (log_1 - (z_label - M));
      if (lane == 0) p.loss[row] = l;
    }
  }
  __syncwarp();
  if (C > 1) cluster_sync();      // a CTA's sums are read by the others
  if (abort_flag) {               // a copy may still be in flight: many times its time
    const uint64_t start = globaltimer_ns();
    while (globaltimer_ns() - start < 2000000) {
    }
  }
}

// How many CTAs share a row, and their size.  A CTA's part is what fits twice or more into an SM's shared memory, so that some CTAs
// copy while others compute; a cluster waits for its slowest part.  Rows of 100 KB (1024 x 50257 bf16) whole, two to an SM: 30 us
// for the loss, 53 with the gradient; halved 37 and 54.  Of 200 KB (2048 x 100000) halved: 119 and 181 us; in four parts 218 and
// 296.  (A CTA that held two rows, the next one on its way, was slower wherever that cost an SM a CTA, and nowhere faster.)
// Gradients of fewer rows than half the SMs are cut further, down to 8 KB: 1 x 32000 7.6 -> 6.6 us, 36 x 32000 7.8 -> 7.4.  The
// loss alone is not (5.3 us against 5.7): there the trade costs what the shorter pass saves.
// 128 threads where four such CTAs fit into an SM, else 256, which two or three CTAs have the registers for: 4096 x 16000 (six
// CTAs) 58 us with 128 threads and 69 with 256, x 24000 (four) 83 and 85, x 28000 (three) 111 and 95.
struct DistillShape {
  int cluster, buffer, smem, threads, per_sm;
};
static DistillShape distill_shape(long long rows, int V, int K, int es, bool grad, int sms) {
  DistillShape s;
  const long long bytes = (long long)V * es + 32;
  s.cluster = 1;
  while (s.cluster < 8 && (bytes / s.cluster > 104 * 1024 || (grad && rows * s.cluster * 2 <= sms && bytes / s.cluster > 8 * 1024))) s.cluster *= 2;
  s.buffer = int((bytes / s.cluster + 32 + 127) / 128 * 128);
  s.smem = s.buffer + 24 * K;
  const int fit = 226 * 1024 / (s.smem + 2560);
  s.threads = fit >= 4 ? 128 : 256;
  const int most = 768 / s.threads;              // (registers for 768 threads)
  s.per_sm = fit > most ? most : fit > 1 ? fit : 1;
  return s;
}

template <typename T, bool GRAD, int MODE, int THREADS>
static int distill_go(const DistillParams& p, const DistillShape& shape, int sms, cudaStream_t stream) {
  auto kernel = distill_kernel<T, GRAD, MODE, THREADS>;
  static SmemLimit limit;
  if (const int rc = limit.allow(kernel, shape.smem)) return rc;
  const long long slots = (long long)sms * shape.per_sm / shape.cluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(int(p.rows < slots ? p.rows : slots) * shape.cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = shape.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = shape.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = shape.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return launch_result(e);
}
template <typename T, bool GRAD, int MODE>
static int distill_threads(const DistillParams& p, const DistillShape& s, int sms, cudaStream_t stream) {
  return s.threads == 256 ? distill_go<T, GRAD, MODE, 256>(p, s, sms, stream) : distill_go<T, GRAD, MODE, 128>(p, s, sms, stream);
}
template <typename T, bool GRAD>
static int distill_mode(DistillParams p, cudaStream_t stream) {
  const int sms = sm_count_of_device();
  const DistillShape s = distill_shape(p.rows, p.V, p.K, sizeof(T), GRAD, sms);
  p.log_cluster = s.cluster == 8 ? 3 : s.cluster == 4 ? 2 : s.cluster == 2;
  p.buffer = s.buffer;
  p.status = jpb_status_device_ptr();
  if (p.alpha == 0.f) p.temperature = 1.f;          // the cross entropy alone
  if (p.labels == nullptr || p.alpha == 1.f || p.temperature == 1.f) return distill_threads<T, GRAD, 0>(p, s, sms, stream);
  if (p.temperature == 2.f) return distill_threads<T, GRAD, 1>(p, s, sms, stream);
  if (p.temperature == 4.f) return distill_threads<T, GRAD, 2>(p, s, sms, stream);
  return distill_threads<T, GRAD, 3>(p, s, sms, stream);
}

}  // namespace jpb

// logits [rows, V] of dtype 0 = fp32 or 1 = bf16, contiguous, on a 16-byte boundary; ids [rows, K] int64 (ids64) or int32; top
// [rows, K] fp32 (top_fp32) or bf16; lse [rows] or null; labels [rows] or null; loss [rows].  With dlogits (like logits) the
// gradient for the row weights dloss is written too.  K <= 1024; a row of logits takes at most
// 8 times 220 KB less 24 bytes an entry.
JPB_API int jpb_distill(int dt, const float* dloss, const void* logits, const void* ids, int ids64, const void* top, int top_fp32,
                        const float* lse, const long long* labels, float temperature, float alpha, float* loss, void* dlogits,
                        long long rows, int V, int K, void* stream) {
  using namespace jpb;
  if (rows <= 0) return 0;
  // (a part of the largest row and its entries take up to 163 bytes more than 220 KB, of the 227 that a CTA may have)
  if (V <= 0 || K < 0 || K > DISTILL_MAX_K || (long long)V * (dt == 0 ? 4 : 2) > 8ll * (220 * 1024 - 24 * K) || (dlogits && !dloss) ||
      ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(dlogits)) & 15))
    return -JPB_ERR_BAD_ARGUMENT;
  DistillParams p = {logits, ids, top, lse, labels, dloss, loss, dlogits, rows, V, K, ids64, top_fp32, temperature, alpha, 0, 0, nullptr};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dt == 0) return dlogits ? distill_mode<float, true>(p, s) : distill_mode<float, false>(p, s);
  if (dt == 1) return dlogits ? distill_mode<__nv_bfloat16, true>(p, s) : distill_mode<__nv_bfloat16, false>(p, s);
  return -JPB_ERR_BAD_ARGUMENT;
}
