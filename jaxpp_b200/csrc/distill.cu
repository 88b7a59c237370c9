// Distillation loss of a row of logits z against a teacher's top entries, with cross entropy mixed in, and its gradient.
//
// With t the temperature, p = softmax(z / t), q_j the teacher's probability of entry j (id i_j), S the set of the listed ids,
// Q = sum of q_j, and (where the teacher's whole log-sum-exp is known) q_o = 1 - Q and p_o = 1 - sum over S of p:
//   soft = sum_j q_j (log q_j - log p_{i_j})  [+ q_o (log q_o - log p_o)]        loss = alpha t^2 soft + (1 - alpha) nll
//   d soft / d z_v = ((Q + q_o) p_v - (sum of q_j with i_j = v)) / t      for v in S
//                    ((Q + q_o) - q_o / p_o) p_v / t                      for the others
// p_o is summed over the entries outside of S, never as a difference: a student that agrees with the teacher leaves almost
// nothing there.  A bit per vocabulary entry in shared memory says what S holds; it also tells repeated ids.
#include "vec.cuh"

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
};

constexpr int DISTILL_THREADS = 512;
constexpr int DISTILL_MAX_K = 1024;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The logarithms of a row's sums are taken once a row, in 64 bits: the fast fp32 logarithm is off by 4e-7 near 1, as much as
// a small loss may be.
__device__ __forceinline__ float log_exact(float x) { return float(log(double(x))); }

__device__ __forceinline__ float block_max(float v, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  v = warp_max(v);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  return warp_max(lane < nwarps ? scratch[lane] : -INFINITY);
}

// exp(z - m) summed with m running: (m, s_t, s_1) of the scaled and the plain exponentials
struct Online {
  float m = -INFINITY, st = 0.f, s1 = 0.f;
  __device__ __forceinline__ void raise(float to, float it2) {   // to >= m
    if (to > m) {
      if (m != -INFINITY) {
        st *= exp2_fast((m - to) * it2);
        s1 *= exp2_fast((m - to) * LOG2E);
      }
      m = to;
    }
  }
  __device__ __forceinline__ void add(float f, float it2) {      // after raise(f) or more
    if (f == -INFINITY) return;
    st += exp2_fast((f - m) * it2);
    s1 += exp2_fast((f - m) * LOG2E);
  }
};

template <typename T, bool GRAD>
__global__ void __launch_bounds__(DISTILL_THREADS) distill_kernel(const __grid_constant__ DistillParams p) {
  constexpr int VN = Vec<T>::N;
  extern __shared__ uint32_t dyn[];
  __shared__ float scratch[4 * 32];
  __shared__ int repeated;
  int* s_id = reinterpret_cast<int*>(dyn);                 // [K]
  float* s_q = reinterpret_cast<float*>(dyn + p.K);        // [K]
  uint32_t* bits = dyn + 2 * p.K;                          // a bit per entry, counted from the first aligned one
  const int words = (p.V + 31) / 32 + 1;
  const int tid = threadIdx.x, V = p.V, K = p.K;
  const float it = 1.f / p.temperature, it2 = it * LOG2E;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* z = static_cast<const T*>(p.logits) + size_t(row) * V;
    // vectors start at the first element on a 16-byte boundary
    const int head = min(V, int((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / int(sizeof(T)));
    const int nvec = (V - head) / VN, tail = head + nvec * VN;
    auto bit_at = [&](int v) { return v - head + 32; };    // the head's bits come first, from 32 - head on
    // ---- the teacher's entries ----
    __syncthreads();
    if (tid == 0) repeated = 0;
    for (int w = tid; w < words; w += DISTILL_THREADS) bits[w] = 0;
    float tmax = -INFINITY;
    for (int j = tid; j < K; j += DISTILL_THREADS) {
      const size_t at = size_t(row) * K + j;
      const long long id = p.ids64 ? static_cast<const long long*>(p.ids)[at] : (long long)static_cast<const int*>(p.ids)[at];
      const float top = p.top_fp32 ? static_cast<const float*>(p.top)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.top)[at]);
      const bool valid = id >= 0 && id < V && top != -INFINITY;
      s_id[j] = valid ? int(id) : -1;
      s_q[j] = top * it;
      if (valid) tmax = fmaxf(tmax, top * it);
    }
    tmax = block_max(tmax, scratch);
    const bool some = tmax != -INFINITY;                   // (also where an entry is NaN beside others; all NaN: no entry)
    float sums[2] = {0.f, 0.f};
    if (p.lse == nullptr) {
      for (int j = tid; j < K; j += DISTILL_THREADS)
        if (s_id[j] >= 0) sums[0] += exp2_fast((s_q[j] - tmax) * LOG2E);
      block_sum<1>(reinterpret_cast<float(&)[1]>(sums[0]), scratch);
    }
    // log q_j = s_q[j] - tmax - log of the sum, or s_q[j] - lse
    const float q_sub = p.lse ? p.lse[row] : tmax, q_log = p.lse || !some ? 0.f : log_exact(sums[0]);
    for (int j = tid; j < K; j += DISTILL_THREADS) {
      const int id = s_id[j];
      if (id < 0) continue;
      const int b = bit_at(id);
      if (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) { repeated = 1; }
    }
    __syncthreads();
    // ---- sums over the row: outside of S, then S ----
    Online o;
    auto inside = [&](int v) { const int b = bit_at(v); return (bits[b >> 5] >> (b & 31)) & 1u; };
    for (int v = tid; v < nvec; v += DISTILL_THREADS) {
      Vec<T> x;
      x.load(z + head + v * VN);
      float f[VN];
      x.to_float(f);
      const int b = bit_at(head + v * VN);
      const uint32_t in = (bits[b >> 5] >> (b & 31)) & ((1u << VN) - 1u);
      if (in) {
#pragma unroll
        for (int j = 0; j < VN; ++j)
          if (in >> j & 1) f[j] = -INFINITY;
      }
      float mx = f[0];
#pragma unroll
      for (int j = 1; j < VN; ++j) mx = fmaxf(mx, f[j]);
      o.raise(mx, it2);
#pragma unroll
      for (int j = 0; j < VN; ++j) o.add(f[j], it2);
    }
    for (int c = tid; c < head + (V - tail); c += DISTILL_THREADS) {
      const int v = c < head ? c : tail + c - head;
      if (inside(v)) continue;
      const float f = to_f(z[v]);
      o.raise(f, it2);
      o.add(f, it2);
    }
    float m = o.m;
    for (int j = tid; j < K; j += DISTILL_THREADS)
      if (s_id[j] >= 0) m = fmaxf(m, to_f(z[s_id[j]]));
    m = block_max(m, scratch);
    if (m == -INFINITY) m = 0.f;                           // a row of nothing but -inf: sums of zero
    const float keep = o.m == -INFINITY ? 0.f : 1.f;
    float acc[4] = {keep * o.st * exp2_fast(keep == 0.f ? 0.f : (o.m - m) * it2), keep * o.s1 * exp2_fast(keep == 0.f ? 0.f : (o.m - m) * LOG2E), 0.f, 0.f};
    // S: an id that is listed twice counts once, for its first entry
    const bool twice = repeated != 0;
    for (int j = tid; j < K; j += DISTILL_THREADS) {
      const int id = s_id[j];
      if (id < 0) continue;
      bool first = true;
      if (twice) for (int i = 0; i < j; ++i) if (s_id[i] == id) { first = false; break; }
      if (!first) continue;
      const float f = to_f(z[id]) - m;
      acc[2] += exp2_fast(f * it2);
      acc[3] += exp2_fast(f * LOG2E);
    }
    block_sum<4>(acc, scratch);
    const float s_out = acc[0], s_t = acc[0] + acc[2], s_1 = acc[1] + acc[3];
    const float log_t = log_exact(s_t);
    // ---- the loss ----
    sums[0] = sums[1] = 0.f;
    for (int j = tid; j < K; j += DISTILL_THREADS) {
      const int id = s_id[j];
      if (id < 0) continue;
      const float logq = s_q[j] - q_sub - q_log, q = exp2_fast(logq * LOG2E);
      if (q > 0.f) sums[0] += q * (logq - ((to_f(z[id]) - m) * it - log_t));
      sums[1] += q;
      s_q[j] = q;
    }
    block_sum<2>(sums, scratch);
    float soft = sums[0], mass = sums[1], ratio = 0.f;
    if (p.lse) {
      const float q_o = fmaxf(0.f, 1.f - mass), p_o = s_out / s_t;
      if (q_o > 0.f && p_o > 0.f) {
        ratio = q_o / p_o;
        soft += q_o * log_exact(ratio);
        mass += q_o;
      }
    }
    const long long lab = p.labels ? p.labels[row] : -1;
    const bool hard = lab >= 0 && lab < V;
    if (tid == 0) {
      float l = some ? p.alpha * p.temperature * p.temperature * soft : 0.f;
      if (hard) l += (1.f - p.alpha) * (log_exact(s_1) - (to_f(z[lab]) - m));
      p.loss[row] = l;
    }
    if constexpr (GRAD) {
      T* dz = static_cast<T*>(p.dlogits) + size_t(row) * V;
      const float g = p.dloss[row];
      const float gs = some ? g * p.alpha * p.temperature : 0.f;   // alpha t^2 / t
      const float gh = hard ? g * (1.f - p.alpha) : 0.f;
      const float ct = gs * (mass - ratio) / s_t, c1 = gh / s_1, ct_in = gs * mass / s_t;
      const bool zero = g == 0.f || (gs == 0.f && gh == 0.f);
      auto grad = [&](float f, int v) {
        float d = 0.f;
        if (gs != 0.f) d = ct * exp2_fast((f - m) * it2);
        if (gh != 0.f) {
          d += c1 * exp2_fast((f - m) * LOG2E);
          if (v == lab) d -= gh;
        }
        return d;
      };
      for (int v = tid; v < nvec; v += DISTILL_THREADS) {
        Vec<T> x;
        float f[VN];
        if (zero) {
#pragma unroll
          for (int j = 0; j < VN; ++j) f[j] = 0.f;
        } else {
          x.load(z + head + v * VN);
          x.to_float(f);
#pragma unroll
          for (int j = 0; j < VN; ++j) f[j] = grad(f[j], head + v * VN + j);
        }
        x.from_float(f);
        x.store(dz + head + v * VN);
      }
      for (int c = tid; c < head + (V - tail); c += DISTILL_THREADS) {
        const int v = c < head ? c : tail + c - head;
        dz[v] = from_f<T>(zero ? 0.f : grad(to_f(z[v]), v));
      }
      if (!zero && gs != 0.f) {
        __syncthreads();          // the entries of S are written again
        for (int j = tid; j < K; j += DISTILL_THREADS) {
          const int id = s_id[j];
          if (id < 0) continue;
          float q = s_q[j];
          bool first = true;
          if (twice) {
            for (int i = 0; i < j; ++i) if (s_id[i] == id) { first = false; break; }
            if (first) for (int i = j + 1; i < K; ++i) if (s_id[i] == id) q += s_q[i];
          }
          if (!first) continue;
          const float f = to_f(z[id]) - m;
          float d = ct_in * exp2_fast(f * it2) - gs * q;
          if (gh != 0.f) d += c1 * exp2_fast(f * LOG2E) - (id == lab ? gh : 0.f);
          dz[id] = from_f<T>(d);
        }
      }
    }
  }
}

template <typename T>
static int distill_launch(const DistillParams& p, cudaStream_t stream) {
  const int smem = (2 * p.K + (p.V + 31) / 32 + 2) * 4;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = int(p.rows < 4ll * sms ? p.rows : 4ll * sms);
  auto go = [&](auto kernel) {
    if (smem > 40 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return int(e);
    }
    kernel<<<grid, DISTILL_THREADS, smem, stream>>>(p);
    return int(cudaGetLastError());
  };
  return p.dlogits ? go(distill_kernel<T, true>) : go(distill_kernel<T, false>);
}

}  // namespace jpb

// logits [rows, V] of dtype 0 = fp32 or 1 = bf16, contiguous; ids [rows, K] int64 (ids64) or int32; top [rows, K] fp32 (top_fp32)
// or bf16; lse [rows] or null; labels [rows] or null; loss [rows].  With dlogits (like logits, its address alike modulo 16) the
// gradient for the row weights dloss is written too.  K <= 1024; V at most 1.4 million.
JPB_API int jpb_distill(int dt, const float* dloss, const void* logits, const void* ids, int ids64, const void* top, int top_fp32,
                        const float* lse, const long long* labels, float temperature, float alpha, float* loss, void* dlogits,
                        long long rows, int V, int K, void* stream) {
  using namespace jpb;
  if (rows <= 0) return 0;
  if (V <= 0 || K < 0 || K > DISTILL_MAX_K || V > 1400000 || (dlogits && !dloss) ||
      (dlogits && ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15)))
    return -JPB_ERR_BAD_ARGUMENT;
  DistillParams p = {logits, ids, top, lse, labels, dloss, loss, dlogits, rows, V, K, ids64, top_fp32, temperature, alpha};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dt == 0) return distill_launch<float>(p, s);
  if (dt == 1) return distill_launch<__nv_bfloat16>(p, s);
  return -JPB_ERR_BAD_ARGUMENT;
}
