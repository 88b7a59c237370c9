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
// What bounds it: HBM, four rows moved per row forward (x, y, r, h) and six backward (dr, dh, x, y, dx, dy).
#include "vec.cuh"

#include <initializer_list>

namespace jpb {

struct ResNormParams {
  const void *x, *y, *w_post, *gate, *w_pre;
  void *r, *h;
  float *rstd_post, *rstd_pre;
  const void *dr, *dh;
  void *dx, *dy;
  float* scratch;
  long long rows;
  int d;
  long long group_rows;   // rows of x for each row of the gate
  int groups, chunks;     // backward: every group's rows are cut into `chunks` units
  void* dgate;            // written by the main kernel where chunks == 1
  int wide;
  float scale, eps;
};

constexpr int RN_VECS = 2;   // 16-byte pieces of a row per thread

template <typename T>
__device__ __forceinline__ void load_vec(const void* base, size_t at, float (&f)[Vec<T>::N]) {
  Vec<T> v;
  v.load(static_cast<const T*>(base) + at);
  v.to_float(f);
}
template <typename T>
__device__ __forceinline__ void store_vec(void* base, size_t at, const float (&f)[Vec<T>::N]) {
  Vec<T> v;
  v.from_float(f);
  v.store(static_cast<T*>(base) + at);
}

template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_fwd_kernel(const __grid_constant__ ResNormParams p) {
  constexpr int VN = Vec<T>::N;
  __shared__ float scratch[64];
  const int nvec = p.d / VN;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const size_t base = size_t(row) * p.d;
    const size_t gate_base = p.gate ? size_t(row / p.group_rows) * p.d : 0;
    float y[RN_VECS][VN], r[RN_VECS][VN];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < RN_VECS; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= nvec) continue;
      load_vec<T>(p.y, base + v * VN, y[i]);
      load_vec<T>(p.x, base + v * VN, r[i]);
#pragma unroll
      for (int j = 0; j < VN; ++j) s[0] += y[i][j] * y[i][j];
    }
    float rstd1 = 1.f;
    if (p.w_post) {
      block_sum<1>(s, scratch);
      rstd1 = rsqrtf(s[0] / p.d + p.eps);
      if (threadIdx.x == 0) p.rstd_post[row] = rstd1;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < RN_VECS; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= nvec) continue;
      float w[VN], g[VN];
#pragma unroll
      for (int j = 0; j < VN; ++j) w[j] = g[j] = 1.f;
      if (p.w_post) load_vec<T>(p.w_post, size_t(v) * VN, w);
      if (p.gate) load_vec<T>(p.gate, gate_base + v * VN, g);
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        r[i][j] = p.scale * r[i][j] + g[j] * (y[i][j] * rstd1 * w[j]);
        q[0] += r[i][j] * r[i][j];
      }
      store_vec<T>(p.r, base + v * VN, r[i]);
    }
    if (!p.w_pre) continue;
    block_sum<1>(q, scratch);
    const float rstd2 = rsqrtf(q[0] / p.d + p.eps);
    if (threadIdx.x == 0) p.rstd_pre[row] = rstd2;
#pragma unroll
    for (int i = 0; i < RN_VECS; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= nvec) continue;
      float w[VN];
      load_vec<T>(p.w_pre, size_t(v) * VN, w);
#pragma unroll
      for (int j = 0; j < VN; ++j) w[j] *= r[i][j] * rstd2;
      store_vec<T>(p.h, base + v * VN, w);
    }
  }
}

// A unit is a run of rows that share a gate row; a CTA takes units in turn.  The sums for the gate leave with each unit (as
// the result, where a unit is a whole group), those for the weights when the CTA is done.
template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_bwd_kernel(const __grid_constant__ ResNormParams p) {
  constexpr int VN = Vec<T>::N;
  __shared__ float scratch[64];
  const int nvec = p.d / VN;
  float* part_post = p.scratch;
  float* part_pre = part_post + size_t(gridDim.x) * p.d;
  float* part_gate = part_pre + size_t(gridDim.x) * p.d;
  float a_post[RN_VECS][VN], a_pre[RN_VECS][VN], a_gate[RN_VECS][VN];
#pragma unroll
  for (int i = 0; i < RN_VECS; ++i)
#pragma unroll
    for (int j = 0; j < VN; ++j) a_post[i][j] = a_pre[i][j] = 0.f;
  const long long units = (long long)p.groups * p.chunks;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long group = unit / p.chunks, chunk = unit - group * p.chunks;
    const long long first = group * p.group_rows + p.group_rows * chunk / p.chunks;
    const long long last = group * p.group_rows + p.group_rows * (chunk + 1) / p.chunks;
#pragma unroll
    for (int i = 0; i < RN_VECS; ++i)
#pragma unroll
      for (int j = 0; j < VN; ++j) a_gate[i][j] = 0.f;
    for (long long row = first; row < last; ++row) {
      const size_t base = size_t(row) * p.d;
      const float rstd1 = p.w_post ? p.rstd_post[row] : 1.f;
      const bool pre = p.w_pre && p.dh;
      const float rstd2 = pre ? p.rstd_pre[row] : 0.f;
      float s[1] = {0.f};
      float P[RN_VECS][VN], G[RN_VECS][VN], W[RN_VECS][VN], hat[RN_VECS][VN], u[RN_VECS][VN];
#pragma unroll
      for (int i = 0; i < RN_VECS; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) continue;
#pragma unroll
        for (int j = 0; j < VN; ++j) { G[i][j] = W[i][j] = 1.f; u[i][j] = 0.f; hat[i][j] = 0.f; }
        load_vec<T>(p.y, base + v * VN, P[i]);
        if (p.w_post) load_vec<T>(p.w_post, size_t(v) * VN, W[i]);
        if (p.gate) load_vec<T>(p.gate, size_t(group) * p.d + v * VN, G[i]);
#pragma unroll
        for (int j = 0; j < VN; ++j) P[i][j] *= rstd1;
        if (pre) {
          float w[VN];
          load_vec<T>(p.x, base + v * VN, hat[i]);
          load_vec<T>(p.dh, base + v * VN, u[i]);
          load_vec<T>(p.w_pre, size_t(v) * VN, w);
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            hat[i][j] = (p.scale * hat[i][j] + G[i][j] * (P[i][j] * W[i][j])) * rstd2;
            a_pre[i][j] += u[i][j] * hat[i][j];
            u[i][j] *= w[j];
            s[0] += u[i][j] * hat[i][j];
          }
        }
      }
      if (pre) block_sum<1>(s, scratch);
      const float mean1 = s[0] / p.d;
      float q[1] = {0.f};
#pragma unroll
      for (int i = 0; i < RN_VECS; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) continue;
        float dR[VN], o[VN];
#pragma unroll
        for (int j = 0; j < VN; ++j) dR[j] = 0.f;
        if (p.dr) load_vec<T>(p.dr, base + v * VN, dR);
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          dR[j] += rstd2 * (u[i][j] - hat[i][j] * mean1);
          o[j] = p.scale * dR[j];
          a_gate[i][j] += dR[j] * (P[i][j] * W[i][j]);
          const float dn = dR[j] * G[i][j];
          a_post[i][j] += dn * P[i][j];
          u[i][j] = dn * W[i][j];            // from here on v
          q[0] += u[i][j] * P[i][j];
        }
        store_vec<T>(p.dx, base + v * VN, o);
      }
      float mean2 = 0.f;
      if (p.w_post) {
        block_sum<1>(q, scratch);
        mean2 = q[0] / p.d;
      }
#pragma unroll
      for (int i = 0; i < RN_VECS; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) continue;
        float o[VN];
#pragma unroll
        for (int j = 0; j < VN; ++j) o[j] = rstd1 * (u[i][j] - P[i][j] * mean2);
        store_vec<T>(p.dy, base + v * VN, o);
      }
    }
    if (p.gate) {
#pragma unroll
      for (int i = 0; i < RN_VECS; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) continue;
        if (p.chunks == 1 && !p.wide) store_vec<T>(p.dgate, size_t(group) * p.d + v * VN, a_gate[i]);
        else {
          float* to = (p.chunks == 1 ? static_cast<float*>(p.dgate) + size_t(group) * p.d : part_gate + size_t(unit) * p.d) + v * VN;
#pragma unroll
          for (int j = 0; j < VN; ++j) to[j] = a_gate[i][j];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RN_VECS; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v >= nvec) continue;
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      if (p.w_post) part_post[size_t(blockIdx.x) * p.d + v * VN + j] = a_post[i][j];
      if (p.w_pre) part_pre[size_t(blockIdx.x) * p.d + v * VN + j] = a_pre[i][j];
    }
  }
}

// Sums of partial rows: blockIdx.y 0 and 1 the weights' (`parts` rows each), 2 + g the gate's group g (`chunks` rows).  A CTA
// owns 32 columns, its warps every 8th row, four loads in flight each; the eight sums meet in shared memory.
template <typename T>
__global__ void __launch_bounds__(256) residual_norm_sums_kernel(const float* scratch, void* dw_post, void* dw_pre, void* dgate, int parts,
                                                                 int chunks, int d, int wide) {
  __shared__ float red[8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  const int which = blockIdx.y;
  void* out = which == 0 ? dw_post : which == 1 ? dw_pre : dgate;
  if (out == nullptr) return;      // the same for the whole CTA
  const int n = which < 2 ? parts : chunks;
  const size_t at = which < 2 ? size_t(which) * parts * d : (size_t(2) * parts + size_t(which - 2) * chunks) * d;
  const size_t out_at = which < 2 ? 0 : size_t(which - 2) * d;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < d) {
    const float* s = scratch + at + c;
    int i = ry;
    for (; i + 24 < n; i += 32) {
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] += s[size_t(i + 8 * k) * d];
    }
    for (; i < n; i += 8) a[0] += s[size_t(i) * d];
  }
  red[ry][cx] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (ry == 0 && c < d) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += red[k][cx];
    if (wide) static_cast<float*>(out)[out_at + c] = v;
    else static_cast<T*>(out)[out_at + c] = from_f<T>(v);
  }
}

static int rn_sms() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}
static int rn_threads(int d, int vn) {
  const int t = (d / vn + RN_VECS - 1) / RN_VECS;
  return t <= 32 ? 32 : (t + 31) / 32 * 32;
}
struct RnPlan {
  int grid, chunks;
};
// CTAs of the backward, and the units that a group's rows are cut into: about as many units as CTAs.
static RnPlan rn_bwd_plan(long long rows, int d, int groups, int vn) {
  const int threads = rn_threads(d, vn);
  const int per_sm = threads >= 512 ? 1 : 512 / threads < 8 ? 512 / threads : 8;
  const long long want = (long long)rn_sms() * per_sm;
  const long long group_rows = groups ? rows / groups : 0;
  long long chunks = groups ? want / groups : 1;
  if (chunks > group_rows) chunks = group_rows;
  if (chunks < 1) chunks = 1;
  const long long units = groups * chunks;
  return {int(units < want ? units : want), int(chunks)};
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
    if (d <= 0 || d % VN || d / VN > RN_VECS * 1024 || groups < 1 || rows % groups || !rn_aligned({x, y, w_post, gate, w_pre, r, h}))
      return -int(JPB_ERR_BAD_ARGUMENT);
    ResNormParams p = {};
    p.x = x; p.y = y; p.w_post = w_post; p.gate = gate; p.w_pre = w_pre; p.r = r; p.h = h;
    p.rstd_post = rstd_post; p.rstd_pre = rstd_pre; p.rows = rows; p.d = d; p.group_rows = rows / groups;
    p.scale = scale; p.eps = eps;
    const int threads = rn_threads(d, VN);
    const long long most = (long long)rn_sms() * (2048 / threads < 16 ? 2048 / threads : 16);
    residual_norm_fwd_kernel<T><<<int(rows < most ? rows : most), threads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return int(cudaGetLastError());
  });
}

// fp32 elements of scratch for jpb_residual_norm_bwd.
JPB_API long long jpb_residual_norm_bwd_scratch_elems(int dt, long long rows, int d, int groups) {
  const jpb::RnPlan plan = jpb::rn_bwd_plan(rows, d, groups, dt == 0 ? 4 : 8);
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
    if (rows < 0 || d <= 0 || d % VN || d / VN > RN_VECS * 1024 || groups < 1 || rows % groups ||
        !rn_aligned({dr, dh, x, y, w_post, gate, w_pre, dx, dy, dgate}))
      return -int(JPB_ERR_BAD_ARGUMENT);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const RnPlan plan = rn_bwd_plan(rows, d, groups, VN);
    ResNormParams p = {};
    p.x = x; p.y = y; p.w_post = w_post; p.gate = gate; p.w_pre = w_pre;
    p.rstd_post = const_cast<float*>(rstd_post); p.rstd_pre = const_cast<float*>(rstd_pre);
    p.dr = dr; p.dh = dh; p.dx = dx; p.dy = dy; p.scratch = scratch; p.rows = rows; p.d = d; p.group_rows = rows / groups;
    p.groups = groups; p.chunks = plan.chunks; p.dgate = dgate; p.wide = wide; p.scale = scale;
    residual_norm_bwd_kernel<T><<<plan.grid, rn_threads(d, VN), 0, s>>>(p);
    const bool gate_sums = gate && plan.chunks > 1;
    if (w_post || w_pre || gate_sums)
      residual_norm_sums_kernel<T><<<dim3((d + 31) / 32, gate_sums ? 2 + groups : 2), 256, 0, s>>>(
          scratch, w_post ? dw_post : nullptr, w_pre ? dw_pre : nullptr, gate_sums ? dgate : nullptr, plan.grid, plan.chunks, d, wide);
    return int(cudaGetLastError());
  });
}
