// Layer norm over the last dimension, any width, forward and backward.
//
//   y  = (x - mu) r w + b,           mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = r (u - mean(u) - h mean(u h)),   u = g w,  h = (x - mu) r
//   dw = sum over rows of g h,       db = sum over rows of g
//
// Bound by memory: x in and y out (backward: x, g in, dx out) once each. A row lives in the
// registers of its group of TPR threads (a part of a warp up to 512 elements, a block up to
// 8192), so the two-pass variance costs no second read; all statistics and sums are fp32.
// Each thread owns the same columns of every row it meets, so the weight and bias stay in
// registers and the backward's dw / db are per-thread sums: reduced per block, written as
// one partial row per block, and added up over the blocks in a fixed order by a second
// kernel -- no atomics, the same bits on every run. Elements per thread stay at 16 or less
// (five such arrays in the backward), which keeps 64 to 128 registers and 2-4 blocks per SM.
// Loads are 16 bytes where width, stride and pointers allow it, else 4 bytes or one element.
// Widths beyond 8192 take a plain block-per-row loop that re-reads the row from cache.
#include "ftm_kernels.h"

namespace ftm {
namespace {

constexpr int kLnThreads = 256;    // block of the warp-row kernels
constexpr int kLnMaxReg = 8192;    // widest row held in registers
constexpr int kLnMaxWidth = (1 << 30) - 1024;   // columns of dw and db together are counted in 32 bits

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// element `c` of a parameter vector of any supported type
__device__ __forceinline__ float param_at(const void* p, int dtype, int c) {
  if (dtype == FTM_F32) return static_cast<const float*>(p)[c];
  if (dtype == FTM_F16) return __half2float(static_cast<const __half*>(p)[c]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
}
__device__ __forceinline__ void param_set(void* p, int dtype, int c, float v) {
  if (dtype == FTM_F32) static_cast<float*>(p)[c] = v;
  else if (dtype == FTM_F16) static_cast<__half*>(p)[c] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
}

// Sums of K values over the TPR threads of a row group; every thread gets them. Groups
// wider than a warp are whole blocks (`red` is their scratch, one row per use so that
// two uses in a row need no extra barrier).
template <int TPR, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float (*red)[K]) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (TPR > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[threadIdx.x >> 5][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) v[k] += red[w][k];
    }
  }
}

template <typename T, int VEC, int TPR, int ITER, int R>
__global__ void __launch_bounds__(TPR > 32 ? TPR : kLnThreads)
ln_fwd_kernel(const T* __restrict__ x, long long xs, const void* __restrict__ w, int wdt,
              const void* __restrict__ b, int bdt, float eps, T* __restrict__ y,
              float2* __restrict__ stats, long long rows, int width) {
  constexpr int kBlock = TPR > 32 ? TPR : kLnThreads;
  constexpr int kGroups = kBlock / TPR;
  using P = Pack<T, VEC>;
  __shared__ float red[TPR > 32 ? TPR / 32 : 1][R];
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const float inv = 1.0f / static_cast<float>(width);
  grid_dep_wait();
  float wv[ITER][VEC], bv[ITER][VEC];
#pragma unroll
  for (int i = 0; i < ITER; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = (i * TPR + t) * VEC + e;
      wv[i][e] = (w && c < width) ? param_at(w, wdt, c) : 1.f;
      bv[i][e] = (b && c < width) ? param_at(b, bdt, c) : 0.f;
    }
  // the loop bound is the same for every group of a block: group_sum has barriers
  for (long long r0 = static_cast<long long>(blockIdx.x) * kGroups * R; r0 < rows;
       r0 += static_cast<long long>(gridDim.x) * kGroups * R) {
    P raw[R][ITER];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const long long r = r0 + q * kGroups + grp;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (r < rows && c < width) raw[q][i] = *reinterpret_cast<const P*>(x + r * xs + c);
        else
#pragma unroll
          for (int e = 0; e < VEC; ++e) raw[q][i].v[e] = from_f<T>(0.f);
      }
    }
    float s[R], d[R], mu[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      s[q] = 0.f;
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[q] += to_f(raw[q][i].v[e]);
    }
    group_sum<TPR, R>(s, red);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mu[q] = s[q] * inv;
      d[q] = 0.f;
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float k = to_f(raw[q][i].v[e]) - mu[q];
          if ((i * TPR + t) * VEC + e < width) d[q] = fmaf(k, k, d[q]);
        }
    }
    group_sum<TPR, R>(d, red);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const long long r = r0 + q * kGroups + grp;
      if (r >= rows) continue;
      const float rstd = 1.0f / sqrtf(d[q] * inv + eps);
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c >= width) continue;
        P o;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          o.v[e] = from_f<T>(fmaf((to_f(raw[q][i].v[e]) - mu[q]) * rstd, wv[i][e], bv[i][e]));
        *reinterpret_cast<P*>(y + r * width + c) = o;
      }
      if (stats && t == 0) stats[r] = make_float2(mu[q], rstd);
    }
  }
  grid_dep_release();
}

// dx (null: not wanted) and, where `partial` is given, this block's sums of g h and g as
// partial[block][2][width]
template <typename T, int VEC, int TPR, int ITER, int R>
__global__ void __launch_bounds__(TPR > 32 ? TPR : kLnThreads,
                                  (ITER * VEC <= 8 ? 1024 : 512) / (TPR > 32 ? TPR : kLnThreads))
ln_bwd_kernel(const T* __restrict__ x, long long xs, const T* __restrict__ g, long long gs,
              const void* __restrict__ w, int wdt, const float2* __restrict__ stats,
              T* __restrict__ dx, float* __restrict__ partial, long long rows, int width) {
  constexpr int kBlock = TPR > 32 ? TPR : kLnThreads;
  constexpr int kGroups = kBlock / TPR;
  constexpr int E = ITER * VEC;
  using P = Pack<T, VEC>;
  __shared__ float red[TPR > 32 ? TPR / 32 : 1][2 * R];
  __shared__ float sums[TPR > 32 ? 1 : kBlock / 32][TPR > 32 ? 1 : 32 * E];
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const float inv = 1.0f / static_cast<float>(width);
  grid_dep_wait();
  float wv[ITER][VEC], dw[ITER][VEC], db[ITER][VEC];
#pragma unroll
  for (int i = 0; i < ITER; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = (i * TPR + t) * VEC + e;
      wv[i][e] = (w && c < width) ? param_at(w, wdt, c) : 1.f;
      dw[i][e] = db[i][e] = 0.f;
    }
  for (long long r0 = static_cast<long long>(blockIdx.x) * kGroups * R; r0 < rows;
       r0 += static_cast<long long>(gridDim.x) * kGroups * R) {
    P xr[R][ITER], gr[R][ITER];
    float2 st[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const long long r = r0 + q * kGroups + grp;
      st[q] = r < rows ? stats[r] : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (r < rows && c < width) {
          xr[q][i] = *reinterpret_cast<const P*>(x + r * xs + c);
          gr[q][i] = *reinterpret_cast<const P*>(g + r * gs + c);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) xr[q][i].v[e] = gr[q][i].v[e] = from_f<T>(0.f);
        }
      }
    }
    float s[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      s[2 * q] = s[2 * q + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          // columns past the row and rows past the end hold g = 0: they add nothing
          const float gv = to_f(gr[q][i].v[e]);
          const float h = (to_f(xr[q][i].v[e]) - st[q].x) * st[q].y;
          const float u = gv * wv[i][e];
          s[2 * q] += u;
          s[2 * q + 1] = fmaf(u, h, s[2 * q + 1]);
          dw[i][e] = fmaf(gv, h, dw[i][e]);
          db[i][e] += gv;
        }
    }
    if (dx == nullptr) continue;
    group_sum<TPR, 2 * R>(s, red);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const long long r = r0 + q * kGroups + grp;
      if (r >= rows) continue;
      const float m1 = s[2 * q] * inv, m2 = s[2 * q + 1] * inv;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c >= width) continue;
        P o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = (to_f(xr[q][i].v[e]) - st[q].x) * st[q].y;
          o.v[e] = from_f<T>(st[q].y * (to_f(gr[q][i].v[e]) * wv[i][e] - m1 - h * m2));
        }
        *reinterpret_cast<P*>(dx + r * width + c) = o;
      }
    }
  }
  if (partial) {
    float* out = partial + static_cast<size_t>(blockIdx.x) * 2 * width;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (TPR > 32) {
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int c = (i * TPR + t) * VEC + e;
            if (c < width) out[half * width + c] = half ? db[i][e] : dw[i][e];
          }
      } else {
        // groups of one warp by shuffles, then the block's warps in order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float a = half ? db[i][e] : dw[i][e];
#pragma unroll
            for (int o = 16; o >= TPR; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            if ((threadIdx.x & 31) < TPR) sums[threadIdx.x >> 5][(i * TPR + t) * VEC + e] = a;
          }
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += kBlock) {
          float a = 0.f;
#pragma unroll
          for (int k = 0; k < kBlock / 32; ++k) a += sums[k][c];
          out[half * width + c] = a;
        }
      }
    }
  }
  grid_dep_release();
}

// dw / db = sums of the blocks' partials, in block order within each of 32 interleaved
// runs and then over the runs: the same order on every call
__global__ void __launch_bounds__(1024)
ln_reduce_kernel(const float* __restrict__ partial, int blocks, int width, void* __restrict__ dw,
                 int dwt, void* __restrict__ db, int dbt) {
  __shared__ float red[32][33];
  grid_dep_wait();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float a = 0.f;
  if (c < 2 * width) {
#pragma unroll 4
    for (int k = threadIdx.y; k < blocks; k += 32) a += partial[static_cast<size_t>(k) * 2 * width + c];
  }
  red[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  a = red[threadIdx.x][threadIdx.y];   // a warp now holds the 32 runs of one column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < 2 * width) {
    if (col < width) {
      if (dw) param_set(dw, dwt, col, a);
    } else if (db) {
      param_set(db, dbt, col - width, a);
    }
  }
  grid_dep_release();
}

// ------------------------------------------------- rows wider than the register kernels
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int k = 0; k < static_cast<int>(blockDim.x >> 5); ++k) v += red[k];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(512)
ln_fwd_wide_kernel(const T* __restrict__ x, long long xs, const void* __restrict__ w, int wdt,
                   const void* __restrict__ b, int bdt, float eps, T* __restrict__ y,
                   float2* __restrict__ stats, long long rows, int width) {
  __shared__ float red[16];
  grid_dep_wait();
  const float inv = 1.0f / static_cast<float>(width);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * xs;
    float s = 0.f, d = 0.f;
    for (int c = threadIdx.x; c < width; c += blockDim.x) s += to_f(row[c]);
    const float mu = block_sum(s, red) * inv;
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      const float k = to_f(row[c]) - mu;
      d = fmaf(k, k, d);
    }
    const float rstd = 1.0f / sqrtf(block_sum(d, red) * inv + eps);
    for (int c = threadIdx.x; c < width; c += blockDim.x)
      y[r * width + c] = from_f<T>(fmaf((to_f(row[c]) - mu) * rstd, w ? param_at(w, wdt, c) : 1.f,
                                        b ? param_at(b, bdt, c) : 0.f));
    if (stats && threadIdx.x == 0) stats[r] = make_float2(mu, rstd);
  }
  grid_dep_release();
}

template <typename T>
__global__ void __launch_bounds__(512)
ln_bwd_wide_kernel(const T* __restrict__ x, long long xs, const T* __restrict__ g, long long gs,
                   const void* __restrict__ w, int wdt, const float2* __restrict__ stats,
                   T* __restrict__ dx, float* __restrict__ partial, long long rows, int width) {
  __shared__ float red[16];
  grid_dep_wait();
  const float inv = 1.0f / static_cast<float>(width);
  if (partial)
    for (int c = threadIdx.x; c < 2 * width; c += blockDim.x)
      partial[static_cast<size_t>(blockIdx.x) * 2 * width + c] = 0.f;
  __syncthreads();   // the sums' columns are dealt to the threads in another order
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    const T* gr = g + r * gs;
    const float2 st = stats[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      const float gv = to_f(gr[c]), h = (to_f(xr[c]) - st.x) * st.y;
      const float u = gv * (w ? param_at(w, wdt, c) : 1.f);
      s1 += u;
      s2 = fmaf(u, h, s2);
      if (partial) {   // a column always belongs to the same thread of its block
        float* p = partial + static_cast<size_t>(blockIdx.x) * 2 * width;
        p[c] = fmaf(gv, h, p[c]);
        p[width + c] += gv;
      }
    }
    if (dx == nullptr) continue;
    const float m1 = block_sum(s1, red) * inv;
    const float m2 = block_sum(s2, red) * inv;
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      const float h = (to_f(xr[c]) - st.x) * st.y;
      dx[r * width + c] =
          from_f<T>(st.y * (to_f(gr[c]) * (w ? param_at(w, wdt, c) : 1.f) - m1 - h * m2));
    }
  }
  grid_dep_release();
}

// ------------------------------------------------------------------------- dispatch
struct LnArgs {
  const void* x; long long xs;
  const void* g; long long gs;
  const void* w; int wdt;
  const void* b; int bdt;
  float eps;
  void* out;          // y or dx
  float2* stats;
  float* partial;
  long long rows; int width;
  int sms;
  cudaStream_t stream;
  int blocks;         // set by the backward: rows of `partial`
};

int ln_sms() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Blocks of a launch: enough to fill the GPU (about 2048 threads per SM forward, 1024
// backward, whose registers allow no more), never more than there are row groups.
int ln_blocks(long long rows, int groups_rows, int block, int sms, bool bwd) {
  const long long need = (rows + groups_rows - 1) / groups_rows;
  const long long cap = static_cast<long long>(sms) * (bwd ? 1024 : 2048) / block;
  return static_cast<int>(need < cap ? need : cap);
}

template <typename T, int VEC, int TPR, int ITER>
cudaError_t ln_go(LnArgs& a, bool bwd) {
  constexpr int E = VEC * ITER;
  constexpr int kBlock = TPR > 32 ? TPR : kLnThreads;
  // rows in flight per group: 1048576 x 128 bf16 forward took 131 / 112 / 109 us with 1 / 2 / 4
  // rows (4.9 TB/s); backward 159 us with one row in 64 registers and four blocks per SM
  // (5.1 TB/s) against 212 and 398 us with 2 and 4 rows, whose registers spill
  constexpr int RF = TPR > 32 ? (E <= 8 ? 2 : 1) : (E <= 2 ? 4 : E <= 8 ? 4 : 2);
  constexpr int RB = 1;
  if (!bwd) {
    const int blocks = ln_blocks(a.rows, kBlock / TPR * RF, kBlock, a.sms, false);
    return launch_pdl(ln_fwd_kernel<T, VEC, TPR, ITER, RF>, dim3(blocks), dim3(kBlock), 0, a.stream,
                      nullptr, 0, static_cast<const T*>(a.x), a.xs, a.w, a.wdt, a.b, a.bdt, a.eps,
                      static_cast<T*>(a.out), a.stats, a.rows, a.width);
  }
  a.blocks = ln_blocks(a.rows, kBlock / TPR * RB, kBlock, a.sms, true);
  return launch_pdl(ln_bwd_kernel<T, VEC, TPR, ITER, RB>, dim3(a.blocks), dim3(kBlock), 0, a.stream,
                    nullptr, 0, static_cast<const T*>(a.x), a.xs, static_cast<const T*>(a.g), a.gs,
                    a.w, a.wdt, static_cast<const float2*>(a.stats), static_cast<T*>(a.out), a.partial,
                    a.rows, a.width);
}

// Row groups by width: a part of a warp, a warp, then blocks of 128 to 512 threads, with
// at most 16 elements per thread.
template <typename T, int VEC>
cudaError_t ln_width(LnArgs& a, bool bwd) {
  constexpr int I8 = VEC >= 8 ? 1 : 8 / VEC, I16 = 16 / VEC;
  const int w = a.width;
  if (VEC >= 4 && w <= 8 * VEC) return ln_go<T, VEC, 8, 1>(a, bwd);
  if (VEC >= 4 && w <= 16 * VEC) return ln_go<T, VEC, 16, 1>(a, bwd);
  if (w <= 32 * VEC) return ln_go<T, VEC, 32, 1>(a, bwd);
  if (VEC <= 2 && w <= 128) return ln_go<T, VEC, 32, VEC == 1 ? 4 : 2>(a, bwd);
  if (w <= 256) return ln_go<T, VEC, 32, I8>(a, bwd);
  if (w <= 512) return ln_go<T, VEC, 32, I16>(a, bwd);
  if (w <= 1024) return ln_go<T, VEC, 128, I8>(a, bwd);
  if (w <= 2048) return ln_go<T, VEC, 128, I16>(a, bwd);
  if (w <= 4096) return ln_go<T, VEC, 256, I16>(a, bwd);
  return ln_go<T, VEC, 512, I16>(a, bwd);
}

template <typename T>
cudaError_t ln_type(LnArgs& a, bool bwd) {
  if (a.width > kLnMaxReg) {
    const long long cap = static_cast<long long>(a.sms) * (bwd ? 2 : 4);
    const int blocks = static_cast<int>(a.rows < cap ? a.rows : cap);
    a.blocks = blocks;
    if (!bwd)
      return launch_pdl(ln_fwd_wide_kernel<T>, dim3(blocks), dim3(512), 0, a.stream, nullptr, 0,
                        static_cast<const T*>(a.x), a.xs, a.w, a.wdt, a.b, a.bdt, a.eps,
                        static_cast<T*>(a.out), a.stats, a.rows, a.width);
    return launch_pdl(ln_bwd_wide_kernel<T>, dim3(blocks), dim3(512), 0, a.stream, nullptr, 0,
                      static_cast<const T*>(a.x), a.xs, static_cast<const T*>(a.g), a.gs, a.w, a.wdt,
                      static_cast<const float2*>(a.stats), static_cast<T*>(a.out), a.partial, a.rows,
                      a.width);
  }
  // the widest loads that width, strides and pointers all allow
  const uint64_t bits = reinterpret_cast<uint64_t>(a.x) | reinterpret_cast<uint64_t>(a.out) |
                        reinterpret_cast<uint64_t>(a.g) |
                        (static_cast<uint64_t>(a.xs) | static_cast<uint64_t>(a.gs) |
                         static_cast<uint64_t>(a.width)) * sizeof(T);
  if (bits % 16 == 0) return ln_width<T, 16 / sizeof(T)>(a, bwd);
  if (sizeof(T) == 2 && bits % 4 == 0) return ln_width<T, 2>(a, bwd);
  return ln_width<T, 1>(a, bwd);
}

cudaError_t ln_run(LnArgs& a, int dtype, bool bwd) {
  if (dtype == FTM_F32) return ln_type<float>(a, bwd);
  if (dtype == FTM_F16) return ln_type<__half>(a, bwd);
  return ln_type<__nv_bfloat16>(a, bwd);
}

bool dt_ok(int d) { return d == FTM_F32 || d == FTM_F16 || d == FTM_BF16; }

bool elem_aligned(const void* p, int dt) {
  return (reinterpret_cast<uintptr_t>(p) & (dt == FTM_F32 ? 3u : 1u)) == 0;
}

}  // namespace
}  // namespace ftm

using namespace ftm;

extern "C" {

size_t ftm_layer_norm_bwd_workspace_bytes(int64_t rows, int32_t width) {
  if (rows < 1 || width < 1 || width > kLnMaxWidth) return 0;
  // at most 1024 / 128 blocks per SM, and never more than rows
  const long long cap = static_cast<long long>(ln_sms()) * 8;
  return static_cast<size_t>(rows < cap ? rows : cap) * 2 * width * sizeof(float);
}

int ftm_layer_norm_fwd(const void* x, int32_t dtype, int64_t x_row_stride, const void* weight,
                       int32_t weight_dtype, const void* bias, int32_t bias_dtype, float eps, void* y,
                       float* stats, int64_t rows, int32_t width, ftm_stream_t stream) {
  if (!x || !y || !(eps >= 0.f)) return FTM_BAD_ARGUMENT;
  if (rows < 1 || width < 1 || width > kLnMaxWidth || x_row_stride < 0) return FTM_BAD_SHAPE;
  if (!dt_ok(dtype) || (weight && !dt_ok(weight_dtype)) || (bias && !dt_ok(bias_dtype)))
    return FTM_BAD_DTYPE;
  if (!elem_aligned(x, dtype) || !elem_aligned(y, dtype) || (stats && (reinterpret_cast<uintptr_t>(stats) & 7)))
    return FTM_BAD_ALIGN;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ftm_device_supported(dev) != 1) return FTM_UNSUPPORTED_ARCH;
  LnArgs a{};
  a.x = x; a.xs = x_row_stride; a.w = weight; a.wdt = weight_dtype; a.b = bias; a.bdt = bias_dtype;
  a.eps = eps; a.out = y; a.stats = reinterpret_cast<float2*>(stats); a.rows = rows; a.width = width;
  a.sms = ln_sms(); a.stream = reinterpret_cast<cudaStream_t>(stream);
  if (ln_run(a, dtype, false) != cudaSuccess) return FTM_LAUNCH_FAILED;
  set_last_launch_count(1);
  return FTM_OK;
}

int ftm_layer_norm_bwd(const void* x, int32_t dtype, int64_t x_row_stride, const void* grad,
                       int64_t grad_row_stride, const void* weight, int32_t weight_dtype,
                       const float* stats, void* dx, void* dweight, void* dbias, int32_t dbias_dtype,
                       void* workspace, size_t workspace_bytes, int64_t rows, int32_t width,
                       ftm_stream_t stream) {
  if (!x || !grad || !stats || (!dx && !dweight && !dbias)) return FTM_BAD_ARGUMENT;
  if (rows < 1 || width < 1 || width > kLnMaxWidth || x_row_stride < 0 || grad_row_stride < 0) return FTM_BAD_SHAPE;
  if (!dt_ok(dtype) || ((weight || dweight) && !dt_ok(weight_dtype)) || (dbias && !dt_ok(dbias_dtype)))
    return FTM_BAD_DTYPE;
  if (!elem_aligned(x, dtype) || !elem_aligned(grad, dtype) || (dx && !elem_aligned(dx, dtype)) ||
      (reinterpret_cast<uintptr_t>(stats) & 7))
    return FTM_BAD_ALIGN;
  const bool sums = dweight || dbias;
  if (sums && (!workspace || workspace_bytes < ftm_layer_norm_bwd_workspace_bytes(rows, width)))
    return FTM_BAD_WORKSPACE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ftm_device_supported(dev) != 1) return FTM_UNSUPPORTED_ARCH;
  LnArgs a{};
  a.x = x; a.xs = x_row_stride; a.g = grad; a.gs = grad_row_stride; a.w = weight; a.wdt = weight_dtype;
  a.out = dx; a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.partial = sums ? static_cast<float*>(workspace) : nullptr; a.rows = rows; a.width = width;
  a.sms = ln_sms(); a.stream = reinterpret_cast<cudaStream_t>(stream);
  if (ln_run(a, dtype, true) != cudaSuccess) return FTM_LAUNCH_FAILED;
  if (sums) {
    if (launch_pdl(ln_reduce_kernel, dim3((2 * width + 31) / 32), dim3(32, 32), 0, a.stream, nullptr, 0,
                   static_cast<const float*>(a.partial), a.blocks, width, dweight, static_cast<int>(weight_dtype),
                   dbias, static_cast<int>(dbias_dtype)) != cudaSuccess)
      return FTM_LAUNCH_FAILED;
  }
  set_last_launch_count(sums ? 2 : 1);
  return FTM_OK;
}

}  // extern "C"
