// Layer norm over the channels of pixel rows, forward and backward with the gradients of gamma and beta.
//
//   y = xhat * gamma + beta,  xhat = (x - mu) * rstd,  rstd = (mean (x - mu)^2 + eps)^-1/2
//   gx = rstd * (g - mean g - xhat * mean(g * xhat)),  g = gout * gamma;   dgamma = sum_rows gout * xhat;  dbeta = sum_rows gout
//
// The statistics, the row sums and the parameter sums are fp32; the variance is the mean of squared differences from the mean already
// formed (no E[x^2] - mu^2 cancellation), the result is rounded once.
#include "myolo_dev.h"

namespace {

struct Rows {              // the pixel rows of a view, numbered n-major
  char* p;
  int64_t sn, sh, sw;      // bytes
  int w, hw;
  int flat;                // the rows are evenly spaced: one stride (sw) reaches them all
};
Rows rows_of(const myolo_tensor& t) {
  const int64_t es = t.dtype == MYOLO_F16 ? 2 : 4;
  Rows r{(char*)t.ptr, t.sn * es, t.sh * es, t.sw * es, t.w, 0, 0};
  r.flat = (t.h == 1 || t.sh == (int64_t)t.w * t.sw) && (t.n == 1 || (t.h == 1 ? t.sn == (int64_t)t.w * t.sw : t.sn == (int64_t)t.h * t.sh));
  r.hw = t.h * t.w;
  return r;
}
template <typename T> __device__ __forceinline__ T* row_ptr(const Rows& t, int64_t r) {
  if (t.flat) return (T*)(t.p + r * t.sw);
  const int64_t n = r / t.hw;
  const int q = (int)(r - n * t.hw);
  const int y = q / t.w;
  return (T*)(t.p + n * t.sn + (int64_t)y * t.sh + (int64_t)(q - y * t.w) * t.sw);
}

// VEC consecutive elements as floats: one 16-byte access (VEC = ET<T>::SEG) or element by element (VEC = 1: odd counts, odd alignment)
template <typename T, int VEC> __device__ __forceinline__ void ldv(const T* p, float* f) {
  if constexpr (VEC == 1) f[0] = (float)p[0];
  else Vec<T>::unpack(ldg16(p), f);
}
template <typename T, int VEC> __device__ __forceinline__ void stv(T* p, const float* f) {
  if constexpr (VEC == 1) p[0] = (T)f[0];
  else stg16(p, Vec<T>::pack(f));
}

template <int NT> __device__ __forceinline__ float block_sum(float v, float* sm) {
  v = wave_sum(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += sm[i];
  return s;
}

// one workgroup a row, the row read again for every pass (any channel count)
template <typename T, int VEC>
__global__ __launch_bounds__(256) void ln_fwd_any_kernel(Rows x, Rows o, int64_t rows, int c, const float* gamma, const float* beta, float eps,
                                                         float* saved) {
  __shared__ float sm[4];
  const float rc = 1.f / (float)c;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xp = row_ptr<T>(x, r);
    T* op = row_ptr<T>(o, r);
    float f[VEC], s = 0.f;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += f[e];
    }
    const float mu = block_sum<256>(s, sm) * rc;
    s = 0.f;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += (f[e] - mu) * (f[e] - mu);
    }
    const float rstd = 1.f / sqrtf(block_sum<256>(s, sm) * rc + eps);
    if (saved && threadIdx.x == 0) { saved[r] = mu; saved[rows + r] = rstd; }
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = (f[e] - mu) * rstd * (gamma ? gamma[i + e] : 1.f) + (beta ? beta[i + e] : 0.f);
      stv<T, VEC>(op + i, f);
    }
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void ln_bwd_any_kernel(Rows go, Rows x, Rows gx, int64_t rows, int c, const float* saved, const float* gamma,
                                                         int acc) {
  __shared__ float sm[4];
  const float rc = 1.f / (float)c;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xp = row_ptr<T>(x, r);
    const T* gp = row_ptr<T>(go, r);
    T* op = row_ptr<T>(gx, r);
    const float mu = saved[r], rstd = saved[rows + r];
    float f[VEC], g[VEC], s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
      ldv<T, VEC>(gp + i, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = g[e] * (gamma ? gamma[i + e] : 1.f);
        s1 += v;
        s2 += v * ((f[e] - mu) * rstd);
      }
    }
    s1 = block_sum<256>(s1, sm) * rc;
    s2 = block_sum<256>(s2, sm) * rc;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
      ldv<T, VEC>(gp + i, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = rstd * (g[e] * (gamma ? gamma[i + e] : 1.f) - s1 - (f[e] - mu) * rstd * s2);
      if (acc) {
        ldv<T, VEC>(op + i, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] += g[e];
      }
      stv<T, VEC>(op + i, f);
    }
  }
}

// parameter sums of one slice of the rows: a workgroup owns 64 channels, its four waves take every fourth row of the slice
template <typename T>
__global__ __launch_bounds__(256) void ln_param_any_kernel(Rows go, Rows x, int64_t rows, int c, const float* saved, float* ws) {
  __shared__ float sm[2][4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int ch = blockIdx.x * 64 + lane;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = per * blockIdx.y, r1 = r0 + per < rows ? r0 + per : rows;
  float dg = 0.f, db = 0.f;
  if (ch < c)
    for (int64_t r = r0 + wv; r < r1; r += 4) {
      const float g = (float)row_ptr<T>(go, r)[ch];
      dg += g * (((float)row_ptr<T>(x, r)[ch] - saved[r]) * saved[rows + r]);
      db += g;
    }
  sm[0][wv][lane] = dg;
  sm[1][wv][lane] = db;
  __syncthreads();
  if (wv < 2 && ch < c)
    ws[((int64_t)blockIdx.y * 2 + wv) * c + ch] = (sm[wv][0][lane] + sm[wv][1][lane]) + (sm[wv][2][lane] + sm[wv][3][lane]);
}

// ws [n][2][c] -> dgamma, dbeta: 16 channels x 16 slices of the partial rows a workgroup, combined in a fixed order
__global__ __launch_bounds__(256) void ln_param_reduce_kernel(const float* ws, int n, int c, float* dgamma, float* dbeta, int acc) {
  __shared__ float sm[16][17];
  const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + cl;                  // 0 .. 2c: gamma's channels, then beta's
  float s = 0.f;
  if (col < 2 * c)
    for (int i = sl; i < n; i += 16) s += ws[(int64_t)i * 2 * c + col];
  sm[sl][cl] = s;
  __syncthreads();
  if (sl == 0 && col < 2 * c) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sm[i][cl];
    float* d = col < c ? dgamma : dbeta;
    if (d) {
      d += col < c ? col : col - c;
      *d = acc ? *d + s : s;
    }
  }
}

constexpr int kSlices = 256;

bool view_ok(const myolo_tensor& t) {
  return (t.ptr || (int64_t)t.n * t.h * t.w == 0) && (t.dtype == MYOLO_F16 || t.dtype == MYOLO_F32) && t.n >= 0 && t.h >= 0 && t.w >= 0 && t.c >= 1 &&
         (int64_t)t.h * t.w < (1ll << 31) && (double)t.n * t.h * t.w < (double)(1ll << 40);
         // (rows of a map: 31 bits; all rows: 40)
}
bool same_shape(const myolo_tensor& a, const myolo_tensor& b) {
  return a.n == b.n && a.h == b.h && a.w == b.w && a.c == b.c && a.dtype == b.dtype;
}
bool vec_ok(const myolo_tensor& t) {
  const int seg = t.dtype == MYOLO_F16 ? 8 : 4;
  return t.c % seg == 0 && (uintptr_t)t.ptr % 16 == 0 && t.sn % seg == 0 && t.sh % seg == 0 && t.sw % seg == 0;
}

template <typename T>
int ln_fwd(const myolo_tensor* x, const float* gamma, const float* beta, float eps, const myolo_tensor* out, float* saved, hipStream_t st) {
  const int64_t rows = (int64_t)x->n * x->h * x->w;
  const Rows rx = rows_of(*x), ro = rows_of(*out);
  const int grid = (int)(rows < 65536 ? rows : 65536);
  if (vec_ok(*x) && vec_ok(*out))
    hipLaunchKernelGGL((ln_fwd_any_kernel<T, ET<T>::SEG>), dim3(grid), dim3(256), 0, st, rx, ro, rows, x->c, gamma, beta, eps, saved);
  else
    hipLaunchKernelGGL((ln_fwd_any_kernel<T, 1>), dim3(grid), dim3(256), 0, st, rx, ro, rows, x->c, gamma, beta, eps, saved);
  MYOLO_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int ln_bwd(const myolo_tensor* gout, const myolo_tensor* x, const float* saved, const float* gamma, const myolo_tensor* gx, int acc_x,
           float* dgamma, float* dbeta, int acc_params, float* ws, hipStream_t st) {
  const int64_t rows = (int64_t)x->n * x->h * x->w;
  const Rows rx = rows_of(*x), rg = rows_of(*gout);
  if (dgamma || dbeta) {
    const int ns = (int)(rows < kSlices ? rows : kSlices);
    if (ns) {
      hipLaunchKernelGGL((ln_param_any_kernel<T>), dim3((x->c + 63) / 64, ns), dim3(256), 0, st, rg, rx, rows, x->c, saved, ws);
      MYOLO_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(ln_param_reduce_kernel, dim3((2 * x->c + 15) / 16), dim3(256), 0, st, ws, ns, x->c, dgamma, dbeta, acc_params);
    MYOLO_CHECK_LAUNCH();
  }
  if (gx && rows) {
    const Rows ro = rows_of(*gx);
    const int grid = (int)(rows < 65536 ? rows : 65536);
    if (vec_ok(*x) && vec_ok(*gout) && vec_ok(*gx))
      hipLaunchKernelGGL((ln_bwd_any_kernel<T, ET<T>::SEG>), dim3(grid), dim3(256), 0, st, rg, rx, ro, rows, x->c, saved, gamma, acc_x);
    else
      hipLaunchKernelGGL((ln_bwd_any_kernel<T, 1>), dim3(grid), dim3(256), 0, st, rg, rx, ro, rows, x->c, saved, gamma, acc_x);
    MYOLO_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" int myolo_layernorm_fwd(const myolo_tensor* x, const float* gamma, const float* beta, float eps, const myolo_tensor* out,
                                   float* saved, void* stream) {
  if (!x || !out || !view_ok(*x) || !view_ok(*out) || !same_shape(*x, *out) || !(eps >= 0.f)) return MYOLO_EINVAL;
  if ((int64_t)x->n * x->h * x->w == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  return x->dtype == MYOLO_F16 ? ln_fwd<half_t>(x, gamma, beta, eps, out, saved, st) : ln_fwd<float>(x, gamma, beta, eps, out, saved, st);
}

extern "C" int64_t myolo_layernorm_ws_bytes(int64_t rows, int c) {
  if (rows <= 0 || c <= 0) return 0;
  return (rows < kSlices ? rows : kSlices) * 2 * (int64_t)c * 4;
}

extern "C" int myolo_layernorm_bwd(const myolo_tensor* gout, const myolo_tensor* x, const float* saved, const float* gamma,
                                   const myolo_tensor* gx, int acc_x, float* dgamma, float* dbeta, int acc_params, float* ws,
                                   int64_t ws_bytes, void* stream) {
  if (!gout || !x || !view_ok(*x) || !view_ok(*gout) || !same_shape(*x, *gout)) return MYOLO_EINVAL;
  const int64_t rows = (int64_t)x->n * x->h * x->w;
  if (rows && !saved) return MYOLO_EINVAL;
  if (gx && !gx->ptr) gx = nullptr;       // (also: no rows)
  if (gx && (!view_ok(*gx) || !same_shape(*x, *gx))) return MYOLO_EINVAL;
  if ((dgamma || dbeta) && rows && (!ws || (uintptr_t)ws % 16 || ws_bytes < myolo_layernorm_ws_bytes(rows, x->c))) return MYOLO_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return x->dtype == MYOLO_F16 ? ln_bwd<half_t>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st)
                               : ln_bwd<float>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st);
}
