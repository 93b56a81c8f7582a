// Layer norm over the channels of pixel rows, forward and backward with the gradients of gamma and beta.
//
//   y = xhat * gamma + beta,  xhat = (x - mu) * rstd,  rstd = (mean (x - mu)^2 + eps)^-1/2
//   gx = rstd * (g - mean g - xhat * mean(g * xhat)),  g = gout * gamma;   dgamma = sum_rows gout * xhat;  dbeta = sum_rows gout
//
// The statistics, the row sums and the parameter sums are fp32; the variance is the mean of squared differences from the mean already
// formed (no E[x^2] - mu^2 cancellation), the result is rounded once.  The mean is a true quotient: a constant row whose sum is exact gives
// xhat = 0 exactly (a product with 1/c, contracted into the subtraction, would leave its rounding times rstd).
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
  const float fc = (float)c;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xp = row_ptr<T>(x, r);
    T* op = row_ptr<T>(o, r);
    float f[VEC], s = 0.f;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += f[e];
    }
    const float mu = block_sum<256>(s, sm) / fc;
    s = 0.f;
    for (int i = threadIdx.x * VEC; i < c; i += 256 * VEC) {
      ldv<T, VEC>(xp + i, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += (f[e] - mu) * (f[e] - mu);
    }
    const float rstd = 1.f / sqrtf(block_sum<256>(s, sm) / fc + eps);
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
  const float fc = (float)c;
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
    s1 = block_sum<256>(s1, sm) / fc;
    s2 = block_sum<256>(s2, sm) / fc;
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

// ---- rows held in registers ----------------------------------------------------------------------------------------------------------
// A row belongs to G adjacent lanes (4 .. 64 of a wave, or the whole workgroup of 256), each holding NV vectors of it: x and gout are read once,
// their next row is in flight while this one is reduced and written, gamma / beta and the parameter sums stay in registers over all rows
// of a workgroup.  HBM bound: 131072 rows of 192 fp16 channels forward 21.6 us (4.7 TB/s), backward 34 us (4.4 TB/s; 74 % of the vector
// unit's issue slots), 4 us for the parameter sums; 4097 rows of 1003 fp32 channels, element by element, 9 and 20 us.
template <typename T, int VEC, int NV> struct RowRegs {
  uint4 raw[VEC > 1 ? NV : 1];
  T el[VEC > 1 ? 1 : NV];
  __device__ __forceinline__ void load(const T* p, int t, int g, int c, bool live) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * g + t) * VEC;
      const bool ok = live && col < c;
      if constexpr (VEC > 1) raw[i] = ldg16(ok ? (const char*)(p + col) : zero_page());
      else el[i] = *(const __attribute__((address_space(1))) T*)(ok ? (const char*)(p + col) : zero_page());
    }
  }
  __device__ __forceinline__ void get(int i, float* f) const {
    if constexpr (VEC > 1) Vec<T>::unpack(raw[i], f);
    else f[0] = (float)el[i];
  }
};
template <int VEC, int NV> struct ParamRegs {
  float v[NV * VEC];
  // (16-byte loads where the parameter vector allows them: 4 lanes' worth of scalar loads would outnumber the row's own)
  __device__ __forceinline__ void load(const float* p, int t, int g, int c, float none) {
    const bool al = VEC > 1 && ((uintptr_t)p & 15) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * g + t) * VEC;
      const bool ok = p && col < c;
      if (al) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const uint4 q = ldg16(ok ? (const char*)(p + col + e) : zero_page());
          const float* f = reinterpret_cast<const float*>(&q);
#pragma unroll
          for (int k = 0; k < (VEC > 1 ? 4 : 1); ++k) v[i * VEC + e + k] = p ? f[k] : none;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i * VEC + e] = p ? (ok ? p[col + e] : 0.f) : none;
      }
    }
  }
};
// sums over the 2^glog lanes of a row (WIDE: over the workgroup), both at once, in every lane.  Lane exchanges of the vector unit (quad
// permutes, mirrors of 8 and 16 lanes, row swaps): shuffles through LDS cost ten round trips a row, which is what bounded the backward
// (131072 rows of 192 channels: 42 -> 36 us)
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float swap16_add(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap32_add(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <bool WIDE> __device__ __forceinline__ void row_sums(float& a, float& b, int glog, float* sm) {
  if constexpr (WIDE) {
    a = block_sum<256>(a, sm);
    b = block_sum<256>(b, sm);
    return;
  }
  a = dpp_add<0x4e>(dpp_add<0xb1>(a));                     // (groups have at least 4 lanes)
  b = dpp_add<0x4e>(dpp_add<0xb1>(b));
  if (glog >= 3) { a = dpp_add<0x141>(a); b = dpp_add<0x141>(b); }
  if (glog >= 4) { a = dpp_add<0x140>(a); b = dpp_add<0x140>(b); }
  if (glog >= 5) { a = swap16_add(a); b = swap16_add(b); }
  if (glog >= 6) { a = swap32_add(a); b = swap32_add(b); }
}
template <bool WIDE> __device__ __forceinline__ float row_sum(float v, int glog, float* sm) {
  if constexpr (WIDE) return block_sum<256>(v, sm);
  v = dpp_add<0x4e>(dpp_add<0xb1>(v));
  if (glog >= 3) v = dpp_add<0x141>(v);
  if (glog >= 4) v = dpp_add<0x140>(v);
  if (glog >= 5) v = swap16_add(v);
  if (glog >= 6) v = swap32_add(v);
  return v;
}

template <typename T, int VEC, int NV, bool WIDE>
__global__ __launch_bounds__(256) void ln_fwd_kernel(Rows x, Rows o, int64_t rows, int c, int glog, const float* gamma, const float* beta, float eps,
                                                     float* saved) {
  __shared__ float sm[4];
  const int g = WIDE ? 256 : 1 << glog, t = WIDE ? threadIdx.x : threadIdx.x & (g - 1);
  const int64_t step = WIDE ? gridDim.x : (int64_t)gridDim.x << (8 - glog);
  int64_t r = WIDE ? blockIdx.x : ((int64_t)blockIdx.x << (8 - glog)) + (threadIdx.x >> glog);
  const int64_t turns = WIDE ? (rows - blockIdx.x + step - 1) / step : (rows - ((int64_t)blockIdx.x << (8 - glog)) + step - 1) / step;
  const float fc = (float)c;
  RowRegs<T, VEC, NV> cur, nxt;
  cur.load(row_ptr<T>(x, r < rows ? r : 0), t, g, c, r < rows);
  ParamRegs<VEC, NV> w, b;
  w.load(gamma, t, g, c, 1.f);
  b.load(beta, t, g, c, 0.f);
  for (int64_t it = 0; it < turns; ++it, r += step) {
    const int64_t rn = r + step;
    if (it + 1 < turns) nxt.load(row_ptr<T>(x, rn < rows ? rn : 0), t, g, c, rn < rows);
    float f[NV * VEC], s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      cur.get(i, f + i * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += f[i * VEC + e];
    }
    const float mu = row_sum<WIDE>(s, glog, sm) / fc;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float& v = f[i * VEC + e];
        v = (i * g + t) * VEC < c ? v - mu : 0.f;
        s += v * v;
      }
    const float rstd = 1.f / sqrtf(row_sum<WIDE>(s, glog, sm) / fc + eps);
    if (r < rows) {
      if (saved && t == 0) { saved[r] = mu; saved[rows + r] = rstd; }
      T* op = row_ptr<T>(o, r);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * g + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[i * VEC + e] = f[i * VEC + e] * rstd * w.v[i * VEC + e] + b.v[i * VEC + e];
        if (col < c) stv<T, VEC>(op + col, f + i * VEC);
      }
    }
    cur = nxt;
  }
}

// PARAM: the workgroup's sums for gamma / beta go to ws[blockIdx.x][2][c]
template <typename T, int VEC, int NV, bool WIDE, bool PARAM>
__global__ __launch_bounds__(256) void ln_bwd_kernel(Rows go, Rows x, Rows gx, int want_gx, int64_t rows, int c, int glog, const float* saved,
                                                     const float* gamma, int acc, float* ws) {
  __shared__ float sm[4];
  extern __shared__ float tot[];                            // PARAM && !WIDE: [2][c]
  const int g = WIDE ? 256 : 1 << glog, t = WIDE ? threadIdx.x : threadIdx.x & (g - 1);
  const int64_t step = WIDE ? gridDim.x : (int64_t)gridDim.x << (8 - glog);
  int64_t r = WIDE ? blockIdx.x : ((int64_t)blockIdx.x << (8 - glog)) + (threadIdx.x >> glog);
  const int64_t turns = WIDE ? (rows - blockIdx.x + step - 1) / step : (rows - ((int64_t)blockIdx.x << (8 - glog)) + step - 1) / step;
  const float fc = (float)c;
  RowRegs<T, VEC, NV> cx, cg, nx, ng;
  {
    const int64_t q = r < rows ? r : 0;
    cx.load(row_ptr<T>(x, q), t, g, c, r < rows);
    cg.load(row_ptr<T>(go, q), t, g, c, r < rows);
  }
  ParamRegs<VEC, NV> w;
  w.load(gamma, t, g, c, 1.f);
  float dg[PARAM ? NV * VEC : 1], db[PARAM ? NV * VEC : 1];
#pragma unroll
  for (int i = 0; i < (PARAM ? NV * VEC : 1); ++i) dg[i] = db[i] = 0.f;
  for (int64_t it = 0; it < turns; ++it, r += step) {
    const int64_t rn = r + step, q = r < rows ? r : 0;
    const float mu = saved[q], rstd = saved[rows + q];
    if (it + 1 < turns) {
      const int64_t qn = rn < rows ? rn : 0;
      nx.load(row_ptr<T>(x, qn), t, g, c, rn < rows);
      ng.load(row_ptr<T>(go, qn), t, g, c, rn < rows);
    }
    float xh[NV * VEC], v[NV * VEC], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      cx.get(i, xh + i * VEC);
      cg.get(i, v + i * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int k = i * VEC + e;
        xh[k] = r < rows && (i * g + t) * VEC < c ? (xh[k] - mu) * rstd : 0.f;
        if constexpr (PARAM) { dg[k] += v[k] * xh[k]; db[k] += v[k]; }
        v[k] *= w.v[k];
        s1 += v[k];
        s2 += v[k] * xh[k];
      }
    }
    if (want_gx) {
      row_sums<WIDE>(s1, s2, glog, sm);
      s1 /= fc;
      s2 /= fc;
      if (r < rows) {
        T* op = row_ptr<T>(gx, r);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * g + t) * VEC;
          if (col >= c) continue;
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i * VEC + e] = rstd * (v[i * VEC + e] - s1 - xh[i * VEC + e] * s2);
          if (acc) {
            float old[VEC];
            ldv<T, VEC>(op + col, old);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i * VEC + e] += old[e];
          }
          stv<T, VEC>(op + col, v + i * VEC);
        }
      }
    }
    cx = nx;
    cg = ng;
  }
  if constexpr (PARAM) {
    float* wp = ws + (int64_t)blockIdx.x * 2 * c;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < NV * VEC; ++i) {
        const int col = ((i / VEC) * g + t) * VEC + i % VEC;
        if (col < c) { wp[col] = dg[i]; wp[c + col] = db[i]; }
      }
    } else {
      // rows of a wave (a butterfly over its groups), then the four waves one after the other: one order, whatever runs when
      for (int o = g; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) { dg[i] += __shfl_xor(dg[i], o, 64); db[i] += __shfl_xor(db[i], o, 64); }
      for (int k = 0; k < 4; ++k) {
        if ((threadIdx.x >> 6) == k && (threadIdx.x & 63) < g) {
#pragma unroll
          for (int i = 0; i < NV * VEC; ++i) {
            const int col = ((i / VEC) * g + t) * VEC + i % VEC;
            if (col < c) {
              tot[col] = k ? tot[col] + dg[i] : dg[i];
              tot[c + col] = k ? tot[c + col] + db[i] : db[i];
            }
          }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < 2 * c; i += 256) wp[i] = tot[i];
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

// ws [n][2][c] -> dgamma, dbeta: 16 channels x 64 slices of the partial rows a workgroup, combined in a fixed order
__global__ __launch_bounds__(1024) void ln_param_reduce_kernel(const float* ws, int n, int c, float* dgamma, float* dbeta, int acc) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4;
  for (int c0 = blockIdx.x * 16; c0 < 2 * c; c0 += gridDim.x * 16) {
    const int col = c0 + cl;                             // 0 .. 2c: gamma's channels, then beta's
    float s = 0.f;
    if (col < 2 * c) {
#pragma unroll 8
      for (int i = sl; i < n; i += 64) s += ws[(int64_t)i * 2 * c + col];
    }
    sm[sl][cl] = s;
    __syncthreads();
    if (sl == 0 && col < 2 * c) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i) s += sm[i][cl];
      float* d = col < c ? dgamma : dbeta;
      if (d) {
        d += col < c ? col : col - c;
        *d = acc ? *d + s : s;
      }
    }
    __syncthreads();
  }
}

// how a row is laid out over lanes: vectors a lane, lanes a row (log2), or the whole workgroup; nv == 0: read row by row (any_kernel)
struct Lay { int nv, glog; bool wide; };
// most: vectors a lane may hold while its row has lanes left to spread over.  The forward takes up to four (rows of 192: 8 lanes x 3 vectors, no
// lane idle: 22 us against 39 with 32 lanes x 1), the backward, seven registers an element, needs the waves more than the lanes (36 against 49)
Lay lay_of(int c, int vec, int most = 4) {
  const int n = (c + vec - 1) / vec;
  // the fewest idle lanes of 4 .. 64 times 1 .. 4 vectors, the most lanes where that ties; then whole waves with more, then workgroups; at
  // most 32 elements a lane (the backward holds seven registers an element: 64 of them spill)
  Lay best{0, 0, false};
  int waste = 1 << 30;
  for (int gl = 6; gl >= 2; --gl)
    for (int nv = 1; nv <= 4; ++nv)
      if ((nv <= most || gl == 6) && (nv << gl) >= n && (nv << gl) - n < waste) { waste = (nv << gl) - n; best = Lay{nv, gl, false}; }
  if (best.nv) return best;
  if (vec < 8 && n <= 64 * 8) return Lay{8, 6, false};
  if (vec == 1 && n <= 64 * 16) return Lay{16, 6, false};
  for (int nv = 2; nv <= 4; ++nv)
    if (n <= 256 * nv) return Lay{nv, 8, true};
  if (vec < 8 && n <= 256 * 8) return Lay{8, 8, true};
  if (vec == 1 && n <= 256 * 16) return Lay{16, 8, true};
  return best;
}
constexpr int kSlices = 1024;
// workgroups of the backward (= partial parameter sums): four a CU, each lane group at least four rows (131072 x 192: 512 / 768 / 1024 / 1280
// workgroups take 47 / 39 / 36 / 35 us, their sums another 4.0 / 4.6 / 5.2 / 5.8)
int bwd_groups(int64_t rows, const Lay& l) {
  const int64_t per = l.wide ? 1 : 1 << (8 - l.glog);
  int64_t n = (rows + per * 4 - 1) / (per * 4);
  return (int)(n < kSlices ? n : kSlices);
}

bool view_ok(const myolo_tensor& t) {
  return (t.ptr || (int64_t)t.n * t.h * t.w == 0) && (t.dtype == MYOLO_F16 || t.dtype == MYOLO_F32) && t.n >= 0 && t.h >= 0 && t.w >= 0 && t.c >= 1 && t.c <= MYOLO_LAYERNORM_MAX_C &&
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

#define LN_BY_NV(CALL)                                                                                                \
  if (l.wide) {                                                                                                       \
    if (l.nv == 2) { CALL(2, true); } else if (l.nv == 3) { CALL(3, true); } else if (l.nv == 4) { CALL(4, true); }   \
    else if (l.nv == 8) { if constexpr (VEC < 8) { CALL(8, true); } }                                                 \
    else { if constexpr (VEC == 1) { CALL(16, true); } }                                                              \
  } else if (l.nv == 1) { CALL(1, false); } else if (l.nv == 2) { CALL(2, false); }                                   \
  else if (l.nv == 3) { CALL(3, false); } else if (l.nv == 4) { CALL(4, false); }                                     \
  else if (l.nv == 8) { if constexpr (VEC < 8) { CALL(8, false); } }                                                  \
  else { if constexpr (VEC == 1) { CALL(16, false); } }

template <typename T, int VEC>
int ln_fwd(const myolo_tensor* x, const float* gamma, const float* beta, float eps, const myolo_tensor* out, float* saved, hipStream_t st) {
  const int64_t rows = (int64_t)x->n * x->h * x->w;
  const Rows rx = rows_of(*x), ro = rows_of(*out);
  const Lay l = lay_of(x->c, VEC);
  if (!l.nv) {
    const int grid = (int)(rows < 65536 ? rows : 65536);
    hipLaunchKernelGGL((ln_fwd_any_kernel<T, VEC>), dim3(grid), dim3(256), 0, st, rx, ro, rows, x->c, gamma, beta, eps, saved);
  } else {
    const int64_t per = l.wide ? 1 : 1 << (8 - l.glog), all = (rows + per - 1) / per;
    const int grid = (int)(all < 1024 ? all : 1024);
#define LN_FWD(NV, WIDE) \
  hipLaunchKernelGGL((ln_fwd_kernel<T, VEC, NV, WIDE>), dim3(grid), dim3(256), 0, st, rx, ro, rows, x->c, l.glog, gamma, beta, eps, saved)
    LN_BY_NV(LN_FWD)
#undef LN_FWD
  }
  MYOLO_CHECK_LAUNCH();
  return 0;
}

template <typename T, int VEC>
int ln_bwd(const myolo_tensor* gout, const myolo_tensor* x, const float* saved, const float* gamma, const myolo_tensor* gx, int acc_x,
           float* dgamma, float* dbeta, int acc_params, float* ws, hipStream_t st) {
  const int64_t rows = (int64_t)x->n * x->h * x->w;
  const Rows rx = rows_of(*x), rg = rows_of(*gout), ro = gx ? rows_of(*gx) : Rows{};
  const bool param = dgamma || dbeta;
  const int c = x->c;
  const Lay l = lay_of(c, VEC, 1);
  int ns = 0;
  if (rows && l.nv) {
    ns = bwd_groups(rows, l);
    const int smem = param && !l.wide ? 2 * c * 4 : 0;
#define LN_BWD(NV, WIDE)                                                                                                                   \
  if (param) hipLaunchKernelGGL((ln_bwd_kernel<T, VEC, NV, WIDE, true>), dim3(ns), dim3(256), smem, st, rg, rx, ro, gx != nullptr, rows, c, \
                                l.glog, saved, gamma, acc_x, ws);                                                                          \
  else hipLaunchKernelGGL((ln_bwd_kernel<T, VEC, NV, WIDE, false>), dim3(ns), dim3(256), 0, st, rg, rx, ro, 1, rows, c, l.glog, saved,     \
                          gamma, acc_x, ws)
    if (param || gx) { LN_BY_NV(LN_BWD) }
#undef LN_BWD
    MYOLO_CHECK_LAUNCH();
  } else if (rows) {
    if (param) {              // (before gx, which may be gout)
      ns = (int)(rows < 256 ? rows : 256);
      hipLaunchKernelGGL((ln_param_any_kernel<T>), dim3((c + 63) / 64, ns), dim3(256), 0, st, rg, rx, rows, c, saved, ws);
      MYOLO_CHECK_LAUNCH();
    }
    if (gx) {
      const int grid = (int)(rows < 65536 ? rows : 65536);
      hipLaunchKernelGGL((ln_bwd_any_kernel<T, VEC>), dim3(grid), dim3(256), 0, st, rg, rx, ro, rows, c, saved, gamma, acc_x);
      MYOLO_CHECK_LAUNCH();
    }
  }
  if (param) {
    hipLaunchKernelGGL(ln_param_reduce_kernel, dim3(grid_for(2 * (int64_t)c, 16, 1 << 16)), dim3(1024), 0, st, ws, ns, c, dgamma, dbeta, acc_params);
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
  const bool v = vec_ok(*x) && vec_ok(*out);
  if (x->dtype == MYOLO_F16)
    return v ? ln_fwd<half_t, 8>(x, gamma, beta, eps, out, saved, st) : ln_fwd<half_t, 1>(x, gamma, beta, eps, out, saved, st);
  return v ? ln_fwd<float, 4>(x, gamma, beta, eps, out, saved, st) : ln_fwd<float, 1>(x, gamma, beta, eps, out, saved, st);
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
  const bool v = vec_ok(*x) && vec_ok(*gout) && (!gx || vec_ok(*gx));
  if (x->dtype == MYOLO_F16)
    return v ? ln_bwd<half_t, 8>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st)
             : ln_bwd<half_t, 1>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st);
  return v ? ln_bwd<float, 4>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st)
           : ln_bwd<float, 1>(gout, x, saved, gamma, gx, acc_x, dgamma, dbeta, acc_params, ws, st);
}
