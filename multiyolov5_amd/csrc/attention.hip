// Attention with a sliding window and leading keys that stay visible (sinks): forward, split over the key axis for few rows, backward.
//
//   S = scale q k^T over the visible keys, P = softmax(S), o = P v
//   dP = do v^T,  delta = rowsum(do * o),  dS = P (dP - delta);   dq = scale dS k,  dk = scale dS^T q,  dv = P^T do
//
// All products run on the 32x32 matrix instruction with the score tile transposed as its consumer needs it: a lane of the result holds ONE
// column (lane % 32) and 16 rows 8*(r/4) + r%4 + 4*(lane/32).  The forward and dq form S^T = K Q^T, so that a lane owns one query: the
// softmax statistics stay in the lane (one exchange between the wave's halves per tile) and the 16 keys it holds are, in this order, the
// contraction operand of O^T = V^T P^T -- no shuffle of P.  dk / dv form S = Q K^T for the same reason with the key in the lane.  The other
// operand of the second product is read across the rows of its LDS tile: transposing 8-byte LDS reads for fp16, plain reads for fp32 (whose
// 8-element operands feed eight 32x32x2 instructions).
// The rows of a (batch, key head) are its query heads' queries, i * group + g: one K / V tile serves all heads of the group.
#include "myolo_dev.h"

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const char *q, *k, *v, *go;
  char *o, *ores, *gq, *gk, *gv;
  float *lse, *delta;
  float* part;             // split forward: [split][b*hk][rows][d] unnormalised sums, then [split][b*hk][rows][2] max and denominator
                           // split dk / dv: [b*hk][nsb][split][dk, dv][128][d] partial sums
  const int *lens, *starts;
  int64_t qs[3], ks[3], vs[3], os[3], gos[3], gqs[3], gks[3], gvs[3];      // bytes
  int b, lq, lk, hq, hk, g, d, causal, window, sinks;
  int rows, nblk, nsplit, nsb;        // nsb: key blocks [0, nsb) of the dk / dv pass are split over nsplit workgroups
  float scale, sl2;        // scale, scale * log2(e)
};

// ---- fragments: 8 elements along the contracted axis --------------------------------------------------------------------------------
template <typename T> struct Frag;
template <> struct Frag<half_t> { h8_t v; };
template <> struct Frag<float> { f4_t a, b; };

__device__ __forceinline__ f16_t mma(const Frag<half_t>& a, const Frag<half_t>& b, f16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f16_t mma(const Frag<float>& a, const Frag<float>& b, f16_t c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.a[i], b.a[i], c, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.b[i], b.b[i], c, 0, 0, 0);
  return c;
}
// 8 accumulator registers 8*S .. 8*S + 7 as an operand
template <int S> __device__ __forceinline__ void frag_from(Frag<half_t>& f, const f16_t& c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.v[i] = (half_t)c[8 * S + i];
}
template <int S> __device__ __forceinline__ void frag_from(Frag<float>& f, const f16_t& c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { f.a[i] = c[8 * S + i]; f.b[i] = c[8 * S + 4 + i]; }
}
// 8 consecutive elements of a row in global memory, zeros where !ok
__device__ __forceinline__ void frag_global(Frag<half_t>& f, const char* p, bool ok) {
  const uint4 v = ldg16(ok ? p : zero_page());
  f.v = *reinterpret_cast<const h8_t*>(&v);
}
__device__ __forceinline__ void frag_global(Frag<float>& f, const char* p, bool ok) {
  const uint4 v = ldg16(ok ? p : zero_page()), w = ldg16(ok ? p + 16 : zero_page());
  f.a = *reinterpret_cast<const f4_t*>(&v);
  f.b = *reinterpret_cast<const f4_t*>(&w);
}
__device__ __forceinline__ float frag_dot(const Frag<half_t>& a, const Frag<half_t>& b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += (float)a.v[i] * (float)b.v[i];
  return s;
}
__device__ __forceinline__ float frag_dot(const Frag<float>& a, const Frag<float>& b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += a.a[i] * b.a[i] + a.b[i] * b.b[i];
  return s;
}

// ---- LDS tiles: rows of DL elements in 16-byte chunks; chunk c of row r sits at c ^ swz(r), so that 16 rows at one chunk (row operands) and 4
// rows x 4 chunks (transposing reads) both cover all 64 banks
template <typename T, int DL> struct Tile {
  static constexpr int EC = 16 / (int)sizeof(T);            // elements a chunk
  static constexpr int CH = DL / EC;                        // chunks a row
  __device__ static __forceinline__ int swz(int r) {
    if constexpr (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (CH == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  __device__ static __forceinline__ int unit(int r, int c) { return r * CH + (c ^ swz(r)); }
  // row operand: 8 elements at column 8*c8 of row r
  __device__ static __forceinline__ void row_frag(Frag<half_t>& f, const uint4* s, int r, int c8) {
    f.v = *reinterpret_cast<const h8_t*>(s + unit(r, c8));
  }
  __device__ static __forceinline__ void row_frag(Frag<float>& f, const uint4* s, int r, int c8) {
    f.a = *reinterpret_cast<const f4_t*>(s + unit(r, 2 * c8));
    f.b = *reinterpret_cast<const f4_t*>(s + unit(r, 2 * c8 + 1));
  }
  // column operand: column c0 + lane % 32, rows r0 + {0..3, 8..11} + 4 * (lane / 32)
  __device__ static __forceinline__ void col_frag(Frag<half_t>& f, const uint4* s, int r0, int c0, int lane) {
    typedef __attribute__((address_space(3))) fp16x4_t lds_t;
    const int sub = lane & 15;
    const int c = (c0 >> 3) + ((lane >> 4) & 1) * 2 + ((sub & 3) >> 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 8 * i + 4 * (lane >> 5) + (sub >> 2);
      const char* p = reinterpret_cast<const char*>(s + unit(r, c)) + (sub & 1) * 8;
      const fp16x4_t t = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_t*)(p));
#pragma unroll
      for (int e = 0; e < 4; ++e) f.v[4 * i + e] = (half_t)t[e];
    }
  }
  __device__ static __forceinline__ void col_frag(Frag<float>& f, const uint4* s, int r0, int c0, int lane) {
    const int col = c0 + (lane & 31);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = r0 + 4 * (lane >> 5) + e;
      f.a[e] = reinterpret_cast<const float*>(s + unit(r, col >> 2))[col & 3];
      f.b[e] = reinterpret_cast<const float*>(s + unit(r + 8, col >> 2))[col & 3];
    }
  }
};

// the column operands of 32 rows from r0 on, 32 columns a step (two 16-row operands): AHEAD reads step m + 1 before step m's matrix
// instructions are issued and keeps the scheduler from moving the reads back to their use
template <typename T, int DL, bool AHEAD> struct Columns {
  const uint4* s;
  int r0, lane;
  Frag<T> f[AHEAD ? 2 : 1][2];
  __device__ __forceinline__ Columns(const uint4* s_, int r0_, int lane_) : s(s_), r0(r0_), lane(lane_) {}
  __device__ __forceinline__ void read(int m) {
    Tile<T, DL>::col_frag(f[AHEAD ? m & 1 : 0][0], s, r0, m * 32, lane);
    Tile<T, DL>::col_frag(f[AHEAD ? m & 1 : 0][1], s, r0 + 16, m * 32, lane);
  }
  __device__ __forceinline__ void first() { if constexpr (AHEAD) read(0); }
  __device__ __forceinline__ void next(int m) { if constexpr (AHEAD) read(m + 1); }
  __device__ __forceinline__ void now(int m) {
    if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
    else read(m);
  }
  __device__ __forceinline__ const Frag<T>& a(int m) const { return f[AHEAD ? m & 1 : 0][0]; }
  __device__ __forceinline__ const Frag<T>& b(int m) const { return f[AHEAD ? m & 1 : 0][1]; }
};
template <typename T> constexpr bool kAheadOf = sizeof(T) == 2;

// a product as a 32-bit value: without this the compiler rounds it straight to fp16 on the paths that need nothing else of it, and results with
// and without the residual differ in the last bit
__device__ __forceinline__ float pin(float x) { asm("" : "+v"(x)); return x; }

// the value of the lane's column in the other half of the wave, combined
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- what is visible -----------------------------------------------------------------------------------------------------------------
// Everything here is an interval of integers: masks are one or two unsigned comparisons and a select, never a branch of the lanes.
struct Range {             // lo <= x < lo + n
  int lo;
  unsigned n;
  __device__ __forceinline__ bool has(int x) const { return (unsigned)x - (unsigned)lo < n; }
};
__device__ __forceinline__ Range range_of(int lo, int hi) { return Range{lo, hi > lo ? (unsigned)hi - (unsigned)lo : 0u}; }
struct Keys {              // keys [0, first) and the band
  int first;
  Range band;
  __device__ __forceinline__ bool has(int j) const { return band.has(j) | (j < first); }
};
struct Vis {
  int start, len, causal, window, sinks;
  // the keys that some query of the consecutive positions [p0, p1] sees
  __device__ __forceinline__ Keys keys(int p0, int p1) const {
    const int hi = causal ? min(len, p1 + 1) : len;
    return Keys{window ? min(sinks, hi) : 0, window ? range_of(max(0, p0 - window + 1), min(hi, p1 + window)) : range_of(0, hi)};
  }
  // the positions that see key j
  __device__ __forceinline__ Range queries(int j) const {
    const bool band = window && j >= sinks;
    int lo = band ? j - window + 1 : -(1 << 30);
    if (causal) lo = max(lo, j);
    return range_of(lo, j < len ? (band ? j + window : 1 << 30) : lo);
  }
  // the positions that see some key
  __device__ __forceinline__ Range rows() const {
    const bool band = window && !sinks;
    const int lo = causal ? 0 : band ? 1 - window : -(1 << 30);
    return range_of(lo, len > 0 ? (band ? len + window - 1 : 1 << 30) : lo);
  }
  // every query of positions [p0, p1] sees every key of [j0, j1]
  __device__ __forceinline__ bool all(int p0, int p1, int j0, int j1) const {
    return (j1 < len) & (!causal | (j1 <= p0)) & (!window | ((p1 - j0 < window) & (j1 - p0 < window)) | (j1 < sinks));
  }
  // some query of [p0, p1] may see some key of [j0, j1]
  __device__ __forceinline__ bool any(int p0, int p1, int j0, int j1) const {
    return (j0 < len) & (!causal | (j0 <= p1)) & (!window | ((p0 - j1 < window) & (j0 - p1 < window)) | (j0 < sinks));
  }
};
// (start is clamped to where nothing changes any more, so that positions and distances stay within 32 bits: all lengths <= 2^28)
__device__ __forceinline__ Vis vis_of(const AttnArgs& a, int b) {
  Vis v{a.lk - a.lq, a.lk, a.causal, a.window, a.sinks};
  if (a.lens) v.len = min(max(a.lens[b], 0), a.lk);
  if (a.starts) v.start = min(max(a.starts[b], -a.lq - a.window), a.lk + a.window);
  return v;
}
// the key tiles of BK that queries [p0, p1] may see: tiles [0, n1) hold sinks only, n - n1 tiles from lo on the band
struct TileList { int n1, lo, n; __device__ __forceinline__ int at(int i) const { return i < n1 ? i : lo + (i - n1); } };
__device__ __forceinline__ TileList tiles_of(const Vis& v, int p0, int p1, int bk) {
  int hi = v.causal ? min(v.len, p1 + 1) : v.len, lo = 0, first = 0;
  if (v.window) {
    first = max(0, min(v.sinks, hi));                       // keys [0, first) stay visible
    lo = max(0, p0 - v.window + 1);
    hi = min(hi, p1 + v.window);
    if (hi <= lo) hi = lo = 0;                              // an empty band
    if (first >= lo) { lo = 0; hi = max(hi, first); first = 0; }       // one run of keys
  }
  const int tlo = lo / bk, thi = max((max(hi, 0) + bk - 1) / bk, tlo), n1 = min((first + bk - 1) / bk, tlo);
  return TileList{n1, tlo, n1 + thi - tlo};
}

// ROWS x DP elements from global rows into registers (zeros for hidden rows and channels >= d), registers into a tile
template <typename T, int DP, int ROWS, int NT> struct Stage {
  static constexpr int EC = 16 / (int)sizeof(T), CH = DP / EC, N = ROWS * CH, PER = (N + NT - 1) / NT;
  uint4 v[PER];
  template <class F> __device__ __forceinline__ void load(const char* base, int64_t stride, int d, int tid, F row_ok) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * NT, r = u / CH, c = u - r * CH;
      const bool ok = (u < N) & (c * EC < d) & row_ok(r);
      v[i] = ldg16(ok ? base + (int64_t)r * stride + c * 16 : zero_page());
    }
  }
  template <int DL> __device__ __forceinline__ void store(uint4* s, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * NT, r = u / CH, c = u - r * CH;
      if (N % NT == 0 || u < N) s[Tile<T, DL>::unit(r, c)] = v[i];
    }
  }
};

__host__ __device__ constexpr int lds_width(int dp) { return dp <= 32 ? 32 : dp <= 64 ? 64 : 128; }

// consecutive workgroups go round the 8 XCDs: give each XCD a contiguous run of the work, so that neighbours share K / V in its L2
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int per = n >> 3, rem = n & 7, x = id & 7, k = id >> 3;
  return x * per + min(x, rem) + k;
}

// ---- forward -------------------------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows (four waves x 32) through its key tiles, or 32 rows in one wave where the call has no more (one token: the key
// axis is split over workgroups).  Bound by the matrix pipe and the softmax's vector instructions in turn, two waves a SIMD covering each
// other: causal 8192 x 128 channels, 32 / 8 heads fp16 in 0.65 ms, 850 TFLOP/s (pipe 43 % busy); 64 channels have half the products for the same
// softmax: 16 x 2048, window 256 both ways, 4 heads in 49 us, 330 TFLOP/s.  One token over 8 caches of up to 32768 x 8 heads x 128: 151 us, 5.3 TB/s,
// bound by HBM.
template <typename T, int DP, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, NW == 4 && (sizeof(T) == 2 || DP <= 64) ? 2 : 1) void attn_fwd_kernel(AttnArgs a) {
  constexpr int BK = sizeof(T) == 2 || NW > 1 ? 64 : 32, U = BK / 32, DL = lds_width(DP), NT = NW * 64, KS = DP / 16, MT = (DP + 31) / 32;
  using TL = Tile<T, DL>;
  __shared__ uint4 sK[BK * TL::CH], sV[BK * TL::CH];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = SPLIT ? id % a.nsplit : 0;
  if (SPLIT) id /= a.nsplit;
  const int blk = a.nblk - 1 - id % a.nblk, bh = id / a.nblk;       // (long causal blocks first)
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const Vis vis = vis_of(a, b);
  const int r0 = blk * 32 * NW, r1 = min(r0 + 32 * NW, a.rows) - 1;
  const int pb0 = vis.start + r0 / a.g, pb1 = vis.start + r1 / a.g;
  const int w0 = min(r0 + wv * 32, r1), w1 = min(w0 + 31, r1);
  const int pw0 = vis.start + w0 / a.g, pw1 = vis.start + w1 / a.g;
  const int row = r0 + wv * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int qi = (live ? row : r1) / a.g, head = kh * a.g + (live ? row : r1) - qi * a.g;
  const int p = vis.start + qi;

  const char* kp = a.k + b * a.ks[0] + kh * a.ks[2];
  const char* vp = a.v + b * a.vs[0] + kh * a.vs[2];
  // fp16 probabilities enter the product as 2^11 .. 2^15 times what they are of the largest: what thousands of weak keys add up to would be lost
  // in subnormals otherwise (40000 keys of 2^-26 each: all of it).  A key's is off by at most 2^-36 now: half a step of a result for 2^25 keys
  constexpr float kLift = sizeof(T) == 2 ? 11.f : 0.f, kSlack = sizeof(T) == 2 ? 4.f : 8.f;
  f16_t o[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) o[m] = f16_t{};
  float mx = -INFINITY, l = 0.f;              // the reference the probabilities are formed with (log2), their sum

  const TileList tl = tiles_of(vis, pb0, pb1, BK);
  const Keys bkeys = vis.keys(pb0, pb1), lkeys = vis.keys(p, p);       // the workgroup's keys, the lane's
  int t0 = 0, t1 = tl.n;
  if (SPLIT) {
    const int per = (tl.n + a.nsplit - 1) / a.nsplit;
    t0 = min(sp * per, tl.n);
    t1 = min(t0 + per, tl.n);
  }
  // the next tile's global loads are in flight while this one is computed
  Stage<T, DP, BK, NT> gk, gv;
  auto fetch = [&](int t) {
    const int j0 = tl.at(t) * BK;
    auto ok = [&](int r) { return bkeys.has(j0 + r); };
    gk.load(kp + (int64_t)j0 * a.ks[1], a.ks[1], a.d, tid, ok);
    gv.load(vp + (int64_t)j0 * a.vs[1], a.vs[1], a.d, tid, ok);
  };
  auto put = [&]() {
    gk.template store<DL>(sK, tid);
    gv.template store<DL>(sV, tid);
  };
  if (t0 < t1) fetch(t0);                                  // (in flight beside the query operands)
  Frag<T> qf[KS];
  const char* qp = a.q + b * a.qs[0] + qi * a.qs[1] + head * a.qs[2];
#pragma unroll
  for (int s = 0; s < KS; ++s) frag_global(qf[s], qp + (s * 16 + h * 8) * sizeof(T), live & (s * 16 + h * 8 < a.d));

  if (t0 < t1) put();
  for (int t = t0; t < t1; ++t) {
    const int j0 = tl.at(t) * BK;
    const bool more = t + 1 < t1;
    __syncthreads();
    if (more) fetch(t + 1);
    if (vis.any(pw0, pw1, j0, j0 + BK - 1)) {
      f16_t s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = f16_t{};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Frag<T> kf;
          TL::row_frag(kf, sK, u * 32 + (lane & 31), k * 2 + h);
          s[u] = mma(kf, qf[k], s[u]);
        }
      }
      if (!vis.all(pw0, pw1, j0, j0 + BK - 1)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[u][r] = lkeys.has(j0 + u * 32 + (r & 3) + 8 * (r >> 2) + 4 * h) ? s[u][r] : -INFINITY;
      }
      float m2 = s[0][0];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) m2 = fmaxf(m2, s[u][r]);
      // the reference lies kLift under the maximum it was taken from and follows the running one only when that has outgrown it by kSlack: the sums are
      // hardly ever rescaled after the first tiles
      m2 = half_max(m2) * a.sl2 - kLift;
      if (__any(m2 > mx + kSlack)) {
        m2 = fmaxf(mx, m2);
        const float al = __builtin_amdgcn_exp2f(mx - (m2 == -INFINITY ? 0.f : m2));
        mx = m2;
        l *= al;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[m][r] *= al;
      }
      const float use = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], a.sl2, -use));
          l += s[u][r];
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Frag<T> p0, p1, vf;
        frag_from<0>(p0, s[u]);
        frag_from<1>(p1, s[u]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          TL::col_frag(vf, sV, u * 32, m * 32, lane);
          o[m] = mma(vf, p0, o[m]);
          TL::col_frag(vf, sV, u * 32 + 16, m * 32, lane);
          o[m] = mma(vf, p1, o[m]);
        }
      }
    }
    __syncthreads();
    if (more) put();
  }
  l = half_sum(l);
  if (!live) return;
  if (SPLIT) {
    const int64_t pr = ((int64_t)sp * (a.b * a.hk) + bh) * a.rows + row;
    float* po = a.part + pr * a.d;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int c = m * 32 + q4 * 8 + 4 * h;
        if (c < a.d) *reinterpret_cast<f4_t*>(po + c) = f4_t{o[m][4 * q4], o[m][4 * q4 + 1], o[m][4 * q4 + 2], o[m][4 * q4 + 3]};
      }
    if (h == 0) {
      float* ml = a.part + (int64_t)a.nsplit * (a.b * a.hk) * a.rows * a.d + pr * 2;
      ml[0] = mx;
      ml[1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (a.lse && h == 0) a.lse[((int64_t)b * a.hq + head) * a.lq + qi] = l == 0.f ? -INFINITY : mx + __log2f(l);
  char* op = a.o + b * a.os[0] + qi * a.os[1] + head * a.os[2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int c = m * 32 + q4 * 8 + 4 * h;
      if (c >= a.d) continue;
      if constexpr (sizeof(T) == 2) {
        h4_t v, w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = pin(o[m][4 * q4 + e] * inv);
          v[e] = (half_t)x;
          w[e] = (half_t)(x - (float)v[e]);
        }
        *reinterpret_cast<h4_t*>(op + c * 2) = v;
        if (a.ores) *reinterpret_cast<h4_t*>(a.ores + (op - a.o) + c * 2) = w;
      } else {
        f4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[m][4 * q4 + e] * inv;
        *reinterpret_cast<f4_t*>(op + c * 4) = v;
      }
    }
}

// joins the splits of a row: o = sum o_s 2^(m_s - M) / sum l_s 2^(m_s - M)
template <typename T> __device__ __forceinline__ void join_store(const AttnArgs& a, int64_t pr, int c, const f4_t& o, float inv) {
  const int bh = (int)(pr / a.rows), row = (int)(pr - (int64_t)bh * a.rows), b = bh / a.hk;
  const int qi = row / a.g, head = (bh - b * a.hk) * a.g + row - qi * a.g;
  T* op = (T*)(a.o + b * a.os[0] + qi * a.os[1] + head * a.os[2]) + c;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = pin(o[e] * inv);
    const T v = (T)x;
    op[e] = v;
    if (a.ores) ((T*)(a.ores + ((char*)op - a.o)))[e] = (T)(x - (float)v);
  }
}
__device__ __forceinline__ void join_lse(const AttnArgs& a, int64_t pr, float mx, float sum) {
  const int bh = (int)(pr / a.rows), row = (int)(pr - (int64_t)bh * a.rows), b = bh / a.hk;
  const int qi = row / a.g, head = (bh - b * a.hk) * a.g + row - qi * a.g;
  a.lse[((int64_t)b * a.hq + head) * a.lq + qi] = sum == 0.f ? -INFINITY : mx + __log2f(sum);
}
// few splits: a thread takes four channels of a row over all of them
constexpr int kFewSplits = 8;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_few_kernel(AttnArgs a) {
  const int c4 = a.d / 4;
  const int64_t nrow = (int64_t)a.b * a.hk * a.rows, total = nrow * c4;
  const float* ml = a.part + (int64_t)a.nsplit * nrow * a.d;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int64_t pr = v / c4;
    const int c = (int)(v - pr * c4) * 4;
    f4_t x[kFewSplits];
    float m[kFewSplits], l[kFewSplits], mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
      const bool on = s < a.nsplit;
      const uint4 q = ldg16(on ? (const char*)(a.part + (s * nrow + pr) * a.d + c) : zero_page());
      x[s] = *reinterpret_cast<const f4_t*>(&q);
      m[s] = on ? ml[(s * nrow + pr) * 2] : -INFINITY;
      l[s] = on ? ml[(s * nrow + pr) * 2 + 1] : 0.f;
    }
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) mx = fmaxf(mx, m[s]);
    f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
      const float w = __builtin_amdgcn_exp2f(m[s] - (mx == -INFINITY ? 0.f : mx));
      sum += w * l[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += w * x[s][e];
    }
    if (a.lse && c == 0) join_lse(a, pr, mx, sum);
    join_store<T>(a, pr, c, o, sum == 0.f ? 0.f : 1.f / sum);
  }
}
// many splits (one token over a long cache): a workgroup a row.  One wave forms the weights (a lane a split), then 8 x 32 threads take every
// eighth split of four channels; the sums meet in LDS in a fixed order.  256 rows x 16 splits: 5 us, 12 with a thread over all splits;
// 4662 rows x 4 splits: 27 us, 5 with a thread.
constexpr int kMaxSplit = 64;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  __shared__ float sw[kMaxSplit];
  __shared__ f4_t so[8][32];
  __shared__ float sinv;
  const int64_t nrow = (int64_t)a.b * a.hk * a.rows;
  const float* ml = a.part + (int64_t)a.nsplit * nrow * a.d;
  const int cg = threadIdx.x & 31, sg = threadIdx.x >> 5, c = cg * 4;
  for (int64_t pr = blockIdx.x; pr < nrow; pr += gridDim.x) {
    f4_t x[kMaxSplit / 8];
#pragma unroll
    for (int i = 0; i < kMaxSplit / 8; ++i) {
      const int s = sg + 8 * i;
      const bool on = (s < a.nsplit) & (c < a.d);
      const uint4 v = ldg16(on ? (const char*)(a.part + (s * nrow + pr) * a.d + c) : zero_page());
      x[i] = *reinterpret_cast<const f4_t*>(&v);
    }
    if (threadIdx.x < 64) {
      const int s = threadIdx.x;
      const bool on = s < a.nsplit;
      const float m = on ? ml[(s * nrow + pr) * 2] : -INFINITY, l = on ? ml[(s * nrow + pr) * 2 + 1] : 0.f;
      float mx = m;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
      const float w = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx)), sum = wave_sum(w * l);
      sw[s] = w;
      if (s == 0) {
        sinv = sum == 0.f ? 0.f : 1.f / sum;
        if (a.lse) join_lse(a, pr, mx, sum);
      }
    }
    __syncthreads();
    f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kMaxSplit / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += sw[sg + 8 * i] * x[i][e];
    so[sg][cg] = o;
    __syncthreads();
    if (sg == 0 && c < a.d) {
#pragma unroll
      for (int k = 1; k < 8; ++k) o += so[k][cg];
      join_store<T>(a, pr, c, o, sinv);
    }
    __syncthreads();
  }
}

// ---- backward: dq (and delta) --------------------------------------------------------------------------------------------------------
// The forward's walk with the two score products formed again per tile: seven products in all instead of the five of one fused pass, whose dq would
// need atomics or a pass over partial sums of every key block.  2 x 4096, window 1024, 16 / 4 heads x 128 fp16: 171 us, 530 TFLOP/s of its
// three products; bound like the forward.
// P enters the fp16 product of dv times 2^12: a probability below 6e-5 (rows of more than 2^14 keys) would lose bits as an fp16 subnormal.
// dS has the size of P times the incoming gradient, anything from 1e-8 (a mean over a map's pixels) to more than the largest half: it enters
// its products times a power of two, the query's own in dq, the key's own in dk.  That starts at 2^24 and falls, with the sums formed so far,
// whenever an element would pass 2^15, to where the largest lies between 2^7 and 2^8: beside its relative half step an element is off by 2^-32 of
// the largest seen at most.  64 queries x 8192 keys, gradients of 1e-4: gq off by 7.2 % with dS as it is, by 0.93 % so, which is its own rounding;
// 16 x 2048 tokens of 64 channels cost 205 -> 215 us a pass for it, 2 x 4096 of 128 channels 526 -> 537.
template <typename T> constexpr float kPShift = sizeof(T) == 2 ? 12.f : 0.f;
template <typename T> constexpr float kPUnshift = sizeof(T) == 2 ? 1.f / 4096.f : 1.f;
constexpr int kMostUp = 24;
constexpr float kTop = 32768.f;
__device__ __forceinline__ int to_room(float m) { return 134 - (int)(__float_as_uint(m) >> 23); }       // 2^that * m lies in [2^7, 2^8), m > 0

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 || DP <= 64 ? 2 : 1) void attn_bwd_q_kernel(AttnArgs a) {
  constexpr bool kAhead = kAheadOf<T> && DP <= 64;         // (more: spills at two waves a SIMD)
  constexpr int NW = 4, BK = sizeof(T) == 2 ? 64 : 32, DL = lds_width(DP), NT = NW * 64, KS = DP / 16, MT = (DP + 31) / 32;
  using TL = Tile<T, DL>;
  __shared__ uint4 sK[BK * TL::CH], sV[BK * TL::CH];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = id % a.nsplit;                             // few blocks over a long key axis: its tiles are shared, the sums joined
  id /= a.nsplit;
  const int blk = a.nblk - 1 - id % a.nblk, bh = id / a.nblk;
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const Vis vis = vis_of(a, b);
  const int r0 = blk * 32 * NW, r1 = min(r0 + 32 * NW, a.rows) - 1;
  const int pb0 = vis.start + r0 / a.g, pb1 = vis.start + r1 / a.g;
  const int w0 = min(r0 + wv * 32, r1), w1 = min(w0 + 31, r1);
  const int pw0 = vis.start + w0 / a.g, pw1 = vis.start + w1 / a.g;
  const int row = r0 + wv * 32 + (lane & 31);
  const bool live = row < a.rows;
  const int qi = (live ? row : r1) / a.g, head = kh * a.g + (live ? row : r1) - qi * a.g;
  const int p = vis.start + qi;

  Frag<T> qf[KS], gf[KS];
  const char* qp = a.q + b * a.qs[0] + qi * a.qs[1] + head * a.qs[2];
  const char* gp = a.go + b * a.gos[0] + qi * a.gos[1] + head * a.gos[2];
  const char* op = a.o + b * a.os[0] + qi * a.os[1] + head * a.os[2];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int c = (s * 16 + h * 8);
    const bool ok = live & (c < a.d);
    Frag<T> of;
    frag_global(qf[s], qp + c * sizeof(T), ok);
    frag_global(gf[s], gp + c * sizeof(T), ok);
    frag_global(of, op + c * sizeof(T), ok);
    delta += frag_dot(gf[s], of);
    if constexpr (sizeof(T) == 2) {                          // (a select, not a branch: eight waits in a row cost a seventh of the kernel)
      frag_global(of, a.ores + (op - a.o) + c * sizeof(T), ok & (a.ores != nullptr));
      delta += frag_dot(gf[s], of);
    }
  }
  delta = half_sum(delta);
  const int64_t lrow = ((int64_t)b * a.hq + head) * a.lq + qi;
  const float lse = a.lse[lrow];
  if (live && h == 0 && sp == 0) a.delta[lrow] = delta;
  constexpr bool kUp = sizeof(T) == 2;
  int up = kUp ? kMostUp : 0;                                // the exponent that dS and dq are lifted by
  float nl = live ? (float)up - lse : -INFINITY;
  const char* kp = a.k + b * a.ks[0] + kh * a.ks[2];
  const char* vp = a.v + b * a.vs[0] + kh * a.vs[2];
  f16_t dq[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) dq[m] = f16_t{};

  const TileList tl = tiles_of(vis, pb0, pb1, BK);
  const Keys bkeys = vis.keys(pb0, pb1), lkeys = vis.keys(p, p);       // the workgroup's keys, the lane's
  const int per = (tl.n + a.nsplit - 1) / a.nsplit, t0 = min(sp * per, tl.n), nt = a.gq ? min(t0 + per, tl.n) : t0;
  Stage<T, DP, BK, NT> gk, gv;
  auto fetch = [&](int t) {
    const int j0 = tl.at(t) * BK;
    auto ok = [&](int r) { return bkeys.has(j0 + r); };
    gk.load(kp + (int64_t)j0 * a.ks[1], a.ks[1], a.d, tid, ok);
    gv.load(vp + (int64_t)j0 * a.vs[1], a.vs[1], a.d, tid, ok);
  };
  auto put = [&]() {
    gk.template store<DL>(sK, tid);
    gv.template store<DL>(sV, tid);
  };
  if (t0 < nt) { fetch(t0); put(); }
  for (int t = t0; t < nt; ++t) {
    const int j0 = tl.at(t) * BK;
    const bool more = t + 1 < nt;
    __syncthreads();
    if (more) fetch(t + 1);
    if (vis.any(pw0, pw1, j0, j0 + BK - 1)) {
      const bool all = vis.all(pw0, pw1, j0, j0 + BK - 1);
#pragma unroll
      for (int u = 0; u < BK / 32; ++u) {
        f16_t s = f16_t{}, dp = f16_t{};
        if constexpr (kAhead) {
          Frag<T> fk[KS], fv[KS];
#pragma unroll
          for (int k = 0; k < KS; ++k) TL::row_frag(fk[k], sK, u * 32 + (lane & 31), k * 2 + h);
#pragma unroll
          for (int k = 0; k < KS; ++k) TL::row_frag(fv[k], sV, u * 32 + (lane & 31), k * 2 + h);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < KS; ++k) s = mma(fk[k], qf[k], s);
#pragma unroll
          for (int k = 0; k < KS; ++k) dp = mma(fv[k], gf[k], dp);
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            Frag<T> f;
            TL::row_frag(f, sK, u * 32 + (lane & 31), k * 2 + h);
            s = mma(f, qf[k], s);
            TL::row_frag(f, sV, u * 32 + (lane & 31), k * 2 + h);
            dp = mma(f, gf[k], dp);
          }
        }
        Columns<T, DL, kAhead> ck(sK, u * 32, lane);
        ck.first();
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.sl2, nl)) * (dp[r] - delta);
        if (!all) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = lkeys.has(j0 + u * 32 + (r & 3) + 8 * (r >> 2) + 4 * h) ? s[r] : 0.f;
        }
        if constexpr (kUp) {
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[r]));
          if (__builtin_expect(__any(top > kTop), 0)) {
            top = half_max(top);
            const int e = top > kTop ? to_room(top) : 0;
            const float f = __builtin_amdgcn_ldexpf(1.f, e);
            up += e;
            nl = live ? (float)up - lse : -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= f;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int r = 0; r < 16; ++r) dq[m][r] *= f;
          }
        }
        Frag<T> d0, d1;
        frag_from<0>(d0, s);
        frag_from<1>(d1, s);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m + 1 < MT) ck.next(m);
          ck.now(m);
          dq[m] = mma(ck.a(m), d0, dq[m]);
          dq[m] = mma(ck.b(m), d1, dq[m]);
        }
      }
    }
    __syncthreads();
    if (more) put();
  }
  if (!live || !a.gq) return;
  const float down = __builtin_amdgcn_ldexpf(a.nsplit > 1 ? 1.f : a.scale, -up);
  if (a.nsplit > 1) {
    float* po = a.part + (((int64_t)sp * (a.b * a.hk) + bh) * a.rows + row) * a.d;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int c = m * 32 + q4 * 8 + 4 * h;
        if (c < a.d) *reinterpret_cast<f4_t*>(po + c) = f4_t{dq[m][4 * q4], dq[m][4 * q4 + 1], dq[m][4 * q4 + 2], dq[m][4 * q4 + 3]} * down;
      }
    return;
  }
  char* dp = a.gq + b * a.gqs[0] + qi * a.gqs[1] + head * a.gqs[2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = m * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
      if (c < a.d) reinterpret_cast<T*>(dp)[c] = (T)(dq[m][r] * down);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_q_join_kernel(AttnArgs a) {
  const int c4 = a.d / 4;
  const int64_t nrow = (int64_t)a.b * a.hk * a.rows, total = nrow * c4;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int64_t pr = v / c4;
    const int c = (int)(v - pr * c4) * 4, bh = (int)(pr / a.rows), row = (int)(pr - (int64_t)bh * a.rows), b = bh / a.hk;
    const int qi = row / a.g, head = (bh - b * a.hk) * a.g + row - qi * a.g;
    f4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < a.nsplit; ++i) s += *reinterpret_cast<const f4_t*>(a.part + (i * nrow + pr) * a.d + c);
    T* g = (T*)(a.gq + b * a.gqs[0] + qi * a.gqs[1] + head * a.gqs[2]) + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = (T)(s[e] * a.scale);
  }
}

// ---- backward: dk, dv ----------------------------------------------------------------------------------------------------------------
// A wave owns 32 keys (operands and both accumulators in registers); the workgroup's four waves walk the query tiles that may see its 128
// keys, once for every head of the group: the gradient of a shared head is one sum in one place.  Blocks that hold sinks see every query,
// and few blocks leave CUs idle: blocks [0, nsb) share their walk between nsplit workgroups, whose partial sums a second kernel adds in
// a fixed order.  128 channels hold 420 registers, one wave a SIMD: 2 x 4096, window 1024, 16 / 4 heads fp16 in 256 us, 470 TFLOP/s of its four products,
// a third of the time waiting; 64 channels run two waves: 16 x 2048, window 256 both ways, 4 heads in 90 us, 360 TFLOP/s, bound by issue slots.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP <= 64 && sizeof(T) == 2 ? 2 : 1) void attn_bwd_kv_kernel(AttnArgs a) {
  constexpr bool kAhead = kAheadOf<T>;
  constexpr int NW = 4, BQ = sizeof(T) == 2 ? 64 : 32, DL = lds_width(DP), NT = NW * 64, KS = DP / 16, MT = (DP + 31) / 32;
  using TL = Tile<T, DL>;
  __shared__ uint4 sQ[BQ * TL::CH], sG[BQ * TL::CH];
  __shared__ float sL[BQ], sD[BQ];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int per = a.nblk + a.nsb * (a.nsplit - 1);            // workgroups a (batch, key head)
  const int id = xcd_order(blockIdx.x, gridDim.x), bh = id / per, it = id - bh * per;
  const bool part = it < a.nsb * a.nsplit && a.nsplit > 1;
  const int blk = part ? it / a.nsplit : it - a.nsb * (a.nsplit - 1), sp = part ? it - blk * a.nsplit : 0;
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const Vis vis = vis_of(a, b);
  const int k0 = blk * 32 * NW, k1 = min(k0 + 32 * NW, a.lk) - 1;
  const int kw0 = k0 + wv * 32, kw1 = min(kw0 + 31, a.lk - 1);
  const int key = kw0 + (lane & 31);
  const bool seen = key < vis.len;
  const Range rows = vis.rows();
  Range lrows = vis.queries(key);                            // the lane's queries; none behind the last one
  lrows.n = min(lrows.n, (unsigned)max(vis.start + a.lq - lrows.lo, 0));

  // queries that may see a key of [k0, k1]
  int ilo = 0, ihi = k0 < vis.len ? a.lq - 1 : -1;
  if (vis.causal) ilo = max(ilo, k0 - vis.start);
  if (vis.window && k0 >= vis.sinks) {
    ihi = min(ihi, k1 + vis.window - 1 - vis.start);
    ilo = max(ilo, k0 - vis.window + 1 - vis.start);
  }
  const int q0 = ilo / BQ, nq = ihi >= ilo ? ihi / BQ - q0 + 1 : 0;
  int t0 = 0, t1 = nq * a.g;
  if (part) {
    const int n = (t1 + a.nsplit - 1) / a.nsplit;
    t0 = min(sp * n, t1);
    t1 = min(t0 + n, t1);
  }

  f16_t dk[MT], dv[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) dk[m] = dv[m] = f16_t{};
  constexpr bool kUp = sizeof(T) == 2;
  int up = kUp ? kMostUp - (int)kPShift<T> : 0;              // what 2^kPShift dS and dk of the lane's key are lifted by
  float upf = __builtin_amdgcn_ldexpf(1.f, up);

  Stage<T, DP, BQ, NT> gq, gg;
  float nl = 0.f, nd = 0.f;
  auto fetch = [&](int t) {
    const int hd = t / nq, i0 = (q0 + t - hd * nq) * BQ, head = kh * a.g + hd;
    // rows behind the last query and rows that see nothing enter as zeros, whatever they hold
    auto ok = [&](int r) { return (i0 + r < a.lq) & rows.has(vis.start + i0 + r); };
    gq.load(a.q + b * a.qs[0] + head * a.qs[2] + (int64_t)i0 * a.qs[1], a.qs[1], a.d, tid, ok);
    gg.load(a.go + b * a.gos[0] + head * a.gos[2] + (int64_t)i0 * a.gos[1], a.gos[1], a.d, tid, ok);
    if (tid < BQ) {
      const bool on = ok(tid);
      const int64_t lr = ((int64_t)b * a.hq + head) * a.lq + (on ? i0 + tid : 0);
      nl = on ? kPShift<T> - a.lse[lr] : 0.f;
      nd = on ? -a.delta[lr] : 0.f;
    }
  };
  auto put = [&]() {
    gq.template store<DL>(sQ, tid);
    gg.template store<DL>(sG, tid);
    if (tid < BQ) { sL[tid] = nl; sD[tid] = nd; }
  };
  if (t0 < t1) fetch(t0);                                  // (in flight beside the key operands)
  Frag<T> kf[KS], vf[KS];
  const char* kp = a.k + b * a.ks[0] + kh * a.ks[2] + (int64_t)key * a.ks[1];
  const char* vp = a.v + b * a.vs[0] + kh * a.vs[2] + (int64_t)key * a.vs[1];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int c = s * 16 + h * 8;
    frag_global(kf[s], kp + c * sizeof(T), seen & (c < a.d));
    frag_global(vf[s], vp + c * sizeof(T), seen & (c < a.d));
  }
  if (t0 < t1) put();
  for (int t = t0; t < t1; ++t) {
    const int hd = t / nq, i0 = (q0 + t - hd * nq) * BQ;
    const bool more = t + 1 < t1;
    __syncthreads();
    if (more) fetch(t + 1);
    const int p0 = vis.start + i0, p1 = p0 + BQ - 1;
    if ((kw0 <= kw1) & vis.any(p0, p1, kw0, kw1)) {
      const bool all = kw0 + 31 < a.lk && i0 + BQ <= a.lq && vis.all(p0, p1, kw0, kw1);
#pragma unroll 1
      for (int u = 0; u < BQ / 32; ++u) {
        // fp16: the row operands of both products are read ahead of their matrix instructions, the column operands a step ahead, so that exp
        // runs beside the second product and dS beside dv (fp32 operands are twice the registers and a sixteenth of the rate: read in place)
        f16_t s = f16_t{}, dp = f16_t{};
        if constexpr (kAhead) {
          Frag<T> fq[KS], fg[KS];
#pragma unroll
          for (int k = 0; k < KS; ++k) TL::row_frag(fq[k], sQ, u * 32 + (lane & 31), k * 2 + h);
#pragma unroll
          for (int k = 0; k < KS; ++k) TL::row_frag(fg[k], sG, u * 32 + (lane & 31), k * 2 + h);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < KS; ++k) s = mma(fq[k], kf[k], s);
#pragma unroll
          for (int k = 0; k < KS; ++k) dp = mma(fg[k], vf[k], dp);
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            Frag<T> f;
            TL::row_frag(f, sQ, u * 32 + (lane & 31), k * 2 + h);
            s = mma(f, kf[k], s);
            TL::row_frag(f, sG, u * 32 + (lane & 31), k * 2 + h);
            dp = mma(f, vf[k], dp);
          }
        }
        Columns<T, DL, kAhead> cg(sG, u * 32, lane), cq(sQ, u * 32, lane);
        cg.first();
        f4_t l4[4], d4[4];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          l4[r4] = *reinterpret_cast<const f4_t*>(sL + u * 32 + 8 * r4 + 4 * h);
          d4[r4] = *reinterpret_cast<const f4_t*>(sD + u * 32 + 8 * r4 + 4 * h);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.sl2, l4[r >> 2][r & 3]));
        if (!all) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = lrows.has(p0 + u * 32 + (r & 3) + 8 * (r >> 2) + 4 * h) ? s[r] : 0.f;
        }
        Frag<T> f0, f1;
        frag_from<0>(f0, s);
        frag_from<1>(f1, s);
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = s[r] * (dp[r] + d4[r >> 2][r & 3]);
        if (!all) {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] = lrows.has(p0 + u * 32 + (r & 3) + 8 * (r >> 2) + 4 * h) ? dp[r] : 0.f;
        }
        if constexpr (kUp) {
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dp[r]));
          if (__builtin_expect(__any(top * upf > kTop), 0)) {
            // (held where the matrix instructions keep them up to here: else the allocator copies all of dk out for this branch in every step)
            if constexpr (DP > 64) {
#pragma unroll
              for (int m = 0; m < MT; ++m) asm("" : "+a"(dk[m]));
            }
            top = half_max(top);
            const int to = top * upf > kTop ? to_room(top) : up;
            const float f = __builtin_amdgcn_ldexpf(1.f, to - up);
            up = to;
            upf = __builtin_amdgcn_ldexpf(1.f, up);
#pragma unroll
            for (int r = 0; r < 16; ++r) {                   // (the sums' rows are keys, other lanes' own)
              const float fr = __shfl(f, (r & 3) + 8 * (r >> 2) + 4 * h, 64);
#pragma unroll
              for (int m = 0; m < MT; ++m) dk[m][r] *= fr;
            }
            if constexpr (DP > 64) {
#pragma unroll
              for (int m = 0; m < MT; ++m) asm("" : "+a"(dk[m]));
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= upf;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m + 1 < MT) cg.next(m); else cq.first();
          cg.now(m);
          dv[m] = mma(f0, cg.a(m), dv[m]);
          dv[m] = mma(f1, cg.b(m), dv[m]);
        }
        frag_from<0>(f0, dp);
        frag_from<1>(f1, dp);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m + 1 < MT) cq.next(m);
          cq.now(m);
          dk[m] = mma(f0, cq.a(m), dk[m]);
          dk[m] = mma(f1, cq.b(m), dk[m]);
        }
      }
    }
    __syncthreads();
    if (more) put();
  }
  // accumulators: column (lane % 32) = channel, rows = keys
  const int col = lane & 31;
  if constexpr (kUp) {
    const float down = __builtin_amdgcn_ldexpf(kPUnshift<T>, -up);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float dr = __shfl(down, (r & 3) + 8 * (r >> 2) + 4 * h, 64);
#pragma unroll
      for (int m = 0; m < MT; ++m) dk[m][r] *= dr;
    }
  }
  if (part) {
    float* pk = a.part + (((int64_t)bh * a.nsb + blk) * a.nsplit + sp) * (2 * 32 * NW) * a.d;
    float* pv = pk + 32 * NW * a.d;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int o = (wv * 32 + (r & 3) + 8 * (r >> 2) + 4 * h) * a.d + m * 32 + col;
        if (m * 32 + col < a.d) { pk[o] = dk[m][r]; pv[o] = dv[m][r]; }
      }
    return;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int kk = kw0 + (r & 3) + 8 * (r >> 2) + 4 * h;
      if (kk < a.lk && m * 32 + col < a.d) {
        reinterpret_cast<T*>(a.gk + b * a.gks[0] + kh * a.gks[2] + (int64_t)kk * a.gks[1])[m * 32 + col] = (T)(dk[m][r] * a.scale);
        reinterpret_cast<T*>(a.gv + b * a.gvs[0] + kh * a.gvs[2] + (int64_t)kk * a.gvs[1])[m * 32 + col] = (T)(dv[m][r] * kPUnshift<T>);
      }
    }
}

// adds the partial sums of the split key blocks
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_kv_join_kernel(AttnArgs a) {
  const int c4 = a.d / 4, per = 2 * 128 * c4;
  const int64_t total = (int64_t)a.b * a.hk * a.nsb * per;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int64_t bb = v / per;
    const int q = (int)(v - bb * per), which = q / (128 * c4), o = q - which * 128 * c4, kr = o / c4, c = (o - kr * c4) * 4;
    const int bh = (int)(bb / a.nsb), kk = (int)(bb - (int64_t)bh * a.nsb) * 128 + kr, b = bh / a.hk, kh = bh - b * a.hk;
    if (kk >= a.lk) continue;
    const float* p = a.part + bb * a.nsplit * 2 * 128 * a.d + (int64_t)which * 128 * a.d + kr * a.d + c;
    f4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < a.nsplit; ++i) s += *reinterpret_cast<const f4_t*>(p + (int64_t)i * 2 * 128 * a.d);
    const float f = which ? kPUnshift<T> : a.scale;
    T* g = which ? (T*)(a.gv + b * a.gvs[0] + kh * a.gvs[2] + (int64_t)kk * a.gvs[1]) : (T*)(a.gk + b * a.gks[0] + kh * a.gks[2] + (int64_t)kk * a.gks[1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) g[c + e] = (T)(s[e] * f);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
bool desc_ok(const myolo_attn_desc* d) {
  return d && (d->dtype == MYOLO_F16 || d->dtype == MYOLO_F32) && d->b >= 0 && d->lq >= 0 && d->lk >= 0 && d->lq <= MYOLO_ATTN_MAX_LEN &&
         d->lk <= MYOLO_ATTN_MAX_LEN && d->hq >= 1 && d->hk >= 1 && d->hq % d->hk == 0 && d->d >= 8 && d->d <= 128 && d->d % 8 == 0 &&
         d->window >= 0 && d->window <= MYOLO_ATTN_MAX_LEN && d->sinks >= 0 && (int64_t)d->b * d->hq < (1 << 24) &&
         (int64_t)d->lq * (d->hq / d->hk) <= MYOLO_ATTN_MAX_LEN;
}
bool side_ok(const void* p, const int64_t* s, int es) {
  if (!p || (uintptr_t)p % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] * es % 16) return false;
  return true;
}
// keys a query may see, at most: what its tiles are shared out over
int64_t key_span(const myolo_attn_desc* d, int rows) {
  if (!d->window) return d->lk;
  const int64_t w = (int64_t)d->window * (d->causal ? 1 : 2) + d->sinks + rows / (d->hq / d->hk) + 128;
  return w < d->lk ? w : d->lk;
}
// workgroups of 256 threads that are resident at once: two a CU, one where a kernel's registers leave a SIMD one wave
int resident(const myolo_attn_desc* d) { return d->dtype == MYOLO_F16 || d->d <= 64 ? 512 : 256; }
bool fits(int64_t groups, int threads) { return groups * threads < (1ll << 32); }         // what one launch may hold
struct FwdShape { int nw, nblk, nsplit; };
FwdShape fwd_shape(const myolo_attn_desc* d) {
  const int64_t rows = (int64_t)d->lq * (d->hq / d->hk), bh = (int64_t)d->b * d->hk;
  FwdShape f;
  f.nw = rows > 32 ? 4 : 1;
  f.nblk = (int)((rows + 32 * f.nw - 1) / (32 * f.nw));
  // few workgroups over a long key axis: split it until every CU has four waves (single waves) or its two workgroups, a split keeping a tile
  const int64_t tiles = (key_span(d, 32 * f.nw) + 63) / 64, want = f.nw == 1 ? 1024 : resident(d), have = bh * f.nblk;
  int64_t n = have > 0 ? want / have : 1;
  if (n > tiles) n = tiles;
  if (n > kMaxSplit) n = kMaxSplit;
  f.nsplit = n < 2 ? 1 : (int)n;
  return f;
}
int q_split(const myolo_attn_desc* d) {
  const int64_t blocks = ((int64_t)d->lq * (d->hq / d->hk) + 127) / 128 * d->b * d->hk, tiles = (key_span(d, 128) + 63) / 64;
  if (!blocks) return 1;
  int64_t n = resident(d) / blocks;
  if (n > tiles) n = tiles;
  if (n > 16) n = 16;
  return n < 2 ? 1 : (int)n;
}
struct KvShape { int nblk, nsb, nsplit; };
KvShape kv_shape(const myolo_attn_desc* d) {
  const int bq = d->dtype == MYOLO_F16 ? 64 : 32;
  const int64_t g = d->hq / d->hk, bh = (int64_t)d->b * d->hk;
  KvShape k{(d->lk + 127) / 128, 0, 1};
  const int64_t full = (d->lq + bq - 1) / bq * g, total = bh * k.nblk;
  if (!total || !full) return k;
  int64_t n = 1;
  const int64_t fill = d->d <= 64 && d->dtype == MYOLO_F16 ? 512 : 256;       // workgroups that are resident at once
  if (d->window && d->sinks) {
    // a block of sinks walks every query, its neighbours the band.  Cut it to the band's length where several rounds of workgroups follow it,
    // to eighths of that where the last round would wait for it (8 x 32 blocks of 128 channels: 300 -> 271 us; 64 x 16 blocks of 64: 92 -> 98)
    const int64_t band = (((int64_t)d->window * (d->causal ? 1 : 2) + 127) / bq + 2) * g;
    if (full > band) {
      n = ((total < 2 * fill ? 8 : 1) * full + band - 1) / band;
      k.nsb = (int)(((d->sinks < d->lk ? d->sinks : d->lk) + 127) / 128);
    }
  }
  if (total < fill) {                   // CUs would idle: every block is shared
    k.nsb = k.nblk;
    const int64_t w = (fill + total - 1) / total;
    if (w > n) n = w;
  }
  if (n > full) n = full;
  if (n > 32) n = 32;
  while (n > 1 && bh * k.nsb * n * 256 * d->d * 4 > (256ll << 20)) --n;      // scratch stays under 256 MiB
  k.nsplit = (int)n;
  if (n == 1) k.nsb = 0;
  return k;
}
int64_t delta_bytes(const myolo_attn_desc* d) { return ((int64_t)d->b * d->hq * d->lq * 4 + 15) / 16 * 16; }
void bytes3(int64_t* o, const int64_t* s, int64_t es) { for (int i = 0; i < 3; ++i) o[i] = s[i] * es; }
AttnArgs args_of(const myolo_attn_desc* d) {
  const int64_t es = d->dtype == MYOLO_F16 ? 2 : 4;
  AttnArgs a{};
  a.q = (const char*)d->q; a.k = (const char*)d->k; a.v = (const char*)d->v; a.o = (char*)d->o; a.ores = d->dtype == MYOLO_F16 ? (char*)d->o_res : nullptr; a.go = (const char*)d->go;
  a.gq = (char*)d->gq; a.gk = (char*)d->gk; a.gv = (char*)d->gv;
  a.lse = d->lse; a.lens = d->lens; a.starts = d->starts;
  bytes3(a.qs, d->qs, es); bytes3(a.ks, d->ks, es); bytes3(a.vs, d->vs, es); bytes3(a.os, d->os, es);
  bytes3(a.gos, d->gos, es); bytes3(a.gqs, d->gqs, es); bytes3(a.gks, d->gks, es); bytes3(a.gvs, d->gvs, es);
  a.b = d->b; a.lq = d->lq; a.lk = d->lk; a.hq = d->hq; a.hk = d->hk; a.g = d->hq / d->hk; a.d = d->d;
  a.causal = d->causal ? 1 : 0; a.window = d->window; a.sinks = d->sinks < d->lk ? d->sinks : d->lk;
  a.rows = d->lq * a.g; a.nsplit = 1;
  a.scale = d->scale; a.sl2 = d->scale * kLog2e;
  return a;
}

template <typename T, int DP, int NW>
int launch_fwd(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.b * a.hk * a.nblk * a.nsplit));
  if (a.nsplit > 1) {
    hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW, true>), grid, dim3(NW * 64), 0, st, a);
    MYOLO_CHECK_LAUNCH();
    const int64_t nrow = (int64_t)a.b * a.hk * a.rows;
    if (a.nsplit <= kFewSplits) hipLaunchKernelGGL((attn_join_few_kernel<T>), dim3(grid_for(nrow * (a.d / 4), 256, 4096)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_join_kernel<T>), dim3(grid_for(nrow, 1, 1 << 16)), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW, false>), grid, dim3(NW * 64), 0, st, a);
  }
  MYOLO_CHECK_LAUNCH();
  return 0;
}
template <typename T, int DP> int launch_fwd_w(const AttnArgs& a, int nw, hipStream_t st) {
  return nw == 4 ? launch_fwd<T, DP, 4>(a, st) : launch_fwd<T, DP, 1>(a, st);
}
template <typename T> int run_fwd(const AttnArgs& a, int nw, hipStream_t st) {
  if (a.d <= 32) return launch_fwd_w<T, 32>(a, nw, st);
  if (a.d <= 48) return launch_fwd_w<T, 48>(a, nw, st);
  if (a.d <= 64) return launch_fwd_w<T, 64>(a, nw, st);
  if (a.d <= 80) return launch_fwd_w<T, 80>(a, nw, st);
  if (a.d <= 96) return launch_fwd_w<T, 96>(a, nw, st);
  return launch_fwd_w<T, 128>(a, nw, st);
}
template <typename T, int DP> int launch_bwd(AttnArgs& a, const KvShape& kv, hipStream_t st) {
  a.nblk = (a.rows + 127) / 128;
  if (a.rows) {
    hipLaunchKernelGGL((attn_bwd_q_kernel<T, DP>), dim3((unsigned)((int64_t)a.b * a.hk * a.nblk * a.nsplit)), dim3(256), 0, st, a);
    MYOLO_CHECK_LAUNCH();
    if (a.nsplit > 1) {
      hipLaunchKernelGGL((attn_bwd_q_join_kernel<T>), dim3(grid_for((int64_t)a.b * a.hk * a.rows * (a.d / 4), 256, 4096)), dim3(256), 0, st, a);
      MYOLO_CHECK_LAUNCH();
    }
  }
  if (a.gk && a.lk) {
    const int64_t bh = (int64_t)a.b * a.hk;
    a.nblk = kv.nblk; a.nsb = kv.nsb; a.nsplit = kv.nsplit;
    hipLaunchKernelGGL((attn_bwd_kv_kernel<T, DP>), dim3((unsigned)(bh * (kv.nblk + kv.nsb * (kv.nsplit - 1)))), dim3(256), 0, st, a);
    MYOLO_CHECK_LAUNCH();
    if (kv.nsplit > 1) {
      hipLaunchKernelGGL((attn_bwd_kv_join_kernel<T>), dim3(grid_for(bh * kv.nsb * 2 * 128 * (a.d / 4), 256, 4096)), dim3(256), 0, st, a);
      MYOLO_CHECK_LAUNCH();
    }
  }
  return 0;
}
template <typename T> int run_bwd(AttnArgs& a, const KvShape& kv, hipStream_t st) {
  if (a.d <= 32) return launch_bwd<T, 32>(a, kv, st);
  if (a.d <= 48) return launch_bwd<T, 48>(a, kv, st);
  if (a.d <= 64) return launch_bwd<T, 64>(a, kv, st);
  if (a.d <= 80) return launch_bwd<T, 80>(a, kv, st);
  if (a.d <= 96) return launch_bwd<T, 96>(a, kv, st);
  return launch_bwd<T, 128>(a, kv, st);
}

}  // namespace

extern "C" int64_t myolo_attn_ws_bytes(const myolo_attn_desc* d, int backward) {
  if (!desc_ok(d)) return 0;
  if (backward) {
    const KvShape k = kv_shape(d);
    const int64_t kv = k.nsplit > 1 ? (int64_t)d->b * d->hk * k.nsb * k.nsplit * 256 * d->d * 4 : 0, nq = q_split(d);
    const int64_t q = nq > 1 ? nq * d->b * d->hq * d->lq * d->d * 4 : 0;
    return delta_bytes(d) + (q > kv ? q : kv);              // (dq's sums are joined before dk / dv's are formed)
  }
  const FwdShape f = fwd_shape(d);
  if (f.nsplit == 1) return 0;
  return (int64_t)f.nsplit * d->b * d->hq * d->lq * (d->d + 2) * 4;
}

extern "C" int myolo_attn_fwd(const myolo_attn_desc* d, void* stream) {
  if (!desc_ok(d) || !(d->scale > 0.f)) return MYOLO_EINVAL;
  if ((int64_t)d->b * d->lq == 0) return 0;
  const int es = d->dtype == MYOLO_F16 ? 2 : 4;
  if (d->o_res && (uintptr_t)d->o_res % 16) return MYOLO_EINVAL;
  if (!side_ok(d->q, d->qs, es) || !side_ok(d->o, d->os, es)) return MYOLO_EINVAL;
  if (d->lk && (!side_ok(d->k, d->ks, es) || !side_ok(d->v, d->vs, es))) return MYOLO_EINVAL;
  const FwdShape f = fwd_shape(d);
  AttnArgs a = args_of(d);
  a.nblk = f.nblk; a.nsplit = f.nsplit; a.part = (float*)d->ws;
  if (!fits((int64_t)a.b * a.hk * a.nblk * a.nsplit, f.nw * 64)) return MYOLO_EINVAL;
  if (f.nsplit > 1 && (!d->ws || (uintptr_t)d->ws % 16 || d->ws_bytes < myolo_attn_ws_bytes(d, 0))) return MYOLO_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return d->dtype == MYOLO_F16 ? run_fwd<half_t>(a, f.nw, st) : run_fwd<float>(a, f.nw, st);
}

extern "C" int myolo_attn_bwd(const myolo_attn_desc* d, void* stream) {
  if (!desc_ok(d) || !(d->scale > 0.f) || (d->gk == nullptr) != (d->gv == nullptr)) return MYOLO_EINVAL;
  if (d->b == 0 || (!d->gq && !d->gk)) return 0;
  const int es = d->dtype == MYOLO_F16 ? 2 : 4;
  if (d->o_res && (uintptr_t)d->o_res % 16) return MYOLO_EINVAL;
  if (d->lq && (!side_ok(d->q, d->qs, es) || !side_ok(d->o, d->os, es) || !side_ok(d->go, d->gos, es) || !d->lse)) return MYOLO_EINVAL;
  if (d->lk && (!side_ok(d->k, d->ks, es) || !side_ok(d->v, d->vs, es))) return MYOLO_EINVAL;
  if ((d->gq && d->lq && !side_ok(d->gq, d->gqs, es)) || (d->gk && d->lk && (!side_ok(d->gk, d->gks, es) || !side_ok(d->gv, d->gvs, es))))
    return MYOLO_EINVAL;
  if (d->lq && (!d->ws || (uintptr_t)d->ws % 16 || d->ws_bytes < myolo_attn_ws_bytes(d, 1))) return MYOLO_EINVAL;
  AttnArgs a = args_of(d);
  const KvShape kv = kv_shape(d);
  a.nsplit = d->gq ? q_split(d) : 1;
  if (!fits((int64_t)a.b * a.hk * ((a.rows + 127) / 128) * a.nsplit, 256) || !fits((int64_t)a.b * a.hk * (kv.nblk + (int64_t)kv.nsb * (kv.nsplit - 1)), 256))
    return MYOLO_EINVAL;
  a.delta = (float*)d->ws;
  a.part = (float*)((char*)d->ws + delta_bytes(d));
  hipStream_t st = (hipStream_t)stream;
  return d->dtype == MYOLO_F16 ? run_bwd<half_t>(a, kv, st) : run_bwd<float>(a, kv, st);
}
