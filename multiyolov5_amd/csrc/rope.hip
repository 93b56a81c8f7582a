// Rotary positions with several axes (time, height, width): pair j of a head is turned by 2 pi * turns[j] * pos[token][axis[j]].
//
//   (u, v) -> (u cos - v sin, v cos + u sin);   the backward is the opposite turn of the incoming gradient
//
// A position of 10^6 times a frequency of 1 is 10^6 radians: fp32 would keep 0.06 of the angle.  The turn count pos * turns[j] is formed in
// fp64 and reduced to [-1/2, 1/2) before sine and cosine are taken in fp32 (sincospi: no further argument reduction), so the angle is good
// to 2^-24 of a turn for positions up to 2^29.  The rotation is fp32, rounded once.
#include "myolo_dev.h"

namespace {

struct RopeSide { const char* x; char* o; int64_t sb, sl, sh, ob, ol, oh; int h; };     // strides in bytes
struct RopeArgs {
  RopeSide s[2];           // q, k
  const int64_t* pos;
  int64_t pb, pl, pa;
  int l, d, npair, interleaved;
  int64_t tokens;
  float sign;
  double turns[MYOLO_ROPE_MAX_PAIRS];
  unsigned char axis[MYOLO_ROPE_MAX_PAIRS];
};

__device__ __forceinline__ void turn_of(const RopeArgs& a, const int64_t* pos, int j, float* s, float* c) {
  const double t = (double)pos[a.axis[j] * a.pa] * a.turns[j];
  sincospif(2.f * (float)(t - rint(t)), s, c);
  *s *= a.sign;
}

// one thread a pair (and one a pass-through channel), heads of q and k in one index space
template <typename T>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs a) {
  const int items = a.npair + (a.d - 2 * a.npair), heads = a.s[0].h + a.s[1].h;
  const int64_t total = a.tokens * heads * items;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int it = (int)(v % items);
    const int64_t th = v / items;
    int h = (int)(th % heads);
    const int64_t tok = th / heads, b = tok / a.l, i = tok - b * a.l;
    const RopeSide& s = h < a.s[0].h ? a.s[0] : a.s[1];
    if (h >= a.s[0].h) h -= a.s[0].h;
    const T* x = (const T*)(s.x + b * s.sb + i * s.sl + h * s.sh);
    T* o = (T*)(s.o + b * s.ob + i * s.ol + h * s.oh);
    if (it < a.npair) {
      float sn, cs;
      turn_of(a, a.pos + b * a.pb + i * a.pl, it, &sn, &cs);
      const int c0 = a.interleaved ? 2 * it : it, c1 = a.interleaved ? 2 * it + 1 : it + a.npair;
      const float u = (float)x[c0], w = (float)x[c1];
      o[c0] = (T)(u * cs - w * sn);
      o[c1] = (T)(w * cs + u * sn);
    } else {
      o[it + a.npair] = x[it + a.npair];
    }
  }
}

// Vector path: a workgroup owns tb tokens.  It forms their sines and cosines once, in LDS, for all heads, behind the loads of what they will
// turn: a thread owns one 16-byte unit of pairs (SEG pairs (j, j + npair) in two vectors, or SEG / 2 neighbouring pairs in one) of HC heads of
// q or of k.  Adjacent lanes take adjacent units, then other heads of the token: HBM sees whole lines.  Units behind the pairs copy the
// pass-through channels.  HBM bound: 35154 tokens x 16 heads x 96 fp32 in 77 us (5.6 TB/s; 121 with the angles formed by every thread),
// 32768 tokens x 16 heads x 64 fp16 in 30 us (4.4 TB/s); one token of 40 heads 3.9 us.
template <typename T, bool IL, int HC> struct RopeItem {
  static constexpr int SEG = ET<T>::SEG, NP = IL ? SEG / 2 : SEG, NV = IL ? 1 : 2;
  uint4 in[HC][NV];
  char* o;
  int64_t ostep;
  int tl, un, n;           // token in the workgroup, unit, heads

  // item it of the workgroup: chunk ch < nq takes heads ch, ch + nq, ... of q, the others likewise of k
  __device__ __forceinline__ void load(const RopeArgs& a, int it, int units, int upt, int nq, int nch, int b, int i0) {
    const int per = upt * nch;
    tl = it / per;
    const int rem = it - tl * per, c = rem / upt;
    un = rem - c * upt;
    const bool isq = c < nq;
    const int h0 = isq ? c : c - nq, step = isq ? nq : nch - nq, heads = isq ? a.s[0].h : a.s[1].h;
    const int64_t i = i0 + tl;
    const int c0 = (un < units ? un * SEG : 2 * a.npair + (un - units) * SEG) * (int)sizeof(T);
    const char* x = isq ? a.s[0].x + (b * a.s[0].sb + i * a.s[0].sl + h0 * a.s[0].sh) : a.s[1].x + (b * a.s[1].sb + i * a.s[1].sl + h0 * a.s[1].sh);
    o = isq ? a.s[0].o + (b * a.s[0].ob + i * a.s[0].ol + h0 * a.s[0].oh) : a.s[1].o + (b * a.s[1].ob + i * a.s[1].ol + h0 * a.s[1].oh);
    const int64_t xstep = step * (isq ? a.s[0].sh : a.s[1].sh);
    ostep = step * (isq ? a.s[0].oh : a.s[1].oh);
    x += c0;
    o += c0;
    n = (heads - h0 + step - 1) / step;
#pragma unroll
    for (int k = 0; k < HC; ++k) {
      const char* xk = k < n ? x + k * xstep : zero_page();
      in[k][0] = ldg16(xk);
      if constexpr (!IL) in[k][1] = ldg16((k < n) & (un < units) ? xk + a.npair * (int)sizeof(T) : zero_page());
    }
  }
  __device__ __forceinline__ void turn(const RopeArgs& a, const float2* tab, int units) const {
    if (un >= units) {
#pragma unroll
      for (int k = 0; k < HC; ++k)
        if (k < n) stg16(o + k * ostep, in[k][0]);
      return;
    }
    float2 sc[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) sc[e] = tab[tl * a.npair + un * NP + e];
#pragma unroll
    for (int k = 0; k < HC; ++k) {
      if (k >= n) break;
      float u[SEG];
      Vec<T>::unpack(in[k][0], u);
      if constexpr (IL) {
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const float x = u[2 * e], y = u[2 * e + 1];
          u[2 * e] = x * sc[e].y - y * sc[e].x;
          u[2 * e + 1] = y * sc[e].y + x * sc[e].x;
        }
        stg16(o + k * ostep, Vec<T>::pack(u));
      } else {
        float v[SEG];
        Vec<T>::unpack(in[k][1], v);
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const float x = u[e], y = v[e];
          u[e] = x * sc[e].y - y * sc[e].x;
          v[e] = y * sc[e].y + x * sc[e].x;
        }
        stg16(o + k * ostep, Vec<T>::pack(u));
        stg16(o + k * ostep + a.npair * (int)sizeof(T), Vec<T>::pack(v));
      }
    }
  }
};

constexpr int kTable = 2048;         // (sine, cosine) entries of a workgroup: 16 KB

template <typename T, bool IL, int HC>
__global__ __launch_bounds__(256) void rope_vec_kernel(RopeArgs a, int units, int pass, int nq, int nch, int tb, int nb) {
  __shared__ float2 tab[kTable];
  const int upt = units + pass, per = upt * nch;
  const int64_t i0 = (int64_t)blockIdx.x * tb;
  const int nt = (int)min((int64_t)tb, a.l - i0), items = nt * per;
  for (int b = blockIdx.y; b < nb; b += gridDim.y) {
    RopeItem<T, IL, HC> cur;
    if (threadIdx.x < items) cur.load(a, threadIdx.x, units, upt, nq, nch, b, (int)i0);
    if (b != (int)blockIdx.y) __syncthreads();
    const int64_t* pos = a.pos + b * a.pb + i0 * a.pl;
    for (int e = threadIdx.x; e < nt * a.npair; e += 256) {
      const int t = e / a.npair, j = e - t * a.npair;
      float sn, cs;
      turn_of(a, pos + t * a.pl, j, &sn, &cs);
      tab[e] = float2{sn, cs};
    }
    __syncthreads();
    for (int it = threadIdx.x; it < items; it += 256) {
      if (it != (int)threadIdx.x) cur.load(a, it, units, upt, nq, nch, b, (int)i0);
      cur.turn(a, tab, units);
    }
  }
}

bool side_vec_ok(const RopeSide& s) {
  if (!s.h) return true;
  return !(((uintptr_t)s.x | (uintptr_t)s.o | s.sb | s.sl | s.sh | s.ob | s.ol | s.oh) & 15);
}

template <typename T> int run_rope(const RopeArgs& a, hipStream_t st) {
  constexpr int SEG = ET<T>::SEG;
  const int np = a.interleaved ? SEG / 2 : SEG, heads = a.s[0].h + a.s[1].h;
  auto any = [&]() {
    const int grid = grid_for(a.tokens * heads * (a.d - a.npair), 256, 1 << 20);
    hipLaunchKernelGGL(rope_any_kernel<T>, dim3(grid), dim3(256), 0, st, a);
    MYOLO_CHECK_LAUNCH();
    return 0;
  };
  if (!(a.npair % np == 0 && (a.d - 2 * a.npair) % SEG == 0 && side_vec_ok(a.s[0]) && side_vec_ok(a.s[1]))) return any();
  const int units = a.npair / np, pass = (a.d - 2 * a.npair) / SEG, upt = units + pass;
  // four heads a thread where that still leaves sixteen waves for every CU, one where the call is that small
  const int hc = a.tokens * heads * upt >= 4 * 16 * 256 * 64 ? 4 : 1;
  const int nq = (a.s[0].h + hc - 1) / hc, nch = nq + (a.s[1].h + hc - 1) / hc, per = upt * nch;
  int tb = 256 / per;                                    // one item a thread; a token at least
  if (tb < 1) tb = 1;
  if (tb > a.l) tb = a.l;
  while (tb > 1 && tb * a.npair > kTable) --tb;          // (npair <= 128: one token always fits)
  const int nb = (int)(a.tokens / a.l);
  if ((a.l - 1) / tb >= (1 << 24) - 1) return any();     // (2^32 threads in one dimension)
  const dim3 grid((unsigned)((a.l - 1) / tb + 1), (unsigned)(nb < 65535 ? nb : 65535));
#define ROPE(IL, HC) hipLaunchKernelGGL((rope_vec_kernel<T, IL, HC>), grid, dim3(256), 0, st, a, units, pass, nq, nch, tb, nb)
  if (a.interleaved) { if (hc == 4) ROPE(true, 4); else ROPE(true, 1); }
  else { if (hc == 4) ROPE(false, 4); else ROPE(false, 1); }
#undef ROPE
  MYOLO_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int myolo_rope(const myolo_rope_desc* d, void* stream) {
  if (!d || (d->dtype != MYOLO_F16 && d->dtype != MYOLO_F32) || !d->turns || !d->axis) return MYOLO_EINVAL;
  if (d->b < 0 || d->l < 0 || d->hq < 1 || d->hk < 0 || d->d < 1 || d->npair < 0 || 2 * d->npair > d->d || d->npair > MYOLO_ROPE_MAX_PAIRS)
    return MYOLO_EINVAL;
  if (d->naxis < 1 || d->naxis > MYOLO_ROPE_MAX_AXES) return MYOLO_EINVAL;
  for (int j = 0; j < d->npair; ++j)
    if (d->axis[j] < 0 || d->axis[j] >= d->naxis) return MYOLO_EINVAL;
  if (((int64_t)d->hq + d->hk) * d->d > MYOLO_ROPE_MAX_TOKEN) return MYOLO_EINVAL;       // (items of a token are counted in 32 bits)
  const int64_t tokens = (int64_t)d->b * d->l;
  if (tokens == 0) return 0;
  if (!d->q || !d->qo || !d->pos || (d->hk && (!d->k || !d->ko))) return MYOLO_EINVAL;
  const int64_t es = d->dtype == MYOLO_F16 ? 2 : 4;
  RopeArgs a{};
  a.s[0] = RopeSide{(const char*)d->q, (char*)d->qo, d->qs[0] * es, d->qs[1] * es, d->qs[2] * es, d->qos[0] * es, d->qos[1] * es, d->qos[2] * es, d->hq};
  a.s[1] = RopeSide{(const char*)d->k, (char*)d->ko, d->ks[0] * es, d->ks[1] * es, d->ks[2] * es, d->kos[0] * es, d->kos[1] * es, d->kos[2] * es, d->hk};
  a.pos = d->pos; a.pb = d->ps[0]; a.pl = d->ps[1]; a.pa = d->ps[2];
  a.l = d->l; a.d = d->d; a.npair = d->npair; a.interleaved = d->interleaved; a.tokens = tokens;
  a.sign = d->inverse ? -1.f : 1.f;
  for (int j = 0; j < d->npair; ++j) { a.turns[j] = d->turns[j]; a.axis[j] = (unsigned char)d->axis[j]; }
  hipStream_t st = (hipStream_t)stream;
  return d->dtype == MYOLO_F16 ? run_rope<half_t>(a, st) : run_rope<float>(a, st);
}
