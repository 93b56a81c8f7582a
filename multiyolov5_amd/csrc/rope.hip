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

}  // namespace

extern "C" int myolo_rope(const myolo_rope_desc* d, void* stream) {
  if (!d || (d->dtype != MYOLO_F16 && d->dtype != MYOLO_F32) || !d->turns || !d->axis) return MYOLO_EINVAL;
  if (d->b < 0 || d->l < 0 || d->hq < 1 || d->hk < 0 || d->d < 1 || d->npair < 0 || 2 * d->npair > d->d || d->npair > MYOLO_ROPE_MAX_PAIRS)
    return MYOLO_EINVAL;
  if (d->naxis < 1 || d->naxis > MYOLO_ROPE_MAX_AXES) return MYOLO_EINVAL;
  for (int j = 0; j < d->npair; ++j)
    if (d->axis[j] < 0 || d->axis[j] >= d->naxis) return MYOLO_EINVAL;
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
  const int grid = grid_for(tokens * (d->hq + d->hk) * (d->d - d->npair), 256, 1 << 20);
  if (d->dtype == MYOLO_F16) hipLaunchKernelGGL(rope_any_kernel<half_t>, dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(rope_any_kernel<float>, dim3(grid), dim3(256), 0, st, a);
  MYOLO_CHECK_LAUNCH();
  return 0;
}
