// One AdamW step over many tensors at once, 32-bit states.
//
//   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2          (g: the gradient, divided by the loss scale where there is one)
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32 whatever p's and g's types; p is rounded once as it is stored, and rounded once more into a 16-bit working copy where the
// caller keeps one beside a 32-bit p.  The bias corrections come from the host in doubles (1 - b2^t of t = 1 would keep 4 digits
// in fp32), or from a one-thread kernel where the step count lives on the device (a captured step).
//
// Bound by HBM: p, m, v are read and written once, g is read once.  A launch takes up to TENSORS tensors: their pointers travel in the
// kernel's arguments (no table in memory that a later step or a replay could find overwritten), each tensor is cut into pieces
// of PIECE elements, one block each, and a block finds its tensor by bisection of the pieces' running count.
// Measured: 106 M fp32 parameters with bf16 gradients and copies 572 us (5.2 TB/s; a copy of 2 GiB reaches 4.9); 60 tensors of 240 ... 960 elements
// 6.5 us of 28 us that the call takes (the dispatcher takes 18 us to hand 240 tensors over).
#include "train_common.h"

namespace {

constexpr int TENSORS = 72;           // 72 x 52 bytes + scalars: inside 4 KiB of kernel arguments
constexpr int THR = 256, V = 4, UNROLL = 2, PIECE = THR * V * UNROLL * 2;

struct AdamwArgs {
  hi3d_adamw_tensor t[TENSORS];
  unsigned first[TENSORS];            // the first block of tensor i
  const float* dev;                   // coefficients in device memory, or NULL: those below
  hi3d_adamw_coefs_t c;
  int n;
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

template <typename P, typename G, typename W>
__global__ __launch_bounds__(THR) void adamw_kernel(const AdamwArgs a) {
  float shrink, size, root, b1, b2, a1, a2, eps, gs;
  if (a.dev) {
    if (a.dev[HI3D_ADAMW_SKIP] != 0.0f) return;        // a gradient was not finite: the step is not taken
    shrink = a.dev[0]; size = a.dev[1]; root = a.dev[2]; gs = a.dev[3];
  } else {
    shrink = a.c.shrink; size = a.c.step_size; root = a.c.inv_root; gs = a.c.grad_scale;
  }
  b1 = a.c.beta1; b2 = a.c.beta2; a1 = a.c.one_minus_beta1; a2 = a.c.one_minus_beta2; eps = a.c.eps;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const long base = (long)(blockIdx.x - a.first[lo]) * PIECE, count = a.t[lo].n;
  P* const p = (P*)a.t[lo].p;
  const G* const g = (const G*)a.t[lo].g;
  float* const m = a.t[lo].m;
  float* const v = a.t[lo].v;
  W* const c = (W*)a.t[lo].copy;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    Pack<P, V> kp[UNROLL];
    Pack<G, V> kg[UNROLL];
    Pack<float, V> km[UNROLL], kv[UNROLL];
    long e[UNROLL];
    int n[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      e[u] = base + ((h * UNROLL + u) * THR + threadIdx.x) * V;
      const long left = count - e[u];
      n[u] = left < V ? (int)(left < 0 ? 0 : left) : V;
      fetch(p + e[u], n[u], e[u], kp[u]);
      fetch(g + e[u], n[u], e[u], kg[u]);
      fetch(m + e[u], n[u], e[u], km[u]);
      fetch(v + e[u], n[u], e[u], kv[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float fp[V], fg[V], fm[V], fv[V];
      unpack(kp[u], fp); unpack(kg[u], fg); unpack(km[u], fm); unpack(kv[u], fv);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gr = fg[j] * gs;
        fm[j] = b1 * fm[j] + a1 * gr;
        fv[j] = b2 * fv[j] + a2 * gr * gr;
        fp[j] = fp[j] * shrink - size * (fm[j] / (sqrtf(fv[j]) * root + eps));
      }
      store_some(m + e[u], n[u], fm);
      store_some(v + e[u], n[u], fv);
      store_some(p + e[u], n[u], fp);
      if (c) store_some(c + e[u], n[u], fp);
    }
  }
}

// the coefficients of a step whose count (and learning rate, loss scale, overflow flag) live in device memory
__global__ void adamw_coefs_kernel(float* out, float* step, const float* lr_dev, const float* scale, const float* found_inf, hi3d_adamw_rates r) {
  const bool skip = found_inf && *found_inf != 0.0f;
  out[HI3D_ADAMW_SKIP] = skip ? 1.0f : 0.0f;
  if (skip) return;
  const float t = *step + 1.0f;
  *step = t;
  const double lr = lr_dev ? (double)*lr_dev : r.lr;
  out[0] = (float)(1.0 - lr * r.weight_decay);
  out[1] = (float)(lr / (1.0 - pow(r.beta1, (double)t)));
  out[2] = (float)(1.0 / sqrt(1.0 - pow(r.beta2, (double)t)));
  out[3] = scale ? (float)(1.0 / (double)*scale) : 1.0f;
}

template <typename P, typename G>
int launch(const AdamwArgs& a, unsigned blocks, int copy_dtype, hipStream_t st) {
  if (copy_dtype == HI3D_F16) hipLaunchKernelGGL((adamw_kernel<P, G, half_t>), dim3(blocks), dim3(THR), 0, st, a);
  else hipLaunchKernelGGL((adamw_kernel<P, G, bf16_t>), dim3(blocks), dim3(THR), 0, st, a);
  HI3D_LAUNCH_CHECK();
  return 0;
}
template <typename P>
int launch_g(const AdamwArgs& a, unsigned blocks, int gdtype, int copy_dtype, hipStream_t st) {
  if (gdtype == HI3D_F32) return launch<P, float>(a, blocks, copy_dtype, st);
  return gdtype == HI3D_BF16 ? launch<P, bf16_t>(a, blocks, copy_dtype, st) : launch<P, half_t>(a, blocks, copy_dtype, st);
}

}  // namespace

extern "C" int hi3d_adamw_coefs(float* out, float* step, const float* lr_dev, const float* grad_scale, const float* found_inf,
                                const hi3d_adamw_rates* rates, void* stream) {
  if (!out || !step || !rates) HI3D_FAIL(HI3D_EINVAL, "adamw_coefs: null pointer");
  hipLaunchKernelGGL(adamw_coefs_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, out, step, lr_dev, grad_scale, found_inf, *rates);
  HI3D_LAUNCH_CHECK();
  return 0;
}

extern "C" int hi3d_adamw_step(const hi3d_adamw_tensor* t, int32_t n, int32_t pdtype, int32_t gdtype, int32_t copy_dtype, const hi3d_adamw_coefs_t* c,
                               const float* coefs_dev, void* stream) {
  if (n < 0 || (n && !t) || !c) HI3D_FAIL(HI3D_EINVAL, "adamw_step: null pointer or negative count");
  if (!hi3d_known_dtype(pdtype) || !hi3d_known_dtype(gdtype) || (copy_dtype != HI3D_BF16 && copy_dtype != HI3D_F16))
    HI3D_FAIL(HI3D_EINVAL, "adamw_step: unknown element type");
  for (int i = 0; i < n; ++i) {
    if (t[i].n < 0 || t[i].n > (1L << 40)) HI3D_FAIL(HI3D_EINVAL, "adamw_step: bad element count");
    if (t[i].n && (!t[i].p || !t[i].g || !t[i].m || !t[i].v)) HI3D_FAIL(HI3D_EINVAL, "adamw_step: null tensor");
  }
  AdamwArgs a = {};
  a.c = *c; a.dev = coefs_dev;
  unsigned long blocks = 0;
  for (int i = 0; i < n; ++i) {
    if (!t[i].n) continue;
    const unsigned long need = (unsigned long)((t[i].n + PIECE - 1) / PIECE);
    if (a.n == TENSORS || (a.n && blocks + need > 0x7fffffffUL)) {
      const int rc = pdtype == HI3D_F32 ? launch_g<float>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream)
                   : pdtype == HI3D_BF16 ? launch_g<bf16_t>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream)
                                         : launch_g<half_t>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream);
      if (rc) return rc;
      a.n = 0; blocks = 0;
    }
    a.t[a.n] = t[i];
    a.first[a.n++] = (unsigned)blocks;
    blocks += need;
  }
  if (!a.n) return 0;
  return pdtype == HI3D_F32 ? launch_g<float>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream)
       : pdtype == HI3D_BF16 ? launch_g<bf16_t>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream)
                             : launch_g<half_t>(a, (unsigned)blocks, gdtype, copy_dtype, (hipStream_t)stream);
}
