// LayerNorm for training: forward with its statistics (and the residual sum in front of it), backward with the gradients of
// weight and bias.  Beside hi3d_layernorm, which is the sampler's form of it.
//
//   z = x (+ residual, rounded to x's type)        mu = mean(z)   s = 1 / sqrt(mean((z - mu)^2) + eps)     h = (z - mu) s
//   y = h w + b
//   dz = s (w dy - mean(w dy) - h mean(w dy h)) (+ the gradient that z's other reader sends)
//   dw = sum over rows of dy h                     db = sum over rows of dy
//
// Both directions are bound by HBM: every element of x and dy is read once and every element of y and dx is written once, the
// row's sums are taken from registers (two passes over them: the variance is of the differences, so a row whose mean is
// large against its spread keeps its digits), all in fp32.
//
// A row is held by LPR lanes of a wave (8 ... 64) as NV vectors of 16 bytes each, so that a wave carries 64 / LPR rows at a
// time and a row sum is log2(LPR) steps for all of them at once; wider rows are held by the block (LPR = 256 or 512).
//
// Measured, bf16 rows with fp32 weights: residual sum + norm of 262144 x 320 126 us (5.3 TB/s; a copy of 2 GiB reaches 4.9), norm of 65536 x 640
// 27.6 us (6.1 TB/s: half of it stays in the last-level cache), gradients of 65536 x 640 with the residual stream's 72 us (4.7 TB/s, 5 us of it the
// columns' sums), of 7013 x 1285 fp16 22 us (2.4 TB/s: too few rows to hide a row's latency).
#include "train_common.h"

namespace {

struct NormFwdParams {
  const void* x; const void* r; const void* w; const void* b;
  void* y; void* z; float* mean; float* rstd;
  long R, ldx, ldr;
  int C, wcode;
  float eps;
};
struct NormBwdParams {
  const void* dy; const void* z; const void* dz; const void* w; const float* mean; const float* rstd;
  void* dx; float* part; void* dw; void* db;
  long R, lddy, ldz, lddz;
  int C, wcode, want;       // want: partial sums of dw, db are asked for
};

// A row's vectors as one lane holds them: vector i covers elements at[i] ... at[i] + V of the row, n[i] of which exist.  The one that the
// row's end cuts is read so that it ends there and moved down once all of the row's loads are out (`settle`).  TINY: rows shorter than a
// vector, element by element.
template <typename T, int LPR, int NV, bool TINY>
struct RowMap {
  static constexpr int V = Elem<T>::VEC;
  int n[NV];
  int cut;                                // which of a lane's vectors the end of the row can cut; -1: none
  __device__ __forceinline__ RowMap(int l, int C) {
#pragma unroll
    for (int i = 0; i < NV; ++i) n[i] = C - (l + i * LPR) * V;
    cut = C % V != 0 ? C / V / LPR : -1;
  }
  __device__ __forceinline__ void load(const T* row, int l, bool in, Pack<T, V> (&k)[NV]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (l + i * LPR) * V;
      if constexpr (TINY) fetch(row + e, in ? n[i] : 0, 0, k[i]);
      else {
#pragma unroll
        for (int j = 0; j < Pack<T, V>::W; ++j) k[i].w[j] = 0;
        if (in && n[i] > 0) k[i] = *(const Pack<T, V>*)(row + e - max(0, V - n[i]));
      }
    }
  }
  __device__ __forceinline__ void settle(Pack<T, V> (&k)[NV]) const {
    if constexpr (!TINY) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == cut) shift_down(k[i], n[i] > 0 && n[i] < V ? V - n[i] : 0);
    }
  }
  // a weight or bias of the run-time type `code` in the lane's columns (1 or 0 where there is none)
  __device__ __forceinline__ void columns(const void* p, int code, int l, float none, float (&f)[NV][V]) const {
    if (!p) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) f[i][j] = none;
    } else if (code == HI3D_F32) columns_of((const float*)p, l, f);
    else if (code == HI3D_BF16) columns_of((const bf16_t*)p, l, f);
    else columns_of((const half_t*)p, l, f);
  }
  template <typename W>
  __device__ __forceinline__ void columns_of(const W* p, int l, float (&f)[NV][V]) const {
    Pack<W, V> k[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch(p + (l + i * LPR) * V, n[i], (l + i * LPR) * V, k[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack(k[i], f[i]);
  }
  __device__ __forceinline__ void store(T* row, int l, bool in, int i, const float (&f)[V]) const { store_some(row + (l + i * LPR) * V, in ? n[i] : 0, f); }
};

// sum over the lanes that hold a row; the block form goes through LDS (`slot` alternates, so that one barrier per sum is enough)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* lds, int& slot) {
  if constexpr (LPR <= 64) return group_sum<LPR>(v);
  constexpr int WAVES = LPR / 64;
  v = group_sum<64>(v);
  float* s = lds + (slot & 1) * WAVES;
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  ++slot;
  v = s[0];
#pragma unroll
  for (int k = 1; k < WAVES; ++k) v += s[k];
  return v;
}
constexpr int threads_of(int lpr) { return lpr < 256 ? 256 : lpr; }

template <typename T, int LPR, int NV, bool ADD, bool TINY>
__global__ __launch_bounds__(threads_of(LPR)) void norm_fwd_kernel(const NormFwdParams p) {
  constexpr int V = Elem<T>::VEC, THR = threads_of(LPR), RPB = THR / LPR;
  __shared__ float lds[2 * THR / 64];
  int slot = 0;
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR, C = p.C;
  const RowMap<T, LPR, NV, TINY> map(l, C);
  float w[NV][V], b[NV][V];
  map.columns(p.w, p.wcode, l, 1.0f, w);
  map.columns(p.b, p.wcode, l, 0.0f, b);
  const bool ragged = C != LPR * NV * V;
  const float inv = 1.0f / (float)C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < p.R; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + sub;
    const bool in = r < p.R;                    // (a whole group of lanes at a time; the others run along on zeros)
    float x[NV][V];
    float s = 0.0f;
    Pack<T, V> kx[NV], kr[ADD ? NV : 1];
    map.load((const T*)p.x + r * p.ldx, l, in, kx);
    if constexpr (ADD) { map.load((const T*)p.r + r * p.ldr, l, in, kr); map.settle(kr); }
    map.settle(kx);
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack(kx[i], x[i]);
    if constexpr (ADD) {
      float q[NV][V];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        unpack(kr[i], q[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) x[i][j] = Elem<T>::get(Elem<T>::put(x[i][j] + q[i][j]));   // the values the backward pass reads
        map.store((T*)p.z + r * C, l, in, i, x[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += x[i][j];
    const float mu = row_sum<LPR>(s, lds, slot) * inv;
    if (ragged) {                               // slots behind the row differ from the mean by nothing
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) x[i][j] = j < map.n[i] ? x[i][j] : mu;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) { x[i][j] -= mu; q += x[i][j] * x[i][j]; }
    const float rs = __builtin_amdgcn_rsqf(row_sum<LPR>(q, lds, slot) * inv + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = x[i][j] * rs * w[i][j] + b[i][j];
      map.store((T*)p.y + r * C, l, in, i, y);
    }
    if (in && l == 0) { p.mean[r] = mu; p.rstd[r] = rs; }
  }
}

// the gradients of a block's rows: dx, and -- where they are asked for -- the block's sums of dy h and dy, in columns held by
// the lane through all of its rows: nothing is added atomically, the order of the sums is that of the rows
template <typename T, int LPR, int NV, bool TINY>
__global__ __launch_bounds__(threads_of(LPR)) void norm_bwd_kernel(const NormBwdParams p) {
  constexpr int V = Elem<T>::VEC, THR = threads_of(LPR), RPB = THR / LPR;
  __shared__ float lds[2 * THR / 64];
  constexpr int WIDTH = LPR * NV * V;
  __shared__ float cols[LPR <= 64 ? 8 * WIDTH : 1];            // [wave][weight, bias][column, as the lanes hold them]
  int slot = 0;
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR, C = p.C;
  const RowMap<T, LPR, NV, TINY> map(l, C);
  float w[NV][V], gw[NV][V] = {}, gb[NV][V] = {};
  map.columns(p.w, p.wcode, l, 1.0f, w);
  const float inv = 1.0f / (float)C;
  for (long r0 = (long)blockIdx.x * RPB; r0 < p.R; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + sub;
    const bool in = r < p.R;
    Pack<T, V> ky[NV], kz[NV], kd[NV];
    map.load((const T*)p.dy + r * p.lddy, l, in, ky);                   // (zero behind the row: adds nothing below)
    map.load((const T*)p.z + r * p.ldz, l, in, kz);
    if (p.dz) map.load((const T*)p.dz + r * p.lddz, l, in, kd);
    const float mu = in ? p.mean[r] : 0.0f, rs = in ? p.rstd[r] : 0.0f;
    float dy[NV][V], h[NV][V];
    map.settle(ky);
    map.settle(kz);
    if (p.dz) map.settle(kd);
#pragma unroll
    for (int i = 0; i < NV; ++i) { unpack(ky[i], dy[i]); unpack(kz[i], h[i]); }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = j < map.n[i] ? (h[i][j] - mu) * rs : 0.0f;
        gb[i][j] += dy[i][j];
        gw[i][j] += dy[i][j] * h[i][j];
        dy[i][j] *= w[i][j];
        s1 += dy[i][j];
        s2 += dy[i][j] * h[i][j];
      }
    s1 = row_sum<LPR>(s1, lds, slot) * inv;
    s2 = row_sum<LPR>(s2, lds, slot) * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = (dy[i][j] - s1 - h[i][j] * s2) * rs;
      if (p.dz) {
        float t[V];
        unpack(kd[i], t);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] += t[j];
      }
      map.store((T*)p.dx + r * C, l, in, i, o);
    }
  }
  if (!p.want) return;
  // the lanes that held the same columns: over the wave's row groups by shuffles, over the waves through LDS
  // (written in the order of the columns: whole lines)
  float* const part = p.part + (long)blockIdx.x * 2 * C;
  void* const out[2] = {p.dw, p.db};
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        t[j] = k ? gb[i][j] : gw[i][j];
        if constexpr (LPR < 64) {
#pragma unroll
          for (int o = LPR; o < 64; o <<= 1) t[j] += __shfl_xor(t[j], o, 64);
        }
        if constexpr (LPR <= 64)
          if ((threadIdx.x & 63) < LPR) cols[((threadIdx.x >> 6) * 2 + k) * WIDTH + (i * V + j) * LPR + l] = t[j];
      }
      if constexpr (LPR > 64) {
        const int e = (l + i * LPR) * V;
        if (p.part) store_some(part + k * C + e, map.n[i], t);
        else if (out[k]) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < map.n[i]) store_as(out[k], p.wcode, e + j, t[j]);
        }
      }
    }
  if constexpr (LPR <= 64) {
    __syncthreads();
    for (int q = threadIdx.x; q < 2 * C; q += THR) {
      const int k = q >= C, e = q - k * C, vec = e / V, i = vec / LPR, s = k * WIDTH + (i * V + e % V) * LPR + vec % LPR;
      const float v = (cols[s] + cols[2 * WIDTH + s]) + (cols[4 * WIDTH + s] + cols[6 * WIDTH + s]);
      if (p.part) part[q] = v;
      else if (out[k]) store_as(out[k], p.wcode, e, v);
    }
  }
}

// out0 / out1[c] = sum over the nblk partial rows of part[blk][0 / 1][c] in a fixed order: 64 slices of the rows, then two levels over the
// slices.  16 columns a block: few columns have to make enough blocks, and a slice's loads are all in flight.
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float* part, void* o0, void* o1, int code0, int code1, int nblk, int C, int width) {
  __shared__ float lds[64][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + tx;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int b = ty; b < nblk; b += 64) s += part[(long)b * width + c];
  }
  lds[ty][tx] = s;
  __syncthreads();
  if (ty < 8) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += lds[ty * 8 + k][tx];
  }
  __syncthreads();
  if (ty < 8) lds[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < width) {
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += lds[k][tx];
    if (c < C) { if (o0) store_as(o0, code0, c, s); }
    else if (o1) store_as(o1, code1, c - C, s);
  }
}

// lanes per row and vectors per lane for a row of `chunks` vectors: the fewest lanes that hold it in at most `most` vectors each (more
// rows per wave, fewer steps per sum), then the fewest vectors of the forms that are built.  Forward holds 5 vectors (320, 640 and 1280
// columns of 16 bits fill 8, 16 and 32 lanes exactly); backward holds 3, since a lane also keeps its columns' sums: with 5 it had one wave
// a SIMD (85 us for 65536 x 640 against 71).
struct Shape { int lpr, nv; };
Shape pick(int chunks, int most) {
  for (int lpr = 8; ; lpr = lpr == 64 ? 256 : lpr * 2)
    if (chunks <= most * lpr || lpr == 512) return {lpr, chunks <= 2 * lpr ? 2 : chunks <= 3 * lpr ? 3 : most < 5 ? 4 : 5};
}

// whether pick() can give (lpr, nv) for a row of at most `chunks` vectors: what it cannot give is not built
constexpr bool given(int lpr, int nv, int most, int chunks) {
  const int before = lpr == 8 ? 0 : most * (lpr == 256 ? 64 : lpr / 2), fewer = nv == 2 ? 0 : nv == 3 ? 2 : 3;
  const int lo = before > fewer * lpr ? before : fewer * lpr, hi = nv > most && lpr < 512 ? 0 : nv * lpr;
  return lo < (hi < chunks ? hi : chunks);
}

constexpr int FWD_BLOCKS = 2048;      // 8 blocks of 4 waves a CU
// Backward, two blocks of 4 waves a CU (registers allow no more).  A block ends with 8 C bytes of partial sums, so that few rows take
// fewer blocks: 4 rows for each group of lanes, 8 where a row takes the block (7013 x 1280 bf16: 1, 2, 4, 8, 16 rows 27, 27, 21, 24, 33 us;
// 2000 x 5120: 37, 37, 29, 28, 37 us)
constexpr int BWD_BLOCKS = 512;
constexpr int bwd_rows(int lpr) { return lpr < 256 ? 4 : 8; }
constexpr int FWD_MOST = 5, BWD_MOST = 3;

long blocks_for(long R, int lpr, long most, int each) {
  const long rpb = (long)(threads_of(lpr) / lpr) * each, n = (R + rpb - 1) / rpb;
  return n < most ? n : most;
}

struct Launch { Shape s; unsigned grid; hipStream_t st; bool tiny; };

template <typename T, int LPR, int NV, bool TINY>
bool fwd_as(const NormFwdParams& p, const Launch& q) {
  if constexpr (TINY || given(LPR, NV, FWD_MOST, HI3D_NORM_MAX_WIDTH / Elem<T>::VEC)) {
    if (TINY ? !q.tiny : q.s.lpr != LPR || q.s.nv != NV) return false;
    if (p.r) hipLaunchKernelGGL((norm_fwd_kernel<T, LPR, NV, true, TINY>), dim3(q.grid), dim3(threads_of(LPR)), 0, q.st, p);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, LPR, NV, false, TINY>), dim3(q.grid), dim3(threads_of(LPR)), 0, q.st, p);
    return true;
  }
  return false;
}
template <typename T, int LPR, int NV, bool TINY>
bool bwd_as(const NormBwdParams& p, const Launch& q) {
  if constexpr (TINY || given(LPR, NV, BWD_MOST, HI3D_NORM_MAX_WIDTH / Elem<T>::VEC)) {
    if (TINY ? !q.tiny : q.s.lpr != LPR || q.s.nv != NV) return false;
    hipLaunchKernelGGL((norm_bwd_kernel<T, LPR, NV, TINY>), dim3(q.grid), dim3(threads_of(LPR)), 0, q.st, p);
    return true;
  }
  return false;
}
template <typename T, int LPR>
bool fwd_row(const NormFwdParams& p, const Launch& q) { return fwd_as<T, LPR, 2, false>(p, q) || fwd_as<T, LPR, 3, false>(p, q) || fwd_as<T, LPR, 5, false>(p, q); }
template <typename T, int LPR>
bool bwd_row(const NormBwdParams& p, const Launch& q) { return bwd_as<T, LPR, 2, false>(p, q) || bwd_as<T, LPR, 3, false>(p, q); }

template <typename T>
int launch_fwd(const NormFwdParams& p, hipStream_t st) {
  const Shape s = pick((p.C + Elem<T>::VEC - 1) / Elem<T>::VEC, FWD_MOST);
  const Launch q = {s, (unsigned)blocks_for(p.R, s.lpr, FWD_BLOCKS, 1), st, p.C < Elem<T>::VEC};
  const bool done = fwd_as<T, 8, 2, true>(p, q) || fwd_row<T, 8>(p, q) || fwd_row<T, 16>(p, q) || fwd_row<T, 32>(p, q) || fwd_row<T, 64>(p, q) || fwd_row<T, 256>(p, q) ||
                    fwd_row<T, 512>(p, q);
  if (!done) HI3D_FAIL(HI3D_ESHAPE, "layernorm_fwd: no kernel holds a row of this width");
  HI3D_LAUNCH_CHECK();
  return 0;
}
template <typename T>
int launch_bwd(const NormBwdParams& p, int nblk, hipStream_t st) {
  const Launch q = {pick((p.C + Elem<T>::VEC - 1) / Elem<T>::VEC, BWD_MOST), (unsigned)nblk, st, p.C < Elem<T>::VEC};
  const bool done = bwd_as<T, 8, 2, true>(p, q) || bwd_row<T, 8>(p, q) || bwd_row<T, 16>(p, q) || bwd_row<T, 32>(p, q) || bwd_row<T, 64>(p, q) || bwd_row<T, 256>(p, q) ||
                    bwd_row<T, 512>(p, q) || bwd_as<T, 512, 4, false>(p, q);
  if (!done) HI3D_FAIL(HI3D_ESHAPE, "layernorm_bwd: no kernel holds a row of this width");
  HI3D_LAUNCH_CHECK();
  return 0;
}

int bwd_blocks(long R, int C, int dtype) {
  const int vec = dtype == HI3D_F32 ? 4 : 8;
  const int lpr = pick((C + vec - 1) / vec, BWD_MOST).lpr;
  return (int)blocks_for(R, lpr, BWD_BLOCKS, bwd_rows(lpr));
}

int bad_sizes(long R, int C, int dtype, int wcode) {
  if (!hi3d_known_dtype(dtype) || !hi3d_known_dtype(wcode)) HI3D_FAIL(HI3D_EINVAL, "layernorm training: unknown element type");
  if (R < 0 || C <= 0) HI3D_FAIL(HI3D_EINVAL, "layernorm training: negative row count or width < 1");
  if (C > HI3D_NORM_MAX_WIDTH) HI3D_FAIL(HI3D_ESHAPE, "layernorm training: width over 8192");
  return 0;
}

}  // namespace

int hi3d_column_reduce(const float* part, void* o0, void* o1, int code0, int code1, int nblk, int C, int width, hipStream_t st) {
  hipLaunchKernelGGL(column_reduce_kernel, dim3((width + 15) / 16), dim3(1024), 0, st, part, o0, o1, code0, code1, nblk, C, width);
  HI3D_LAUNCH_CHECK();
  return 0;
}

extern "C" int hi3d_layernorm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* z, float* mean,
                                  float* rstd, int64_t R, int32_t C, int64_t ldx, int64_t ldr, int32_t dtype, int32_t wdtype, float eps, void* stream) {
  if (const int rc = bad_sizes(R, C, dtype, wdtype)) return rc;
  if (!(eps >= 0.0f) || eps > 3.0e38f) HI3D_FAIL(HI3D_EINVAL, "layernorm_fwd: eps must be finite and not negative");
  if (R == 0) return 0;
  if (!x || !y || !mean || !rstd || (residual && !z)) HI3D_FAIL(HI3D_EINVAL, "layernorm_fwd: null pointer");
  if ((ldx < C && R > 1) || (residual && ldr < C && R > 1)) HI3D_FAIL(HI3D_EINVAL, "layernorm_fwd: row pitch below the width");
  const NormFwdParams p = {x, residual, weight, bias, y, z, mean, rstd, (long)R, (long)ldx, (long)ldr, C, wdtype, eps};
  if (dtype == HI3D_F32) return launch_fwd<float>(p, (hipStream_t)stream);
  return dtype == HI3D_BF16 ? launch_fwd<bf16_t>(p, (hipStream_t)stream) : launch_fwd<half_t>(p, (hipStream_t)stream);
}

extern "C" int64_t hi3d_layernorm_bwd_workspace_floats(int64_t R, int32_t C, int32_t dtype) {
  if (R <= 0 || C <= 0 || C > HI3D_NORM_MAX_WIDTH || !hi3d_known_dtype(dtype)) return 0;
  const int n = bwd_blocks((long)R, C, dtype);
  return n > 1 ? (int64_t)n * 2 * C : 0;
}

extern "C" int hi3d_layernorm_bwd(const void* dy, const void* z, const void* dz, const void* weight, const float* mean, const float* rstd, void* dx,
                                  void* dweight, void* dbias, float* ws, int64_t R, int32_t C, int64_t lddy, int64_t ldz, int64_t lddz, int32_t dtype,
                                  int32_t wdtype, void* stream) {
  if (const int rc = bad_sizes(R, C, dtype, wdtype)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (R == 0) return (dweight || dbias) ? hi3d_column_reduce(nullptr, dweight, dbias, wdtype, wdtype, 0, C, 2 * C, st) : 0;   // sums of nothing
  if (!dy || !z || !mean || !rstd || !dx) HI3D_FAIL(HI3D_EINVAL, "layernorm_bwd: null pointer");
  if (R > 1 && (lddy < C || ldz < C || (dz && lddz < C))) HI3D_FAIL(HI3D_EINVAL, "layernorm_bwd: row pitch below the width");
  const int nblk = bwd_blocks((long)R, C, dtype), want = (dweight || dbias) ? 1 : 0;
  if (want && nblk > 1 && !ws) HI3D_FAIL(HI3D_EINVAL, "layernorm_bwd: workspace required (hi3d_layernorm_bwd_workspace_floats)");
  const NormBwdParams p = {dy, z, dz, weight, mean, rstd, dx, nblk > 1 ? ws : nullptr, dweight, dbias, (long)R, (long)lddy, (long)ldz, (long)lddz, C, wdtype, want};
  const int rc = dtype == HI3D_F32 ? launch_bwd<float>(p, nblk, st) : dtype == HI3D_BF16 ? launch_bwd<bf16_t>(p, nblk, st) : launch_bwd<half_t>(p, nblk, st);
  if (rc || !want || nblk == 1) return rc;
  return hi3d_column_reduce(ws, dweight, dbias, wdtype, wdtype, nblk, C, 2 * C, st);
}
