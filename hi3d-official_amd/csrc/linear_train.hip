// A linear layer with its epilogue, and its gradients:
//
//   z = x w^T + b        y = act(z) (+ residual)                       x [M, K]   w [N, K]   bf16 or fp16, products and sums fp32
//   dz = dy act'(z)      dx = dz w      dw = dz^T x      db = sum over rows of dz
//
// Beside hi3d_gemm_bf16, whose operands are laid out once for the sampler (K a multiple of 64, both operands contiguous along the
// contraction).  Here all three products read the tensors as a training step holds them: an operand is either contiguous along the
// contraction (KC: x and w forward, dz for dx) or across it (KS: w for dx, both for dw), and a KS tile reaches the matrix instruction
// through gfx950's transposing LDS read, so nothing is transposed in memory.
//
// Bound by the matrix instructions where the sizes allow: a step more of K runs at 1400 ... 1460 TFLOP/s with all CUs at work (4096 rows -> 5120 in 256 x 320
// tiles), and each round of tiles has about 10 us of start and end beside that.  Measured back to back, bf16: 16384 x 1280 -> 5120 forward 193 us (1114 TFLOP/s),
// dx 160 (1344), dw 205 (1050, its contraction split in 3, 16 us of it the join); 65536 x 2560 -> 640 192; 8192^3 832 / 836 / 847 (the library's products
// 708 / 832 / 947); 2048 x 1024 -> 1024 10.6 (405); 16 rows 1280 -> 1280 5.6 us, a launch.  GELU and a kept z add 14 us to a round.
#include "train_common.h"

namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bfx8;

constexpr int BK = 64;
// elements between rows that a tile's 32-bit offsets reach (320 rows of 2 bytes an element, 256 rows of 4): more is copied, or stored without them
constexpr long MOST_PITCH = 0x200000, MOST_WIDTH = 0x100000;

// ---- activations ------------------------------------------------------------------------------------------------------------------
// Phi(-a) = exp(-a^2 / 2) P(t), t = 1 / (1 + 0.3 a), a >= 0: P of degree 8 without constant term, fitted to the Mills ratio over
// [0, 14] with least relative error, 1.5e-7 -- relative also where Phi is tiny, which an erf with an absolute error would not give, and small enough
// for the fp32 sums of the bias' gradient.  In fp32 the roundings of the exponent's argument come on top, a^2 2^-24, and a few of 2^-24: 7.5e-7 up to a = 3,
// 1.6e-6 up to 5, 8e-6 at 13, where Phi leaves fp32's normal numbers.
__device__ __forceinline__ void gauss(float x, float& cdf, float& bell) {
  const float a = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.3f * a);
  bell = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);          // exp(-x^2 / 2)
  float q = 0.03567480055634768f;
  q = q * t - 0.15720318772763442f;
  q = q * t + 0.20635367719077033f;
  q = q * t - 0.053683791141534425f;
  q = q * t + 0.12856169845786158f;
  q = q * t + 0.09991347218457869f;
  q = q * t + 0.12075395892859297f;
  q = q * t + 0.11962929865929173f;
  q = q * t * bell;
  cdf = x < 0.0f ? q : 1.0f - q;
}
// x Phi(x) = max(x, 0) - |x| Phi(-|x|), for results of 16 bits: the same with P of degree 6, fitted to 4.7e-6; in fp32 5.4e-6 up to |x| = 5 (fp16's half
// step, 2^-12 ... 2^-11 of a value, is at least 45 times that; its normal numbers end there) and 1.0e-5 at 13.  The epilogue of a
// 256-row tile is bound by these instructions.  |x| is bounded where it multiplies, so that infinity stays (NaN comes through Phi).
__device__ __forceinline__ float gelu(float x) {
  const float a = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.31f * a);
  float q = -0.07392971407271384f;
  q = q * t + 0.1804520365085403f;
  q = q * t + 0.01574284864956139f;
  q = q * t + 0.13343072169148096f;
  q = q * t + 0.1204410684003111f;
  q = q * t + 0.1238607172392901f;
  q = q * t * __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);
  return fmaxf(x, 0.0f) - fminf(a, 64.0f) * q;
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f)); }

template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  if (act == HI3D_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gelu(v[j]);
  } else if (act == HI3D_ACT_SILU || act == HI3D_ACT_QUICK_GELU) {
    const float s = act == HI3D_ACT_SILU ? 1.0f : 1.702f;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= sigmoid(s * v[j]);
  } else if (act == HI3D_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];        // (keeps NaN)
  }
}
// v[j] *= act'(z[j])
template <int N>
__device__ __forceinline__ void times_slope(int act, const float (&z)[N], float (&v)[N]) {
  if (act == HI3D_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) { float c, b; gauss(z[j], c, b); v[j] *= c + z[j] * b * 0.3989422804014327f; }
  } else if (act == HI3D_ACT_SILU || act == HI3D_ACT_QUICK_GELU) {
    const float s = act == HI3D_ACT_SILU ? 1.0f : 1.702f;
#pragma unroll
    for (int j = 0; j < N; ++j) { const float g = sigmoid(s * z[j]); v[j] *= g * (1.0f + s * z[j] * (1.0f - g)); }
  } else if (act == HI3D_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = z[j] <= 0.0f ? 0.0f : v[j];
  }
}

// ---- the epilogue of 8 consecutive columns of a row (the first `n` of them exist) ---------------------------------------------------
struct Epilogue {
  const void* bias; const void* res; void* y; void* z;
  long ldr, ldo;
  int bcode, act;
};
template <typename T>
__device__ __forceinline__ void finish(const Epilogue& e, long m, int c, int n, float (&v)[8]) {
  if (e.bias) {
    float b[8];
    load_vec_as(e.bias, e.bcode, c, n, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
  }
  if (e.z) store_some((T*)e.z + m * e.ldo + c, n, v);
  activate(e.act, v);
  if (e.res) {
    Pack<T, 8> k;
    float r[8];
    fetch((const T*)e.res + m * e.ldr + c, n, c, k);
    unpack(k, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store_some((T*)e.y + m * e.ldo + c, n, v);
}

// ---- the product ------------------------------------------------------------------------------------------------------------------
// out[M, N] = A B over the contraction of length K.  A is [M][K] (KC) or [K][M] (KS), B is [N][K] (KC) or [K][N] (KS); rows at a pitch
// that is a multiple of 8 elements, 16-byte aligned; a row of KC holds zeros from K up to the next multiple of 8.
struct MatParams {
  const char* A; const char* B;
  float* part;            // split contraction: partial sums [split][M][N rounded up to 8]; NULL: the epilogue below
  Epilogue e;
  long lda, ldb;
  int M, N, K, nbm, nbn, splits, per;      // per: K steps of a split
  int group;                               // m-tiles that are walked before n moves on
};

template <typename T> struct Mfma;
template <> struct Mfma<bf16_t> {
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mfma<half_t> {
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

__device__ __forceinline__ int swap23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// One operand's tile of R rows (columns of the output) x 64 of the contraction, 128 bytes x R of LDS, filled by LDS-DMA in pieces of 1 KiB
// (8 LDS rows of 128 bytes; a piece's lanes land in order, so what an LDS slot holds is chosen by the address that its lane reads).
//
// KC: LDS row r is operand row r, its 16-byte chunk c stands in slot c ^ ((r >> 1) & 7): a fragment read (16 rows, one chunk each) takes every
//     bank once.
// KS: panels of 64 columns; LDS row p of a panel is contraction row swap23(p) (bits 2 and 3 exchanged), its 32-byte unit u (16 columns)
//     stands at u ^ ((p >> 1) & 3).  A transposing read takes [4 k][16 columns] per 16 lanes; with lane group g at k = 8 g + 4 h, the 8 LDS
//     rows that half a wave touches are consecutive and their units fall on 8 different eighths of the banks.
template <bool KS, int R, int NW>
struct Tile {
  static constexpr int PIECES = R / 8 / NW;
  static_assert(R % 64 == 0 && (R / 8) % NW == 0, "whole panels, whole pieces");
  unsigned off[PIECES];
  int chunk[PIECES];                      // KC: the lane's 8-element chunk of the K step
  const char* base;
  long ld;                                // bytes
  int rows, cols, first;                  // KC: rows of the tile that exist, K rounded up to 8;  KS: K, the output's columns rounded up to 8; its first column

  __device__ __forceinline__ void init(const char* p, long ld_el, int r0, int total, int K, int wave, int lane) {
    ld = ld_el * 2;
    if (!KS) { base = p + (long)r0 * ld; rows = min(R, total - r0); cols = (K + 7) & ~7; first = 0; }
    else { base = p + (long)r0 * 2; rows = K; cols = (total + 7) & ~7; first = r0; }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int q = wave * PIECES + i;
      if (!KS) {
        const int r = q * 8 + (lane >> 3);
        chunk[i] = (lane & 7) ^ ((r >> 1) & 7);
        off[i] = (unsigned)(r * (int)ld + chunk[i] * 16);
      } else {
        const int pos = (q & 7) * 8 + (lane >> 3), u = ((lane & 7) >> 1) ^ ((pos >> 1) & 3);
        chunk[i] = 0;
        off[i] = (unsigned)(swap23(pos) * (int)ld + ((q >> 3) * 64 + u * 16 + (lane & 1) * 8) * 2);
      }
    }
  }
  // K step `kt` of the contraction into the tile at `lds`; what lies outside the operand is zero (beyond the descriptor's range)
  __device__ __forceinline__ void issue(int kt, char* lds, int wave) const {
    const int k0 = kt * BK;
    const char* b = base + (KS ? (long)k0 * ld : (long)k0 * 2);
    const long valid = KS ? (long)(min(rows - k0, BK) - 1) * ld + (long)(cols - first) * 2 : (long)(rows - 1) * ld + (long)(cols - k0) * 2;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, (int)(valid > 0x7ffffff0 ? 0x7ffffff0 : valid), 0x00020000);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      unsigned o = off[i];
      if (!KS && k0 + chunk[i] * 8 >= cols) o = 0x80000000u;       // behind the end of a row: not the next row's data
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_AS void*)(lds + (wave * PIECES + i) * 1024), 16, o, 0, 0, 0);
    }
  }
};

// The fragments of a wave's 16 * CNT rows (from row `first`) of a tile, half KH of its contraction
template <bool KS, int CNT>
struct Frags {
  int addr[KS ? CNT : 1];
  int sw;
  __device__ __forceinline__ void init(int first, int lane) {
    const int fr = lane & 15, fg = lane >> 4;
    if (!KS) { addr[0] = (first + fr) * 128; sw = (fr >> 1) & 7; }
    else {
      const int x = ((fg & 1) << 1) | (fr >> 3);
#pragma unroll
      for (int t = 0; t < CNT; ++t) {
        const int u = first / 16 + t;
        addr[t] = (u >> 2) * 8192 + (fg >> 1) * 2048 + (fg & 1) * 512 + (fr >> 2) * 128 + (((u & 3) ^ x) << 5) + (fr & 3) * 8;
      }
      sw = 0;
    }
  }
  // The transposing reads are in inline assembly, wait included: as builtins they would be kept behind every LDS-DMA in flight.
  template <int KH>
  __device__ __forceinline__ void read(const char* lds, u32x4 (&f)[CNT], int lane) const {
    if constexpr (!KS) {
      const char* p = lds + addr[0] + (((KH * 4 + (lane >> 4)) ^ sw) << 4);
#pragma unroll
      for (int t = 0; t < CNT; ++t) f[t] = *(const u32x4*)(p + t * 2048);
    } else {
      const unsigned b = (unsigned)(__UINTPTR_TYPE__)(LDS_AS const char*)lds;
#pragma unroll
      for (int t = 0; t < CNT; t += (CNT == 5 ? 5 : CNT == 2 ? 2 : 4)) {
        if constexpr (CNT == 2) {
          u32x2 l0, l1, h0, h1;
          asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %2, %4 offset:%7\n\t"
                       "ds_read_b64_tr_b16 %1, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                       "s_waitcnt lgkmcnt(0)"
                       : "=&v"(l0), "=&v"(l1), "=&v"(h0), "=&v"(h1)
                       : "v"(b + addr[0]), "v"(b + addr[1]), "n"(KH * 4096), "n"(KH * 4096 + 1024)
                       : "memory");
          f[0] = u32x4{l0[0], l0[1], h0[0], h0[1]};
          f[1] = u32x4{l1[0], l1[1], h1[0], h1[1]};
        } else if constexpr (CNT == 5) {
          u32x2 l0, l1, l2, l3, l4, h0, h1, h2, h3, h4;
          asm volatile("ds_read_b64_tr_b16 %0, %10 offset:%15\n\tds_read_b64_tr_b16 %5, %10 offset:%16\n\t"
                       "ds_read_b64_tr_b16 %1, %11 offset:%15\n\tds_read_b64_tr_b16 %6, %11 offset:%16\n\t"
                       "ds_read_b64_tr_b16 %2, %12 offset:%15\n\tds_read_b64_tr_b16 %7, %12 offset:%16\n\t"
                       "ds_read_b64_tr_b16 %3, %13 offset:%15\n\tds_read_b64_tr_b16 %8, %13 offset:%16\n\t"
                       "ds_read_b64_tr_b16 %4, %14 offset:%15\n\tds_read_b64_tr_b16 %9, %14 offset:%16\n\t"
                       "s_waitcnt lgkmcnt(0)"
                       : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "=&v"(l4), "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3), "=&v"(h4)
                       : "v"(b + addr[0]), "v"(b + addr[1]), "v"(b + addr[2]), "v"(b + addr[3]), "v"(b + addr[CNT - 1]), "n"(KH * 4096), "n"(KH * 4096 + 1024)
                       : "memory");
          f[0] = u32x4{l0[0], l0[1], h0[0], h0[1]};
          f[1] = u32x4{l1[0], l1[1], h1[0], h1[1]};
          f[2] = u32x4{l2[0], l2[1], h2[0], h2[1]};
          f[3] = u32x4{l3[0], l3[1], h3[0], h3[1]};
          f[CNT - 1] = u32x4{l4[0], l4[1], h4[0], h4[1]};
        } else {
          u32x2 l0, l1, l2, l3, h0, h1, h2, h3;
          asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
                       "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
                       "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
                       "ds_read_b64_tr_b16 %3, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                       "s_waitcnt lgkmcnt(0)"
                       : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3)
                       : "v"(b + addr[t]), "v"(b + addr[t + 1]), "v"(b + addr[t + 2]), "v"(b + addr[t + 3]), "n"(KH * 4096), "n"(KH * 4096 + 1024)
                       : "memory");
          f[t] = u32x4{l0[0], l0[1], h0[0], h0[1]};
          f[t + 1] = u32x4{l1[0], l1[1], h1[0], h1[1]};
          f[t + 2] = u32x4{l2[0], l2[1], h2[0], h2[1]};
          f[t + 3] = u32x4{l3[0], l3[1], h3[0], h3[1]};
        }
      }
    }
  }
};

// WM x WN waves, each 16 MT x 16 NT of the output; two tiles of the contraction in LDS, the next one on its way while one is used.
// The weight-side fragment is the first operand of the matrix instruction, so that a lane holds 4 consecutive columns of one output row.
template <typename T, bool AKS, bool BKS, int WM, int WN, int MT, int NT>
__device__ __forceinline__ void mat_tile(const MatParams& p, int bid, char* smem) {
#if __HIP_DEVICE_COMPILE__
  constexpr int NW = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / WN, wn = w % WN;

  // block -> tile: neighbours in the order go to one XCD (its L2 keeps what they share); `group` m-tiles are walked for each n-tile
  const int nblk = p.nbm * p.nbn;
  const int ks = bid / nblk;
  bid -= ks * nblk;
  const int q = nblk >> 3, r = nblk & 7, xcd = bid & 7, idx = bid >> 3;
  const int lid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int per = p.group * p.nbn, g = lid / per, rem = lid - g * per;
  const int gh = min(p.group, p.nbm - g * p.group);
  const int tn = rem / gh, tm = g * p.group + rem - tn * gh;
  const int m0 = tm * BM, n0 = tn * BN;

  Tile<AKS, BM, NW> ta;
  Tile<BKS, BN, NW> tb;
  ta.init(p.A, p.lda, m0, p.M, p.K, w, lane);
  tb.init(p.B, p.ldb, n0, p.N, p.K, w, lane);
  Frags<AKS, MT> fa;
  Frags<BKS, NT> fb;
  fa.init(wm * 16 * MT, lane);
  fb.init(wn * 16 * NT, lane);

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int steps = (p.K + BK - 1) / BK, kb = ks * p.per, ke = min(steps, kb + p.per);
  u32x4 a[MT], b[NT];
  auto issue = [&](int kt) {
    char* const d = smem + ((kt - kb) & 1) * STAGE;
    ta.issue(kt, d, w);
    tb.issue(kt, d + ABYTES, w);
  };
  auto read = [&](const char* s, auto kh) {
    fa.template read<decltype(kh)::value>(s, a, lane);
    fb.template read<decltype(kh)::value>(s + ABYTES, b, lane);
  };
  auto multiply = [&]() {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = Mfma<T>::mul(b[j], a[i], acc[i][j]);
  };
  issue(kb);
  if (threadIdx.x < BN / 8) {                       // the bias of the tile's columns (zeros where there is none) behind the tiles
    float f[8] = {};
    const int c = threadIdx.x * 8;
    if (!p.part && p.e.bias) load_vec_as(p.e.bias, p.e.bcode, n0 + c, p.N - n0 - c, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) ((float*)(smem + 2 * STAGE))[c + j] = f[j];
  }
  if constexpr (NW == 8) {
    // Two waves a SIMD, half a phase apart: a phase is [LDS-DMA of the next tile, fragment reads] barrier [matrix instructions] barrier, and
    // waves 4 ... 7 are one barrier behind, so that of the two waves on a SIMD one reads while the other multiplies.  The next tile goes
    // over the one that step kt - 1 read: its last fragment reads had returned (lgkmcnt(0)) before the barrier that ended their segment,
    // and the first wave to issue is one barrier further.  It is waited for in the step's last read segment; the trailing waves do so one
    // barrier before the leading ones read it.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (w >= 4) __builtin_amdgcn_s_barrier();
    auto phase = [&](const char* s, auto kh) {
      constexpr bool LAST = decltype(kh)::value == 1;
      read(s, kh);
      if (LAST) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      multiply();
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int kt = kb; kt < ke; ++kt) {
      const char* const s = smem + ((kt - kb) & 1) * STAGE;
      if (kt + 1 < ke) issue(kt + 1);
      phase(s, std::integral_constant<int, 0>{});
      phase(s, std::integral_constant<int, 1>{});
    }
    if (w < 4) __builtin_amdgcn_s_barrier();
  } else {
    for (int kt = kb; kt < ke; ++kt) {
      const char* const s = smem + ((kt - kb) & 1) * STAGE;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();                              // tile kt is there, and everyone is done with the other one
      if (kt + 1 < ke) issue(kt + 1);
      read(s, std::integral_constant<int, 0>{});
      multiply();
      read(s, std::integral_constant<int, 1>{});
      multiply();
    }
  }
  __syncthreads();                                // the tiles' LDS is free

  // Bias and activation are taken where the accumulators are; the results leave in whole rows of the tile (a wave's own columns are 160 bytes of a
  // row, and lines that several waves write a part of at different times cost a 65536 x 2560 output 60 us of 353), 16 rows of every wave row at a
  // time through LDS: rounded values, or fp32 where a residual or other partial sums are still to be added.  Two buffers in turn, so that one
  // barrier per pass is enough -- a buffer is written again two passes on, behind a barrier that its readers have passed.  Stores and residual
  // loads go through buffer descriptors: what lies outside is dropped there, without a branch for the compiler to wait at.
  //   rounded: pitch 2 BN + 16 bytes, 8 bytes a lane and column block: 32 lanes fall on all 64 banks.
  //   fp32: pitch 4 BN + 16 bytes, the 16-byte units of a row even ones first: a thread's two units are read by two accesses whose lanes lie
  //   side by side (side by side in the row, each access had half the banks).
  constexpr int SROWS = 16 * WM, CPR = BN / 8, TH = NW * 64, CH = (SROWS * CPR + TH - 1) / TH;
  constexpr int FROW = BN * 4 + 16, HROW = BN * 2 + 16, FSLAB = SROWS * FROW, HSLAB = SROWS * HROW;
  static_assert(2 * (FSLAB + HSLAB) <= 2 * STAGE, "two buffers of both kinds fit the tiles' LDS");
  constexpr unsigned NONE = 0x80000000u;
  const int fr = lane & 15, fg = lane >> 4;
  const int width = p.part ? (p.N + 7) & ~7 : p.N, cols = width - n0;           // columns of the tile that exist (partial sums: in whole chunks)
  const bool fits = p.N % 8 == 0 && (((unsigned long)p.e.y | (unsigned long)p.e.z) & 15) == 0 &&
                    (!p.e.res || (p.e.ldr % 8 == 0 && p.e.ldr <= MOST_PITCH && ((unsigned long)p.e.res & 15) == 0));      // 16-byte accesses do
  const bool wide = p.part || p.e.res || !fits;     // fp32 through LDS
  const int wrow = wm * 16 + fr, wcol = wn * 16 * NT + fg * 4;
  f32x4 bias[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) bias[j] = *(const f32x4*)(smem + 2 * STAGE + (wcol + j * 16) * 4);
  const int esz = p.part ? 4 : 2;
  const long ldo = p.part ? width : p.e.ldo;
  unsigned off[CH], roff[CH];                       // of the thread's chunks of 8 columns: bytes in the output and the residual, the LDS places
  int hat[CH], fat[CH];
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    const int c = t * TH + threadIdx.x, r = c / CPR, q = c - r * CPR, row = (r >> 4) * 16 * MT + (r & 15);
    const bool in = c < SROWS * CPR && q * 8 < cols;
    hat[t] = in ? r * HROW + q * 16 : 0;
    fat[t] = in ? r * FROW + q * 16 : 0;
    off[t] = in ? ((unsigned)row * (unsigned)ldo + q * 8) * esz : NONE;
    roff[t] = in ? ((unsigned)row * (unsigned)p.e.ldr + q * 8) * 2 : NONE;
  }
  auto window = [&](const void* base, long ld, int size, int i) {        // rows m0 + 16 i ... of a matrix of M rows, from column n0
    const long rows = p.M - m0 - 16 * i, valid = rows > 0 ? ((rows - 1) * ld + cols) * size : 0;
    return __builtin_amdgcn_make_buffer_rsrc((char*)base + ((m0 + 16L * i) * ld + n0) * size, 0, (int)(valid > 0x7ffffff0 ? 0x7ffffff0 : valid), 0x00020000);
  };
  auto meet = [&]() {                               // this pass's rows are in LDS for everyone; outstanding stores are not waited for
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto to_fp32 = [&](char* slab, int j, const f32x4& v) {
    const int u = (wcol + j * 16) >> 2;
    *(f32x4*)(slab + wrow * FROW + ((u >> 1) + (u & 1) * CPR) * 16) = v;
  };
  auto to_rounded = [&](char* slab, int j, const f32x4& v) {
    const float f[4] = {v[0], v[1], v[2], v[3]};
    const Pack<T, 4> k = pack<T, 4>(f);
    *(u32x2*)(slab + wrow * HROW + (wcol + j * 16) * 2) = u32x2{k.w[0], k.w[1]};
  };
  u32x4 res[CH];
  auto residual = [&](int i) {
    const __amdgpu_buffer_rsrc_t from = window(p.e.res, p.e.ldr, 2, i);
#pragma unroll
    for (int t = 0; t < CH; ++t) res[t] = __builtin_amdgcn_raw_buffer_load_b128(from, roff[t], 0, 0);
  };
  // WIDE: fp32 slabs;  ACT: the activation, or -1 where `finish` takes it (chunks that 16-byte accesses do not fit) or there is nothing to take
  auto passes = [&](auto act_, auto wide_) {
    constexpr int ACT = decltype(act_)::value;
    constexpr bool WIDE = decltype(wide_)::value;
    if (WIDE && ACT >= 0) residual(0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      char* const fslab = smem + (i & 1) * FSLAB;
      char* const hslab = smem + 2 * FSLAB + (i & 1) * HSLAB;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f32x4 v = acc[i][j];
        if constexpr (ACT >= 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] += bias[j][k];
          if (p.e.z) to_rounded(WIDE ? hslab : fslab, j, v);
          float f[4] = {v[0], v[1], v[2], v[3]};
          activate(ACT, f);
          v = f32x4{f[0], f[1], f[2], f[3]};
        }
        if (WIDE) to_fp32(fslab, j, v);
        else to_rounded(hslab, j, v);
      }
      meet();
      if constexpr (ACT < 0) {
        if (p.part) {
          const __amdgpu_buffer_rsrc_t to = window(p.part + (long)ks * p.M * width, ldo, 4, i);
#pragma unroll
          for (int t = 0; t < CH; ++t) {
            __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4*)(fslab + fat[t]), to, off[t], 0, 0);
            __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4*)(fslab + fat[t] + CPR * 16), to, off[t] + 16, 0, 0);
          }
        } else {
#pragma unroll 1
          for (int c = threadIdx.x; c < SROWS * CPR; c += TH) {
            const int r = c / CPR, q = c - r * CPR, n = n0 + q * 8;
            const long m = m0 + (r >> 4) * 16 * MT + (r & 15) + i * 16;
            if (m >= p.M || q * 8 >= cols) continue;
            const f32x4 lo = *(const f32x4*)(fslab + r * FROW + q * 16), hi = *(const f32x4*)(fslab + r * FROW + q * 16 + CPR * 16);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            finish<T>(p.e, m, n, p.N - n, v);
          }
        }
      } else {
        if (p.e.z) {
          const __amdgpu_buffer_rsrc_t to = window(p.e.z, ldo, 2, i);
#pragma unroll
          for (int t = 0; t < CH; ++t) __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4*)((WIDE ? hslab : fslab) + hat[t]), to, off[t], 0, 0);
        }
        const __amdgpu_buffer_rsrc_t to = window(p.e.y, ldo, 2, i);
        u32x4 y[CH];
#pragma unroll
        for (int t = 0; t < CH; ++t) {
          if constexpr (WIDE) {
            const f32x4 lo = *(const f32x4*)(fslab + fat[t]), hi = *(const f32x4*)(fslab + fat[t] + CPR * 16);
            const Pack<T, 8> k = {{res[t][0], res[t][1], res[t][2], res[t][3]}};
            float r[8];
            unpack(k, r);
            const float v[8] = {r[0] + lo[0], r[1] + lo[1], r[2] + lo[2], r[3] + lo[3], r[4] + hi[0], r[5] + hi[1], r[6] + hi[2], r[7] + hi[3]};
            const Pack<T, 8> o = pack<T, 8>(v);
            y[t] = u32x4{o.w[0], o.w[1], o.w[2], o.w[3]};
          } else y[t] = *(const u32x4*)(hslab + hat[t]);
        }
        if (WIDE && i + 1 < MT) residual(i + 1);
#pragma unroll
        for (int t = 0; t < CH; ++t) __builtin_amdgcn_raw_buffer_store_b128(y[t], to, off[t], 0, 0);
      }
    }
  };
  auto with = [&](auto act) {
    if (wide) passes(act, std::true_type{});
    else passes(act, std::false_type{});
  };
  using std::integral_constant;
  if (p.part || !fits) passes(integral_constant<int, -1>{}, std::true_type{});
  else if constexpr (AKS || BKS) passes(integral_constant<int, HI3D_ACT_NONE>{}, std::false_type{});       // a gradient: no epilogue
  else switch (p.e.act) {
    case HI3D_ACT_NONE: with(integral_constant<int, HI3D_ACT_NONE>{}); break;
    case HI3D_ACT_GELU: with(integral_constant<int, HI3D_ACT_GELU>{}); break;
    case HI3D_ACT_RELU: with(integral_constant<int, HI3D_ACT_RELU>{}); break;
    case HI3D_ACT_SILU: with(integral_constant<int, HI3D_ACT_SILU>{}); break;
    default: with(integral_constant<int, HI3D_ACT_QUICK_GELU>{}); break;
  }
#endif
}

template <typename T, bool AKS, bool BKS, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(WM * WN * 64, MT == 2 ? 4 : 2) void mat_kernel(const MatParams p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  mat_tile<T, AKS, BKS, WM, WN, MT, NT>(p, blockIdx.x, smem);
}
// dw and dx of a layer in one launch, where neither fills the chip by itself (3083 x 650 -> 1290: 65 us one after the other, 46 with this and the
// prepared operands in one launch too): the first `first` blocks are dw's (the longer ones)
template <typename T, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(WM * WN * 64, MT == 2 ? 4 : 2) void both_gradients_kernel(const MatParams dw, const MatParams dx, int first) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  if ((int)blockIdx.x < first) mat_tile<T, true, true, WM, WN, MT, NT>(dw, blockIdx.x, smem);
  else mat_tile<T, false, true, WM, WN, MT, NT>(dx, blockIdx.x - first, smem);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------
// y for at most 16 MT rows of x: the weights are all there is to read, once.  A block takes 16 / CS columns of the output and its 16 waves a
// 16th of the contraction each, straight from memory into matrix operands -- no LDS, no padded copies: any pitch and alignment -- with U
// steps of 32 in flight; the waves' sums meet in LDS in the order of the waves.
// CS > 1 (at most 16 / CS rows of x): the 16 rows of the matrix operand are 16 / CS columns of the output times CS pieces of the contraction,
// those of the other operand rows of x times the same pieces, and of the product the entries of equal pieces are used: a long
// contraction makes CS times the blocks (N = 1280, K = 5120, one row: 80 blocks 8.4 us, 160 blocks 6.3 us).
// Rows behind M and columns behind N repeat the last one and are not stored.
constexpr int FEW_WAVES = 16;
struct FewParams { const void* x; const void* w; Epilogue e; long ldx, ldw; int M, N, K; };

template <typename T, int MT, int CS>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_rows_kernel(const FewParams p) {
#if __HIP_DEVICE_COMPILE__
  constexpr int U = MT == 1 ? 8 : 4, COLS = 16 / CS, ROWS = 16 * MT / CS;
  static_assert(MT == 1 || CS == 1, "pieces only where 16 rows are too many");
  __shared__ __attribute__((aligned(16))) float sums[FEW_WAVES][16 * MT][16];
  __shared__ float whole[ROWS][COLS];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fg = lane >> 4;
  const int n0 = blockIdx.x * COLS;
  const int per = ((p.K + 31) / 32 + FEW_WAVES * CS - 1) / (FEW_WAVES * CS);          // steps of 32 of a piece
  const int k0 = (w * CS + fr % CS) * per * 32 + fg * 8, last = (w * CS + CS - 1) * per * 32;       // this lane's; the wave's last piece's
  const T* const wr = (const T*)p.w + (long)min(n0 + fr / CS, p.N - 1) * p.ldw;
  const T* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = (const T*)p.x + (long)min((i * 16 + fr) / CS, p.M - 1) * p.ldx;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < per; s += U) {
    Pack<T, 8> kw[U], kx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + (s + u) * 32;
      if (s + u >= per) continue;
      if (last + (s + u + 1) * 32 <= p.K) {
        kw[u] = *(const Pack<T, 8>*)(wr + k);
#pragma unroll
        for (int i = 0; i < MT; ++i) kx[u][i] = *(const Pack<T, 8>*)(xr[i] + k);
      } else {                                     // the contraction's end in some lanes
        fetch(wr + k, p.K - k, k, kw[u]);
#pragma unroll
        for (int i = 0; i < MT; ++i) fetch(xr[i] + k, p.K - k, k, kx[u][i]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= per) continue;
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = Mfma<T>::mul(u32x4{kw[u].w[0], kw[u].w[1], kw[u].w[2], kw[u].w[3]}, u32x4{kx[u][i].w[0], kx[u][i].w[1], kx[u][i].w[2], kx[u][i].w[3]}, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) *(f32x4*)&sums[w][i * 16 + fr][fg * 4] = acc[i];
  __syncthreads();
  for (int q = threadIdx.x; q < ROWS * COLS; q += FEW_WAVES * 64) {
    const int m = q / COLS, n = q % COLS;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < FEW_WAVES; ++k)
#pragma unroll
      for (int c = 0; c < CS; ++c) t += sums[k][m * CS + c][n * CS + c];
    whole[m][n] = t;
  }
  __syncthreads();
  constexpr int CHUNKS = (COLS + 7) / 8;
  const int m = threadIdx.x / CHUNKS, c = (threadIdx.x % CHUNKS) * 8, n = min(COLS, p.N - n0) - c;
  if (m < p.M && m < ROWS && n > 0) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < COLS ? whole[m][c + j] : 0.0f;
    finish<T>(p.e, m, n0 + c, n, v);
  }
#endif
}

// The partial sums of a split contraction and the epilogue.  G threads take every G-th split of a chunk of 8 columns each, and their sums are added in
// their order: many splits of a small output would otherwise be as many trips to memory, one after the other (31 splits of 3 x 480: 6.5 us).
template <typename T, int G>
__global__ __launch_bounds__(256) void join_kernel(const float* part, Epilogue e, long M, int N, int splits) {
  constexpr int CHUNKS = 256 / G;
  __shared__ float sums[G > 1 ? G : 1][G > 1 ? CHUNKS : 1][9];
  const int cpr = (N + 7) / 8, g = threadIdx.x / CHUNKS, t = threadIdx.x % CHUNKS;
  for (long c0 = (long)blockIdx.x * CHUNKS; c0 < M * cpr; c0 += (long)gridDim.x * CHUNKS) {
    const long c = c0 + t, m = c / cpr;
    const int n = (int)(c - m * cpr) * 8;
    float v[8] = {};
    if (m < M) {
#pragma unroll 4
      for (int s = g; s < splits; s += G) {
        const Pack<float, 8> k = *(const Pack<float, 8>*)(part + (s * M + m) * (cpr * 8L) + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += __uint_as_float(k.w[j]);
      }
    }
    if constexpr (G > 1) {
      __syncthreads();                              // (the last chunk's sums have been read)
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[g][t][j] = v[j];
      __syncthreads();
      if (g) continue;
#pragma unroll
      for (int k = 1; k < G; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += sums[k][t][j];
    }
    if (m < M) finish<T>(e, m, n, N - n, v);
  }
}

// What the products need first, in one launch:
//   dz = dy act'(z), in rows padded with zeros to a multiple of 8 elements, rounded to the operands' type: the matrix instruction takes 16 bits, as every 16-bit
//   backward pass does.  This is the one rounding besides that of the stored results: dx and dw are off by 0.0023 of their norm in bf16 and 0.00029 in fp16
//   where unrounded they would be by 0.0017 and 0.00021 (16384 x 1280 -> 5120, 3083 x 650 -> 1290).  dz as a sum of two 16-bit parts would keep the digits
//   for twice the products (16384 x 1280 -> 5120: about 360 us on top of 467);
//   the column sums of the unrounded dz, one row of partial sums per block row (256 columns x 8 row lanes a block; up to SLOPE_FEW rows
//   64 columns x 32 row lanes, and the sums themselves: one launch less);
//   up to two operands whose rows cannot be read in place, padded likewise.
struct SlopeParams {
  const void* dy; const void* z; void* dz; float* part;
  long M, lddy, ldz;
  void* db;                                // instead of partial sums, where one block has all rows
  int N, act, rows, db_code;               // rows: of a block
};
constexpr int SLOPE_FEW = 128;
struct PadParams { const void* in; void* out; long rows, ld; int cols, blocks; };

template <typename T, int TX>
__device__ __forceinline__ void slope(const SlopeParams& p, int bx, int by, float* lds) {
  constexpr int COLS = TX * 8, TY = 256 / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, c = bx * COLS + tx * 8, n = p.N - c;
  const long r0 = (long)by * p.rows, r1 = min(p.M, r0 + p.rows);
  const long ldo = (p.N + 7) / 8 * 8;
  float s[8] = {};
  if (n > 0)
    for (long r = r0 + ty; r < r1; r += TY) {
      Pack<T, 8> ky, kz;
      float v[8], z[8];
      fetch((const T*)p.dy + r * p.lddy + c, n, c, ky);
      if (p.act) fetch((const T*)p.z + r * p.ldz + c, n, c, kz);
      unpack(ky, v);
      if (p.act) {
        unpack(kz, z);
        times_slope(p.act, z, v);
        if (n < 8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = j < n ? v[j] : 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
      if (p.dz) store_some((T*)p.dz + r * ldo + c, 8, v);
    }
  if (!p.part && !p.db) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) lds[ty * COLS + tx * 8 + j] = s[j];
  __syncthreads();
  const int col = bx * COLS + threadIdx.x;
  if (threadIdx.x < COLS && col < p.N) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < TY; ++k) t += lds[k * COLS + threadIdx.x];
    if (p.db) store_as(p.db, p.db_code, col, t);
    else p.part[(long)by * p.N + col] = t;
  }
}
template <typename T>
__device__ __forceinline__ void pad_rows(const PadParams& p, int block) {
  const int cpr = (p.cols + 7) / 8;
  for (long c = (long)block * 256 + threadIdx.x; c < p.rows * cpr; c += (long)p.blocks * 256) {
    const long r = (c >> 32) ? c / cpr : (long)((unsigned)c / (unsigned)cpr);
    const int e = (int)(c - r * cpr) * 8;
    Pack<T, 8> k;
    fetch((const T*)p.in + r * p.ld + e, p.cols - e, e, k);
    *(Pack<T, 8>*)((T*)p.out + r * (long)cpr * 8 + e) = k;
  }
}
template <typename T>
__global__ __launch_bounds__(256) void prepare_kernel(const SlopeParams s, int across, int slope_blocks, const PadParams a, const PadParams b) {
  __shared__ float lds[2048];
  const int bid = blockIdx.x;
  if (bid < slope_blocks) {
    if (s.M <= SLOPE_FEW) slope<T, 8>(s, bid, 0, lds);
    else slope<T, 32>(s, bid % across, bid / across, lds);
  }
  else if (bid < slope_blocks + a.blocks) pad_rows<T>(a, bid - slope_blocks);
  else pad_rows<T>(b, bid - slope_blocks - a.blocks);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
// Tiles, and what one costs in us: a K step with one block on each CU and with `per_cu`, and a tile's start and end.  Fitted to sweeps of every tile and
// split over M 65 ... 65536, N and K 320 ... 5120, all three products: of 147 products the estimate's pick is within 10 % of the best plan in 125, within 20 %
// in 145, 25 % over it at worst.  64 x 64: small products whose blocks wait for memory and LDS rather than compute (2048 x 1024 x 1024: 14.8 -> 10.4 us).
struct Config { int bm, bn, per_cu; double one, full, fixed; };
constexpr Config CONFIGS[] = {{256, 256, 1, 1.45, 1.45, 10.0}, {256, 320, 1, 1.85, 1.85, 9.0}, {128, 128, 2, 0.85, 1.0, 4.0}, {64, 64, 4, 0.4, 0.65, 3.0}};
constexpr int CUS = 256, MAX_SPLITS = 32;

struct Plan { int cfg, splits, per; double us; };
// the tile and the split of the contraction that the estimate finds fastest: whole rounds of the chip, the rest at the occupancy that it
// leaves, and the joining pass of a split
Plan plan_of(long M, long N, long K) {
  Plan best = {3, 1, 0, 1e300};
  const long steps = (K + BK - 1) / BK;
  for (int c = 0; c < 4; ++c) {
    const Config& f = CONFIGS[c];
    const long tiles = ((M + f.bm - 1) / f.bm) * ((N + f.bn - 1) / f.bn), slots = (long)f.per_cu * CUS;
    for (long s = 1; s <= MAX_SPLITS && s <= steps; ++s) {
      const long per = (steps + s - 1) / s, splits = (steps + per - 1) / per;
      if (splits != s) continue;
      if (s > 1 && tiles * s > 4 * slots) break;
      const long rounds = tiles * s / slots, rest = tiles * s % slots;
      const double on_cu = rest > CUS ? (double)rest / CUS : 1.0, step = f.one + (f.per_cu > 1 ? (f.full - f.one) * (on_cu - 1.0) / (f.per_cu - 1) : 0.0);
      const double us = rounds * (per * f.full + f.fixed) + (rest ? per * step + f.fixed : 0.0) + (s > 1 ? 4.5 + (double)M * N * (8.0 * s + 2.0) / 6.0e6 : 0.0);
      if (us < best.us) best = {c, (int)s, (int)per, us};
    }
  }
  return best;
}

// dx (M x K over N) and dw (N x K over M) in one launch of the same small tile, where that is estimated to be faster than one after the other
struct BothPlan { bool use; Plan dx, dw; };
BothPlan both_plan_of(long M, long N, long K, const Plan& dx, const Plan& dw) {
  BothPlan best = {false, dx, dw};
  double least = dx.us + dw.us + 3.0;                    // (a launch between them)
  const long xs = (N + BK - 1) / BK, ws = (M + BK - 1) / BK;
  for (int c = 2; c < 4; ++c) {
    const Config& f = CONFIGS[c];
    const long tx = ((M + f.bm - 1) / f.bm) * ((K + f.bn - 1) / f.bn), tw = ((N + f.bm - 1) / f.bm) * ((K + f.bn - 1) / f.bn), slots = (long)f.per_cu * CUS;
    for (long s = 1; s <= MAX_SPLITS && s <= ws; ++s) {
      const long per = (ws + s - 1) / s;
      if ((ws + per - 1) / per != s) continue;
      const long blocks = tx + tw * s;
      if (s > 1 && blocks > 4 * slots) break;
      const double on_cu = blocks >= slots ? f.per_cu : blocks > CUS ? (double)blocks / CUS : 1.0, step = f.one + (f.full - f.one) * (on_cu - 1.0) / (f.per_cu - 1);
      const double x = xs * step + f.fixed, w = per * step + f.fixed, all = (tx * x + tw * s * w) / (on_cu * CUS);
      const double us = (all > w ? (all > x ? all : x) : (w > x ? w : x)) + 0.5 * (x < w ? x : w) * (blocks > slots) + (s > 1 ? 4.5 + (double)N * K * (8.0 * s + 2.0) / 6.0e6 : 0.0);
      if (us < least) { least = us; best = {true, {c, 1, (int)xs, us}, {c, (int)s, (int)per, us}}; }
    }
  }
  return best;
}

long round256(long b) { return (b + 255) & ~255L; }
long part_bytes(const Plan& p, long M, long N) { return p.splits > 1 ? round256(p.splits * M * ((N + 7) / 8 * 8) * 4) : 0; }

template <typename T, bool AKS, bool BKS, int WM, int WN, int MT, int NT>
int launch_cfg(const MatParams& p, hipStream_t st) {
  constexpr int LDS = 2 * (16 * MT * WM + 16 * NT * WN) * 128 + 16 * NT * WN * 4;        // the tiles, the bias
  static bool done[HI3D_MAX_DEVICES];
  if (const int rc = hi3d_raise_lds_limit((const void*)mat_kernel<T, AKS, BKS, WM, WN, MT, NT>, LDS, done)) return rc;
  hipLaunchKernelGGL((mat_kernel<T, AKS, BKS, WM, WN, MT, NT>), dim3((unsigned)(p.nbm * p.nbn * p.splits)), dim3(WM * WN * 64), LDS, st, p);
  HI3D_LAUNCH_CHECK();
  return 0;
}
unsigned grid_of(long items) { const long n = (items + 255) / 256; return (unsigned)(n < 1 ? 1 : n > 8192 ? 8192 : n); }

void set_plan(MatParams* p, const Plan& plan, float* part) {
  const Config& f = CONFIGS[plan.cfg];
  p->nbm = (p->M + f.bm - 1) / f.bm; p->nbn = (p->N + f.bn - 1) / f.bn;
  p->splits = plan.splits; p->per = plan.per; p->part = plan.splits > 1 ? part : nullptr;
  p->group = 8;
}
template <typename T>
int join(const MatParams& p, hipStream_t st) {
  if (p.splits == 1) return 0;
  const long chunks = (long)p.M * ((p.N + 7) / 8);
  if (p.splits >= 8) hipLaunchKernelGGL((join_kernel<T, 8>), dim3(grid_of(chunks * 8)), dim3(256), 0, st, (const float*)p.part, p.e, (long)p.M, p.N, p.splits);
  else hipLaunchKernelGGL((join_kernel<T, 1>), dim3(grid_of(chunks)), dim3(256), 0, st, (const float*)p.part, p.e, (long)p.M, p.N, p.splits);
  HI3D_LAUNCH_CHECK();
  return 0;
}
template <typename T, bool AKS, bool BKS>
int launch_mat(MatParams p, const Plan& plan, float* part, hipStream_t st) {
  set_plan(&p, plan, part);
  int rc;
  if (plan.cfg == 0) rc = launch_cfg<T, AKS, BKS, 2, 4, 8, 4>(p, st);
  else if (plan.cfg == 1) rc = launch_cfg<T, AKS, BKS, 2, 4, 8, 5>(p, st);
  else if (plan.cfg == 2) rc = launch_cfg<T, AKS, BKS, 2, 2, 4, 4>(p, st);
  else rc = launch_cfg<T, AKS, BKS, 2, 2, 2, 2>(p, st);
  return rc ? rc : join<T>(p, st);
}
template <typename T, int WM, int WN, int MT, int NT>
int launch_both(const MatParams& dw, const MatParams& dx, hipStream_t st) {
  constexpr int LDS = 2 * (16 * MT * WM + 16 * NT * WN) * 128 + 16 * NT * WN * 4;
  static bool done[HI3D_MAX_DEVICES];
  if (const int rc = hi3d_raise_lds_limit((const void*)both_gradients_kernel<T, WM, WN, MT, NT>, LDS, done)) return rc;
  const int first = dw.nbm * dw.nbn * dw.splits;
  hipLaunchKernelGGL((both_gradients_kernel<T, WM, WN, MT, NT>), dim3((unsigned)(first + dx.nbm * dx.nbn * dx.splits)), dim3(WM * WN * 64), LDS, st, dw, dx, first);
  HI3D_LAUNCH_CHECK();
  return 0;
}

// whether rows of `cols` elements can be read in place
bool in_place(const void* p, long ld, long cols) { return !((uintptr_t)p & 15) && ld % 8 == 0 && ld <= MOST_PITCH && cols % 8 == 0; }
long padded_bytes(long rows, long cols) { return round256(rows * ((cols + 7) / 8 * 8) * 2); }

struct Operand { const void* p; long ld; };
// the operand itself, or -- where the kernel cannot read it in place -- where its padded copy will be at *ws, which moves on; the copy is `job`'s
Operand place(const void* p, long rows, int cols, long ld, char** ws, PadParams* job) {
  if (in_place(p, ld, cols)) return {p, ld};
  char* const to = *ws;
  *ws += padded_bytes(rows, cols);
  const long blocks = (rows * ((cols + 7L) / 8) + 255) / 256;             // (a chunk a thread while that fills the chip: each is a trip to memory)
  *job = {p, to, rows, ld, cols, (int)(blocks < 8192 ? blocks : 8192)};
  return {to, (cols + 7L) / 8 * 8};
}
template <typename T>
int prepare(const SlopeParams& s, int slices, const PadParams& a, const PadParams& b, hipStream_t st) {
  const int cols = s.M <= SLOPE_FEW ? 64 : 256, across = (s.N + cols - 1) / cols, n = across * slices;
  if (n + a.blocks + b.blocks == 0) return 0;
  hipLaunchKernelGGL((prepare_kernel<T>), dim3((unsigned)(n + a.blocks + b.blocks)), dim3(256), 0, st, s, across > 0 ? across : 1, n, a, b);
  HI3D_LAUNCH_CHECK();
  return 0;
}

constexpr int SLOPE_BLOCKS = 2048;
int slope_rows(long M, int N) {
  if (M <= SLOPE_FEW) return SLOPE_FEW;
  const long cols = (N + 255) / 256, want = SLOPE_BLOCKS / cols > 0 ? SLOPE_BLOCKS / cols : 1;
  long rows = (M + want - 1) / want;
  rows = rows < 32 ? 32 : (rows + 7) / 8 * 8;
  return (int)rows;
}
int slope_slices(long M, int N) { const int r = slope_rows(M, N); return (int)((M + r - 1) / r); }

const char* bad_desc(const hi3d_linear_desc* d) {
  if (!d) return "linear training: null descriptor";
  if (d->M < 0 || d->N <= 0 || d->K <= 0) return "linear training: negative row count, or width < 1";
  if (d->dtype != HI3D_BF16 && d->dtype != HI3D_F16) return "linear training: bf16 or fp16 operands";
  if (d->bias_dtype != HI3D_F32 && d->bias_dtype != d->dtype) return "linear training: bias of fp32 or of the operands' type";
  if (d->act < HI3D_ACT_NONE || d->act > HI3D_ACT_RELU) return "linear training: unknown activation";
  return nullptr;
}
// An operand of one row has no pitch: whatever the caller gave, its width stands in for it.  What lies behind the last row of a contraction is kept out by
// its distance from the descriptor's range, so that a pitch under the width would have read the one row again for every row behind it.
hi3d_linear_desc one_row_pitches(hi3d_linear_desc d) {
  if (d.M == 1) { d.ldx = d.K; d.ldr = d.lddy = d.ldz = d.N; }
  if (d.N == 1) d.ldw = d.K;
  return d;
}
bool too_big(const hi3d_linear_desc* d) { return d->M > 0x7fff0000L || d->N > MOST_WIDTH || d->K > MOST_WIDTH; }

// Up to 32 rows the weights are streamed by few_rows_kernel, above that the tiles are faster (N = K = 4096, 32 / 48 / 65 rows: streamed 14 /
// 19 us, tiles 18 us for up to 128).
constexpr int FEW = 32;
template <typename T, int MT, int CS>
int launch_few(const FewParams& p, hipStream_t st) {
  hipLaunchKernelGGL((few_rows_kernel<T, MT, CS>), dim3((p.N + 16 / CS - 1) / (16 / CS)), dim3(FEW_WAVES * 64), 0, st, p);
  HI3D_LAUNCH_CHECK();
  return 0;
}
template <typename T>
int few_rows(const FewParams& p, hipStream_t st) {
  // pieces of the contraction: as the rows leave room for them, while a wave keeps two steps of 32 and there are no more blocks than CUs (one
  // row, N = 4096, K = 4096: 1, 2, 4 pieces 10, 12, 15 us)
  if (p.M > 16) return launch_few<T, 2, 1>(p, st);
  if (p.M <= 4 && p.K >= 4 * FEW_WAVES * 64 && p.N <= 4 * CUS) return launch_few<T, 1, 4>(p, st);
  if (p.M <= 8 && p.K >= 2 * FEW_WAVES * 64 && p.N <= 8 * CUS) return launch_few<T, 1, 2>(p, st);
  return launch_few<T, 1, 1>(p, st);
}

// The rows that tiles take: all of them, or -- where up to 32 rows behind the last whole 256 would cost more as tiles than as streamed
// weights -- all but those (4112 rows of 1280 -> 5120: 4096 fill the chip once, with the 16 in tiles of 128 it takes 75 us, with them streamed 66, gelu and z kept).
struct FwdNeeds { long rows, x, w, part; Plan plan; };
FwdNeeds fwd_needs(const hi3d_linear_desc* d) {
  FwdNeeds n = {};
  if (d->M <= FEW) return n;
  n.rows = d->M;
  n.plan = plan_of(d->M, d->N, d->K);
  const long rest = d->M % 256;
  if (d->M > 256 && rest && rest <= FEW) {
    const Plan p = plan_of(d->M - rest, d->N, d->K);
    if (p.us + 4.0 + (double)d->N * d->K * 2.0 / 2.5e6 < n.plan.us) { n.rows = d->M - rest; n.plan = p; }
  }
  if (!in_place(d->x, d->ldx, d->K)) n.x = padded_bytes(n.rows, d->K);
  if (!in_place(d->w, d->ldw, d->K)) n.w = padded_bytes(d->N, d->K);
  n.part = part_bytes(n.plan, n.rows, d->N);
  return n;
}
struct BwdNeeds { long dz, x, w, part, cols; Plan dx, dw; bool both; };
BwdNeeds bwd_needs(const hi3d_linear_desc* d) {
  BwdNeeds n = {};
  const bool copy = d->act != HI3D_ACT_NONE || !in_place(d->dy, d->lddy, d->N);
  if ((d->dx || d->dw) && copy) n.dz = padded_bytes(d->M, d->N);
  if (d->dw && !in_place(d->x, d->ldx, d->K)) n.x = padded_bytes(d->M, d->K);
  if (d->dx && !in_place(d->w, d->ldw, d->K)) n.w = padded_bytes(d->N, d->K);
  n.dx = plan_of(d->M, d->K, d->N);
  n.dw = plan_of(d->N, d->K, d->M);
  if (d->dx && d->dw) {
    const BothPlan b = both_plan_of(d->M, d->N, d->K, n.dx, n.dw);
    n.both = b.use; n.dx = b.dx; n.dw = b.dw;
  }
  const long a = d->dx ? part_bytes(n.dx, d->M, d->K) : 0, b = d->dw ? part_bytes(n.dw, d->N, d->K) : 0;
  n.part = a > b ? a : b;
  if (d->db && d->M > SLOPE_FEW) n.cols = round256((long)slope_slices(d->M, d->N) * d->N * 4);
  return n;
}

template <typename T>
int fwd(const hi3d_linear_desc* d, hipStream_t st) {
  const FwdNeeds n = fwd_needs(d);
  const Epilogue e = {d->bias, d->residual, d->y, d->z, (long)d->ldr, (long)d->N, d->bias_dtype, d->act};
  if (n.rows < d->M) {
    const long r = n.rows;
    auto down = [&](const void* p, long ld) { return p ? (void*)((T*)p + r * ld) : nullptr; };
    const Epilogue f = {d->bias, down(d->residual, d->ldr), down(d->y, d->N), down(d->z, d->N), (long)d->ldr, (long)d->N, d->bias_dtype, d->act};
    const FewParams p = {down(d->x, d->ldx), d->w, f, (long)d->ldx, (long)d->ldw, (int)(d->M - r), d->N, d->K};
    const int rc = few_rows<T>(p, st);
    if (rc || !r) return rc;
  }
  char* ws = (char*)d->ws;
  PadParams jx = {}, jw = {};
  const Operand x = place(d->x, n.rows, d->K, d->ldx, &ws, &jx), w = place(d->w, d->N, d->K, d->ldw, &ws, &jw);
  if (const int rc = prepare<T>(SlopeParams{}, 0, jx, jw, st)) return rc;
  MatParams p = {};
  p.A = (const char*)x.p; p.B = (const char*)w.p; p.lda = x.ld; p.ldb = w.ld;
  p.M = (int)n.rows; p.N = d->N; p.K = d->K;
  p.e = e;
  return launch_mat<T, false, false>(p, n.plan, (float*)ws, st);
}

template <typename T>
int bwd(const hi3d_linear_desc* d, hipStream_t st) {
  const BwdNeeds n = bwd_needs(d);
  char* ws = (char*)d->ws;
  Operand dz = {d->dy, (long)d->lddy};
  SlopeParams sp = {d->dy, d->z, nullptr, nullptr, (long)d->M, (long)d->lddy, (long)d->ldz, nullptr, d->N, d->act, slope_rows(d->M, d->N), d->bias_dtype};
  if (n.dz) { sp.dz = ws; dz = {ws, (d->N + 7L) / 8 * 8}; ws += n.dz; }
  if (n.cols) { sp.part = (float*)ws; ws += n.cols; }
  else sp.db = d->db;
  const int slices = (n.dz || d->db) ? slope_slices(d->M, d->N) : 0;
  PadParams jw = {}, jx = {};
  Operand w = {}, x = {};
  if (d->dx) w = place(d->w, d->N, d->K, d->ldw, &ws, &jw);
  if (d->dw) x = place(d->x, d->M, d->K, d->ldx, &ws, &jx);
  if (const int rc = prepare<T>(sp, slices, jw, jx, st)) return rc;
  if (sp.part)
    if (const int rc = hi3d_column_reduce(sp.part, d->db, nullptr, d->bias_dtype, 0, slices, d->N, d->N, st)) return rc;
  float* const part = (float*)ws;                   // (dx's and dw's in turn: they follow each other on the stream, and in one launch only dw is split)
  MatParams px = {}, pw = {};
  px.A = (const char*)dz.p; px.B = (const char*)w.p; px.lda = dz.ld; px.ldb = w.ld;
  px.M = (int)d->M; px.N = d->K; px.K = d->N;
  px.e = {nullptr, nullptr, d->dx, nullptr, 0, (long)d->K, HI3D_F32, HI3D_ACT_NONE};
  pw.A = (const char*)dz.p; pw.B = (const char*)x.p; pw.lda = dz.ld; pw.ldb = x.ld;
  pw.M = d->N; pw.N = d->K; pw.K = (int)d->M;
  pw.e = {nullptr, nullptr, d->dw, nullptr, 0, (long)d->K, HI3D_F32, HI3D_ACT_NONE};
  if (n.both) {
    set_plan(&px, n.dx, part);
    set_plan(&pw, n.dw, part);
    const int rc = n.dx.cfg == 2 ? launch_both<T, 2, 2, 4, 4>(pw, px, st) : launch_both<T, 2, 2, 2, 2>(pw, px, st);
    return rc ? rc : join<T>(pw, st);
  }
  if (d->dx)
    if (const int rc = launch_mat<T, false, true>(px, n.dx, part, st)) return rc;
  return d->dw ? launch_mat<T, true, true>(pw, n.dw, part, st) : 0;
}

}  // namespace

extern "C" int64_t hi3d_linear_fwd_workspace_bytes(const hi3d_linear_desc* desc) {
  if (bad_desc(desc) || too_big(desc) || desc->M == 0) return 0;
  const hi3d_linear_desc d = one_row_pitches(*desc);
  const FwdNeeds n = fwd_needs(&d);
  return n.x + n.w + n.part;
}

extern "C" int hi3d_linear_fwd(const hi3d_linear_desc* desc, void* stream) {
  if (const char* why = bad_desc(desc)) HI3D_FAIL(HI3D_EINVAL, why);
  const hi3d_linear_desc local = one_row_pitches(*desc), *const d = &local;
  if (too_big(d)) HI3D_FAIL(HI3D_ESHAPE, "linear_fwd: a width is over 1048576, or too many rows");
  if (d->M == 0) return 0;
  if (!d->x || !d->w || !d->y) HI3D_FAIL(HI3D_EINVAL, "linear_fwd: null pointer");
  if (d->ldx < d->K || (d->residual && d->ldr < d->N) || d->ldw < d->K) HI3D_FAIL(HI3D_EINVAL, "linear_fwd: row pitch below the width");
  const int64_t need = hi3d_linear_fwd_workspace_bytes(d);
  if (need && (!d->ws || d->ws_bytes < need || ((uintptr_t)d->ws & 255))) HI3D_FAIL(HI3D_EINVAL, "linear_fwd: workspace missing, too small or not 256-byte aligned");
  return d->dtype == HI3D_BF16 ? fwd<bf16_t>(d, (hipStream_t)stream) : fwd<half_t>(d, (hipStream_t)stream);
}

extern "C" int64_t hi3d_linear_bwd_workspace_bytes(const hi3d_linear_desc* desc) {
  if (bad_desc(desc) || too_big(desc) || desc->M == 0) return 0;
  const hi3d_linear_desc d = one_row_pitches(*desc);
  const BwdNeeds n = bwd_needs(&d);
  return n.dz + n.x + n.w + n.cols + n.part;
}

extern "C" int hi3d_linear_bwd(const hi3d_linear_desc* desc, void* stream) {
  if (const char* why = bad_desc(desc)) HI3D_FAIL(HI3D_EINVAL, why);
  const hi3d_linear_desc local = one_row_pitches(*desc), *const d = &local;
  if (too_big(d)) HI3D_FAIL(HI3D_ESHAPE, "linear_bwd: a width is over 1048576, or too many rows");
  const hipStream_t st = (hipStream_t)stream;
  if (d->M == 0) {                       // sums over no rows
    if (d->db)
      if (const int rc = hi3d_column_reduce(nullptr, d->db, nullptr, d->bias_dtype, 0, 0, d->N, d->N, st)) return rc;
    if (d->dw) {
      const Epilogue e = {nullptr, nullptr, d->dw, nullptr, 0, (long)d->K, HI3D_F32, HI3D_ACT_NONE};
      const dim3 grid(grid_of((long)d->N * ((d->K + 7) / 8)));
      if (d->dtype == HI3D_BF16) hipLaunchKernelGGL((join_kernel<bf16_t, 1>), grid, dim3(256), 0, st, nullptr, e, (long)d->N, d->K, 0);
      else hipLaunchKernelGGL((join_kernel<half_t, 1>), grid, dim3(256), 0, st, nullptr, e, (long)d->N, d->K, 0);
      HI3D_LAUNCH_CHECK();
    }
    return 0;
  }
  if (!d->dy || (d->dx && !d->w) || (d->dw && !d->x) || (d->act != HI3D_ACT_NONE && !d->z)) HI3D_FAIL(HI3D_EINVAL, "linear_bwd: null pointer");
  if (d->lddy < d->N || (d->act != HI3D_ACT_NONE && d->ldz < d->N) || (d->dw && d->ldx < d->K) || (d->dx && d->ldw < d->K))
    HI3D_FAIL(HI3D_EINVAL, "linear_bwd: row pitch below the width");
  const int64_t need = hi3d_linear_bwd_workspace_bytes(d);
  if (need && (!d->ws || d->ws_bytes < need || ((uintptr_t)d->ws & 255))) HI3D_FAIL(HI3D_EINVAL, "linear_bwd: workspace missing, too small or not 256-byte aligned");
  return d->dtype == HI3D_BF16 ? bwd<bf16_t>(d, st) : bwd<half_t>(d, st);
}
