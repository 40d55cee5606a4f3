// kernels_snap.hip -- served snapshots of a population's nets (gfx950): laying a net out in 32 or 4 bits, answering rows with
// every agent's net, a mixture of all nets behind a router, and the router's gradient.  Layout: snap_internal.h.
#include "pop_internal.h"
#include "snap_internal.h"
#include <math.h>

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// a run-time index into a by-value kernel argument makes the compiler copy the argument to scratch: select instead
template <class T>
__device__ __forceinline__ T pick(const T (&v)[SNAP_MAXL], int l) {
  T r = v[0];
#pragma unroll
  for (int i = 1; i < SNAP_MAXL; ++i) r = l == i ? v[i] + 0 : r;       // (a value: of two lvalues ?: would select the address)
  return r;
}

__device__ __forceinline__ float snap_act(int t, float x) {
  if (t == 1) return x > 0.f ? x : 0.01f * x;
  if (t == 2) return tanhf(x);
  if (t == 3) return x > 0.f ? x : (x != x ? x : 0.f);
  return x;
}

// ------------------------------------------------------------------------------------------------------------------------
// Loading.  One wave per (agent, layer, strip): lane (r, q) walks the k-steps of output r; the four lanes of an output agree
// on a block's largest magnitude.  With amax = m 2^e, m in [1, 2): amax <= 6 2^s for the least s = e - 2 (m <= 1.5) or e - 1,
// so the scale comes out of the exponent field alone, and w 2^-s is exact: the codes do not depend on any rounding of the
// machine's.  Bound by the reads of the fp32 parameters.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned snap_code(float v) {          // v = w / scale, |v| <= 6: nearest of the grid, halves to the even code
  const float a = fabsf(v);
  const unsigned c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c | (v < 0.f && c ? 8u : 0u);
}

extern "C" __global__ void __launch_bounds__(256)
snap_load_kernel(const SnapDesc nd, char *__restrict__ img, const SnapSource src, int all_strips) {
  const int wave = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if (wave >= all_strips) return;
  int l = 0, strip = wave;
  while (strip >= pick(nd.strips, l)) { strip -= pick(nd.strips, l); ++l; }
  const int K = pick(nd.in, l), N = pick(nd.out, l), n = strip * 16 + r, steps = pick(nd.steps, l);
  const float *w = src.w + (size_t)blockIdx.x * src.agent + pick(src.offw, l);
  const float *b = src.w + (size_t)blockIdx.x * src.agent + pick(src.offb, l);
  char *im = img + (size_t)blockIdx.x * nd.stride;
  const int kp = pick(src.kp, l);
  auto weight = [&](int k) -> float {
    if (n >= N || k >= K) return 0.f;
    return src.tiled ? w[ddrl_widx(n, k, kp)] : w[(size_t)n * K + k];
  };
  bool bad = false;
  if (nd.bits == 4) {
    for (int s = 0; s < steps; ++s) {
      float v[8], amax = 0.f;
      bool wild = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = weight(32 * s + 8 * q + i);
        const float a = fabsf(v[i]);
        wild = wild || !(a < 0x1p126f);
        amax = fmaxf(amax, a);
      }
      amax = fmaxf(amax, __shfl_xor(amax, 16)); amax = fmaxf(amax, __shfl_xor(amax, 32));
      int any = wild ? 1 : 0;
      any |= __shfl_xor(any, 16); any |= __shfl_xor(any, 32);
      bad = bad || any;
      const unsigned bits = __float_as_uint(amax);
      const int e = (int)(bits >> 23) - 127, sh = (bits & 0x7fffffu) <= 0x400000u ? e - 2 : e - 1;
      const bool none = any || amax < 0x1p-118f;
      const float inv = none ? 0.f : __uint_as_float((unsigned)(127 - sh) << 23);
      unsigned c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) c |= (none ? 0u : snap_code(v[i] * inv)) << (4 * i);
      *(unsigned *)(im + pick(nd.woff, l) + snap_code_off(steps, strip, s, lane)) = c;
      if (q == 0) im[pick(nd.soff, l) + snap_scale_off(steps, strip, s, r)] = (char)(none ? 127 : sh + 127);
    }
    if (q == 0) for (int s = steps; s & 3; ++s) im[pick(nd.soff, l) + snap_scale_off(steps, strip, s, r)] = 127;
  } else {
    for (int s = 0; s < steps; ++s) {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = weight(16 * s + 4 * q + i);
      *(f32x4 *)(im + pick(nd.woff, l) + ((size_t)strip * steps + s) * 1024 + lane * 16) = v;
    }
  }
  if (q == 0) ((float *)(im + pick(nd.boff, l)))[n] = n >= N ? 0.f : bad ? __uint_as_float(0x7fc00000u) : b[n];
}

extern "C" hipError_t snap_load_launch(const SnapDesc *nd, char *img, const SnapSource *src, int G, hipStream_t st) {
  int all = 0;
  for (int l = 0; l < nd->L; ++l) all += nd->strips[l];
  hipLaunchKernelGGL(snap_load_kernel, dim3(G, (all + 3) / 4), dim3(256), 0, st, *nd, img, *src, all);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------------
// One net on a tile of rows, by one workgroup: D[16 outputs x 16 rows] += A (weights) B (activations) on the matrix cores, a
// wave per strip of outputs, activations in LDS between the layers (one barrier a layer).
//   32 bits: v_mfma_f32_16x16x4_f32.
//    4 bits: v_mfma_f32_16x16x32_bf16.  A weight (2 significant bits times a power of two) is exact in bf16, decoded with its
//            scale by v_cvt_scalef32_pk_bf16_fp4, two weights an instruction; an activation x is exactly the sum of three
//            bf16 numbers (x's leading 8 bits, the next 8, the last 8), so three products with fp32 accumulation lose no more
//            than an fp32 product does, at 5 times the fp32 matrix rate.
//            PACK (up to 5 rows): the three parts of a row are three columns of ONE matrix instruction, summed over the
//            columns at the end, instead of three instructions with 16 rows each.
// ------------------------------------------------------------------------------------------------------------------------
struct SnapLds { int second; };       // the inputs of layers 0, 2 lie in the first LDS buffer, those of 1, 3 in the second: where that starts

template <int BITS, int NT, bool PACK>
struct SnapShape {
  static constexpr int T = PACK ? 5 : 16 * NT;                               // rows of a tile
  static constexpr int ROWS = BITS == 4 ? (PACK ? 15 : 48 * NT) : 16 * NT;   // rows of an LDS buffer
  // a row's stride = 16 (mod 32) bytes, so that the 16 lanes that read 16 bytes of 16 rows at once start on distinct banks
  __host__ __device__ static int ld(int K) { return BITS == 4 ? ddrl_roundup(K, 32) * 2 + 16 : ddrl_roundup(K, 16) * 4 + 16; }
  static int bytes(const SnapDesc &nd, SnapLds &m) {
    int a = 0, b = 0;
    for (int l = 0; l < nd.L; ++l) { int &w = l & 1 ? b : a; w = ld(nd.d[l]) > w ? ld(nd.d[l]) : w; }
    m.second = ROWS * a;
    return ROWS * (a + b);
  }
};

__device__ __forceinline__ unsigned short bf_top(float x) { return (unsigned short)(__float_as_uint(x) >> 16); }
// x = p[0] + p[1] + p[2] exactly (down to 2^-133; an infinity or NaN is all in p[0])
__device__ __forceinline__ void split3(float x, unsigned short (&p)[3]) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const bool fin = fabsf(x) < __uint_as_float(0x7f800000u);
  const float r1 = fin ? x - hi : 0.f, mid = __uint_as_float(__float_as_uint(r1) & 0xffff0000u), lo = r1 - mid;
  p[0] = x != x ? 0x7fc0 : bf_top(x); p[1] = bf_top(mid); p[2] = bf_top(lo);
}
// the row of an LDS buffer that holds part p of a tile's row t
template <int BITS, int NT, bool PACK>
__device__ __forceinline__ int part_row(int t, int p) { return PACK ? 3 * t + p : p * 16 * NT + t; }

// `rows(t)`: where row t of the tile lies, or null; all threads of the workgroup, no barrier inside
template <int BITS, int NT, bool PACK, class Rows>
__device__ __forceinline__ void tile_in(int K, char *buf, Rows rows) {
  using S = SnapShape<BITS, NT, PACK>;
  const int ld = S::ld(K), Kp = BITS == 4 ? (K + 31) & ~31 : (K + 15) & ~15;
  for (int i = threadIdx.x; i < S::T * Kp; i += blockDim.x) {
    const int t = i / Kp, k = i - t * Kp;
    const float *x = rows(t);
    const float v = x && k < K ? x[k] : 0.f;
    if (BITS == 4) {
      unsigned short p[3];
      split3(v, p);
#pragma unroll
      for (int j = 0; j < 3; ++j) *(unsigned short *)(buf + part_row<BITS, NT, PACK>(t, j) * ld + k * 2) = p[j];
    } else *(float *)(buf + t * ld + k * 4) = v;
  }
}

template <int BITS, int NT, bool PACK, class Out>
__device__ __forceinline__ void net_tile(const SnapDesc &nd, const SnapLds &m, const char *__restrict__ img, char *lds, Out out) {
  constexpr int P = BITS == 4 && !PACK ? 3 : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, c = lane & 15, q = lane >> 4;
  for (int l = 0; l < nd.L; ++l) {
    const char *xin = lds + (l & 1 ? m.second : 0);
    char *xout = lds + (l & 1 ? 0 : m.second);
    const int N = pick(nd.out, l), strips = pick(nd.strips, l), steps = pick(nd.steps, l), ldi = SnapShape<BITS, NT, PACK>::ld(pick(nd.in, l));
    const bool last = l == nd.L - 1;
    const int ldo = SnapShape<BITS, NT, PACK>::ld(N), act = last ? nd.oact : nd.hact;
    const char *wl = img + pick(nd.woff, l), *sl = img + pick(nd.soff, l);
    const float *bl = (const float *)(img + pick(nd.boff, l));
    for (int s = wave; s < strips; s += waves) {
      f32x4 acc[NT][P];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) acc[i][p] = f32x4{0.f, 0.f, 0.f, 0.f};
      const f32x4 bias = *(const f32x4 *)(bl + s * 16 + 4 * q);
      if constexpr (BITS == 4) {
        const int xrow = PACK ? (c < 15 ? c : 0) : c;
        auto step = [&](unsigned code, unsigned sb, int at) {
          const float sc = __uint_as_float(sb << 23);
          union { bf16x2 h[4]; bf16x8 v; } a;
          a.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 0);
          a.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 1);
          a.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 2);
          a.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, sc, 3);
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int p = 0; p < P; ++p) {
              const bf16x8 b = *(const bf16x8 *)(xin + (p * 16 * NT + 16 * i + xrow) * ldi + at * 64 + q * 16);
              acc[i][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b, acc[i][p], 0, 0, 0);
            }
        };
        const char *ws = wl + (size_t)s * steps * 256, *ss = sl + (size_t)s * ((steps + 3) >> 2) * 64 + c * 4;
        const int full = steps >> 2;
        for (int b = 0; b < full; ++b) {
          const u32x4 code = *(const u32x4 *)(ws + b * 1024 + lane * 16);
          const unsigned sb = *(const unsigned *)(ss + b * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) step(code[j], (sb >> (8 * j)) & 255u, 4 * b + j);
        }
        if (steps & 3) {
          const unsigned sb = *(const unsigned *)(ss + full * 64);
          for (int j = 0; j < (steps & 3); ++j)
            step(*(const unsigned *)(ws + full * 1024 + j * 256 + lane * 4), (sb >> (8 * j)) & 255u, 4 * full + j);
        }
      } else {
        const char *ws = wl + (size_t)s * steps * 1024 + lane * 16;
        for (int b = 0; b < steps; ++b) {
          const f32x4 a = *(const f32x4 *)(ws + b * 1024);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const f32x4 x = *(const f32x4 *)(xin + (16 * i + c) * ldi + b * 64 + q * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], x[j], acc[i][0], 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f32x4 v = acc[i][0];
        if constexpr (P == 3) v = (acc[i][2] + acc[i][1]) + v;
        if constexpr (PACK) {                             // columns 3t, 3t + 1, 3t + 2 are the parts of row t
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int iv = __float_as_int(v[j]);
            const float m1 = __int_as_float(__builtin_amdgcn_update_dpp(0, iv, 0x101, 0xf, 0xf, true));   // row_shl:1 = column + 1
            const float m2 = __int_as_float(__builtin_amdgcn_update_dpp(0, iv, 0x102, 0xf, 0xf, true));
            v[j] = (m2 + m1) + v[j];
          }
        }
        const int t = PACK ? c / 3 : 16 * i + c;
        const bool mine = !PACK || (c % 3 == 0 && c < 15);
        const int n0 = s * 16 + 4 * q;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = n0 + j < N ? snap_act(act, v[j] + bias[j]) : 0.f;
        if (last) {
          if (mine) {
#pragma unroll
            for (int j = 0; j < 4; ++j) if (n0 + j < N) out(t, n0 + j, y[j]);
          }
        } else if (mine) {
          if constexpr (BITS == 4) {
            unsigned short p[4][3];
#pragma unroll
            for (int j = 0; j < 4; ++j) split3(y[j], p[j]);
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              char *o = xout + part_row<BITS, NT, PACK>(t, k) * ldo + n0 * 2;
              *(u32x2 *)o = u32x2{p[0][k] | (unsigned)p[1][k] << 16, p[2][k] | (unsigned)p[3][k] << 16};
              if (s == strips - 1 && (strips & 1)) *(u32x2 *)(o + 32) = u32x2{0u, 0u};      // the next layer's k-steps are 32 wide
            }
          } else *(f32x4 *)(xout + t * ldo + n0 * 4) = f32x4{y[0], y[1], y[2], y[3]};
        }
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// Every agent's net on its rows
// ------------------------------------------------------------------------------------------------------------------------
template <int BITS, int NT, bool PACK>
__global__ void __launch_bounds__(256)
snap_forward_kernel(const SnapDesc nd, const SnapLds m, const SnapForward p) {
  extern __shared__ __align__(16) char lds[];
  using S = SnapShape<BITS, NT, PACK>;
  const int g = blockIdx.x;
  if (p.mask && !p.mask[g]) return;
  const char *img = p.img + (size_t)g * nd.stride;
  const int from = blockIdx.y * p.per, to = min(p.n, from + p.per);
  for (int t0 = from; t0 < to; t0 += S::T) {
    const float *x = p.x + g * p.x_agent + t0 * p.x_row;
    tile_in<BITS, NT, PACK>(nd.in[0], lds, [&](int t) { return t0 + t < to ? x + t * p.x_row : (const float *)nullptr; });
    __syncthreads();
    float *o = p.out + g * p.out_agent + t0 * p.out_row;
    net_tile<BITS, NT, PACK>(nd, m, img, lds, [&](int t, int n, float v) { if (t0 + t < to) o[t * p.out_row + n] = v; });
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// The router.  One workgroup per 16 rows; a wave takes strips of 16 agents: logits[16 agents x 16 rows] on
// v_mfma_f64_16x16x4_f64.  Both factors are 32-bit numbers, so their products are exact and the sums are wrong by ~1e-16: two
// logits change places only where they are equal to 15 digits.  A lane holds 4 logits of one row a strip and keeps the KM best
// it has met, as keys that sort as the numbers do (NaN above all, 0 = barred); the lanes of a row, then the waves, merge their
// lists.  The index decides between equal keys.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long logit_key(double v) {
  if (v != v) return ~0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);       // -0 -> +0
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
#define KEY_NONE 0x000fffffffffffffull                     // the key of -infinity
__device__ __forceinline__ double key_logit(unsigned long long k) {
  if (k == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}
__device__ __forceinline__ bool key_before(unsigned long long ka, int ia, unsigned long long kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

template <int KM>
__global__ void __launch_bounds__(1024)
snap_router_kernel(const SnapMixture p, int S, int A, int ld) {
  extern __shared__ __align__(16) char lds[];
  float *xs = (float *)lds;                                // [16][ld]
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  unsigned long long *ck = (unsigned long long *)(lds + 16 * ld * 4);       // [16][waves][KM]
  int *ci = (int *)(ck + 16 * waves * KM);
  const int t0 = blockIdx.x * 16;
  const int Sp = (S + 15) & ~15;
  for (int i = threadIdx.x; i < 16 * Sp; i += blockDim.x) {
    const int t = i / Sp, k = i - t * Sp;
    xs[t * ld + k] = t0 + t < p.n && k < S ? p.x[(t0 + t) * p.x_row + k] : 0.f;
  }
  __syncthreads();
  unsigned long long K[KM];
  int I[KM];
#pragma unroll
  for (int j = 0; j < KM; ++j) { K[j] = KEY_NONE; I[j] = 0x7fffffff; }
  const int row = min(t0 + c, p.n - 1);
  const uint8_t *al = p.allowed ? p.allowed + row * p.a_row : nullptr;
  for (int s = wave; s * 16 < p.G; s += waves) {
    const float *w = p.rw + (int64_t)min(s * 16 + c, p.G - 1) * p.r_row;
    f64x4 acc = {0., 0., 0., 0.};
    for (int k = 0; k < S; k += 16) {
      const int at = k + 4 * q;
      float a[4];
      if (at + 3 < S) { const f32x4u v = *(const f32x4u *)(w + at); a[0] = v[0]; a[1] = v[1]; a[2] = v[2]; a[3] = v[3]; }
      else {
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = at + j < S ? w[at + j] : 0.f;
      }
      const f32x4 x = *(const f32x4 *)(xs + c * ld + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[j], (double)x[j], acc, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int e = s * 16 + 4 * j + q;
      unsigned long long key = KEY_NONE;
      if (e < p.G && (!al || al[e])) key = logit_key(acc[j] + (p.rb ? (double)p.rb[e] : 0.));
      if (key > K[KM - 1]) {
#pragma unroll
        for (int i = 0; i < KM; ++i) {
          const bool up = key > K[i];
          const unsigned long long tk = K[i]; const int te = I[i];
          K[i] = up ? key : tk; I[i] = up ? e : te;
          key = up ? tk : key; e = up ? te : e;
        }
      }
    }
  }
  // the four lanes of a row
  for (int j = 0; j < p.k; ++j) {
    unsigned long long bk = K[0];
    int bi = I[0];
#pragma unroll
    for (int d = 16; d <= 32; d *= 2) {
      const unsigned long long ok = __shfl_xor(bk, d);
      const int oi = __shfl_xor(bi, d);
      if (key_before(ok, oi, bk, bi)) { bk = ok; bi = oi; }
    }
    if (I[0] == bi) {
#pragma unroll
      for (int i = 0; i + 1 < KM; ++i) { K[i] = K[i + 1]; I[i] = I[i + 1]; }
      K[KM - 1] = KEY_NONE; I[KM - 1] = 0x7fffffff;
    }
    if (q == 0) { ck[(c * waves + wave) * KM + j] = bk; ci[(c * waves + wave) * KM + j] = bi; }
  }
  __syncthreads();
  // the waves: 16 lanes a row, lane u holds wave u's list; lane j keeps the j-th pick
  const int u = threadIdx.x & 15;
  for (int t = threadIdx.x >> 4; t < 16; t += blockDim.x >> 4) {
    const int tok = t0 + t;
    const bool live = tok < p.n;
    int head = 0, mi = 0x7fffffff;
    unsigned long long mk = KEY_NONE;
    for (int j = 0; j < p.k; ++j) {
      unsigned long long bk = KEY_NONE;
      int bi = 0x7fffffff;
      if (u < waves && head < p.k) { bk = ck[(t * waves + u) * KM + head]; bi = ci[(t * waves + u) * KM + head]; }
      const int own = bi;
#pragma unroll
      for (int d = 1; d <= 8; d *= 2) {
        const unsigned long long ok = __shfl_xor(bk, d);
        const int oi = __shfl_xor(bi, d);
        if (key_before(ok, oi, bk, bi)) { bk = ok; bi = oi; }
      }
      if (own == bi && bi != 0x7fffffff) ++head;
      if (u == j) { mk = bk; mi = bi; }
    }
    const bool have = mi != 0x7fffffff;
    const double l = key_logit(mk), top = __shfl(l, 0, 16);
    const float ex = have ? expf((float)(l - top)) : 0.f;
    float sum = 0.f;
    for (int j = 0; j < p.k; ++j) sum += __shfl(ex, j, 16);
    if (live && u < p.k) {
      p.idx[(int64_t)tok * p.k + u] = have ? mi : -1;
      p.prob[(int64_t)tok * p.k + u] = have ? ex / sum : 0.f;
      if (!have) for (int a = 0; a < A; ++a) p.y[((int64_t)tok * p.k + u) * A + a] = 0.f;
    }
    const int first = __shfl(mi, 0, 16);
    if (live && first == 0x7fffffff) for (int a = u; a < A; a += 16) p.out[tok * p.out_row + a] = 0.f;
    if (live && u == 0) p.count[tok] = 0;
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// The picked nets.  A workgroup answers, for one net, the places (row, j) of a piece of idx that picked it, T at a time, and
// whoever answers a row's last place sums the row up, in the order of its places whatever the order they were answered in.
// Few places: one workgroup per place, and the first place of a net takes the others along; many: one per (net, piece).
// ------------------------------------------------------------------------------------------------------------------------
#define SNAP_LIST 1024
template <int BITS, int NT, bool PACK>
__global__ void __launch_bounds__(256)
snap_experts_kernel(const SnapDesc nd, const SnapLds m, const SnapMixture p, int by_place, int piece) {
  extern __shared__ __align__(16) char lds[];
  using S = SnapShape<BITS, NT, PACK>;
  __shared__ int list[SNAP_LIST + 256], cnt, done[16 * NT > 5 ? 16 * NT : 5];
  const int tid = threadIdx.x, A = nd.A, total = p.n * p.k;
  int e, from, to;
  if (by_place) {
    from = blockIdx.x; to = total;
    e = p.idx[from];
    if (e < 0) return;
    int before = 0;
    for (int i = tid; i < from; i += 256) before |= p.idx[i] == e;
    if (__syncthreads_or(before)) return;
  } else {
    e = blockIdx.x;
    from = blockIdx.y * piece; to = min(total, from + piece);
  }
  const char *img = p.img + (size_t)e * nd.stride;
  while (from < to) {
    if (tid == 0) cnt = 0;
    __syncthreads();
    for (;;) {                                             // from and cnt are the same in all threads
      const int i = from + tid;
      if (i < to && p.idx[i] == e) list[atomicAdd(&cnt, 1)] = i;
      from += 256;
      __syncthreads();
      const int have = cnt;
      __syncthreads();
      if (from >= to || have > SNAP_LIST) break;
    }
    const int have = cnt;
    for (int i0 = 0; i0 < have; i0 += S::T) {
      tile_in<BITS, NT, PACK>(nd.in[0], lds, [&](int t) { return i0 + t < have ? p.x + (int64_t)(list[i0 + t] / p.k) * p.x_row : (const float *)nullptr; });
      __syncthreads();
      net_tile<BITS, NT, PACK>(nd, m, img, lds, [&](int t, int n, float v) {
        if (i0 + t < have) __hip_atomic_store(p.y + (int64_t)list[i0 + t] * A + n, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      });
      __threadfence();
      __syncthreads();
      if (tid < S::T) {
        int row = -1;
        if (i0 + tid < have) {
          const int r = list[i0 + tid] / p.k;
          int want = 0;
          for (int j = 0; j < p.k; ++j) want += p.idx[r * p.k + j] >= 0;
          if (__hip_atomic_fetch_add(p.count + r, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == want - 1) row = r;
        }
        done[tid] = row;
      }
      __syncthreads();
      __threadfence();
      for (int i = tid; i < S::T * A; i += 256) {
        const int t = i / A, a = i - t * A, r = done[t];
        if (r < 0) continue;
        float sum = 0.f;
        for (int j = 0; j < p.k; ++j)
          if (p.idx[r * p.k + j] >= 0)
            sum = fmaf(p.prob[r * p.k + j], __hip_atomic_load(p.y + ((int64_t)r * p.k + j) * A + a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), sum);
        p.out[r * p.out_row + a] = sum;
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// The router's gradient.  One workgroup per agent (and one more for the places that picked nobody): it walks idx in order and,
// for every 256 places that are its own, one thread each takes the place's dlogit, then all sum dlogit x over them: thread
// (u, s) over the places u, u + parts, .. of input s, in fp64 (an agent may be picked by every row).
// ------------------------------------------------------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256)
snap_grad_kernel(const SnapGrad p) {
  __shared__ int list[512], wsum[4];
  __shared__ float dl[512];
  __shared__ double part[256];
  const int e = blockIdx.x, tid = threadIdx.x, total = p.n * p.k, S = p.S, A = p.A;
  if (e == p.G) {                                          // dy of places that picked nobody
    if (!p.dy) return;
    for (int i = tid; i < total; i += 256) {
      const int v = p.idx[i];
      if (v >= 0 && v < p.G) continue;
      for (int a = 0; a < A; ++a) p.dy[(int64_t)i * A + a] = 0.f;
    }
    return;
  }
  const int s0 = S < 256 ? S : 256, parts = 256 / s0, u = tid / s0, sx = tid - u * s0;
  double acc[4] = {0., 0., 0., 0.}, bacc = 0.;             // S <= 1024
  int from = 0, have = 0;
  while (from < total) {
    while (from < total && have <= 256) {                  // ordered: wave by wave, lane by lane
      const int i = from + tid;
      const bool mine = i < total && p.idx[i] == e;
      const unsigned long long b = __ballot(mine);
      const int w = tid >> 6, lane = tid & 63;
      if (lane == 0) wsum[w] = __popcll(b);
      __syncthreads();
      int at = have;
      for (int j = 0; j < w; ++j) at += wsum[j];
      if (mine) list[at + __popcll(b & ((1ull << lane) - 1ull))] = i;
      have += wsum[0] + wsum[1] + wsum[2] + wsum[3];
      from += 256;
      __syncthreads();
    }
    for (int i = tid; i < have; i += 256) {
      const int place = list[i], r = place / p.k, j = place - r * p.k;
      const float *dout = p.dout + (int64_t)r * p.dout_row;
      float all = 0.f, own = 0.f;
      for (int v = 0; v < p.k; ++v) {
        const int ev = p.idx[r * p.k + v];
        if (ev < 0 || ev >= p.G) continue;
        float dot = 0.f;
        const float *y = p.y + ((int64_t)r * p.k + v) * A;
        for (int a = 0; a < A; ++a) dot = fmaf(y[a], dout[a], dot);
        all = fmaf(p.prob[r * p.k + v], dot, all);
        if (v == j) own = dot;
      }
      const float pr = p.prob[place];
      dl[i] = pr * (own - all);
      if (p.dy) for (int a = 0; a < A; ++a) p.dy[(int64_t)place * A + a] = pr * dout[a];
    }
    __syncthreads();
    if (u < parts)
      for (int i = u; i < have; i += parts) {
        const float *x = p.x + (int64_t)(list[i] / p.k) * p.x_row;
        const double d = dl[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) { const int s = sx + 256 * j; if (s < S && (j == 0 || s0 == 256)) acc[j] = fma(d, (double)x[s], acc[j]); }
        if (sx == 0) bacc += d;
      }
    have = 0;
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (256 * j >= S) break;
    part[tid] = acc[j];
    __syncthreads();
    if (u == 0 && sx + 256 * j < S) {
      double v = 0.;
      for (int i = 0; i < parts; ++i) v += part[i * s0 + sx];
      p.dw[(int64_t)e * p.dw_row + sx + 256 * j] = (float)v;
    }
    __syncthreads();
  }
  if (p.db) {
    part[tid] = bacc;
    __syncthreads();
    if (tid == 0) {
      double v = 0.;
      for (int i = 0; i < parts; ++i) v += part[i * s0];
      p.db[e] = (float)v;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------------------------------------
template <int BITS, int NT, bool PACK>
static hipError_t forward_run(const SnapDesc &nd, SnapForward p, hipStream_t st) {
  SnapLds m;
  const int lds = SnapShape<BITS, NT, PACK>::bytes(nd, m), T = SnapShape<BITS, NT, PACK>::T;
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_forward_kernel<BITS, NT, PACK>, lds, cfg);
  if (e != hipSuccess) return e;
  const int tiles = (p.n + T - 1) / T;
  int chunks = p.G >= 1024 ? 1 : (1024 + p.G - 1) / p.G;
  if (chunks > tiles) chunks = tiles;
  const int per = (tiles + chunks - 1) / chunks;
  p.per = per * T;
  hipLaunchKernelGGL((snap_forward_kernel<BITS, NT, PACK>), dim3(p.G, (tiles + per - 1) / per), dim3(256), lds, st, nd, m, p);
  return hipGetLastError();
}
template <int BITS, int NT, bool PACK>
static bool fits(const SnapDesc &nd, int more) { SnapLds m; return SnapShape<BITS, NT, PACK>::bytes(nd, m) + more <= SNAP_LDS; }

extern "C" hipError_t snap_forward_launch(const SnapDesc *nd, const SnapForward *p, hipStream_t st) {
  if (nd->bits == 4) {
    if (p->n > 16 && fits<4, 2, false>(*nd, 0)) return forward_run<4, 2, false>(*nd, *p, st);
    if (p->n > 5 && fits<4, 1, false>(*nd, 0)) return forward_run<4, 1, false>(*nd, *p, st);
    return forward_run<4, 1, true>(*nd, *p, st);
  }
  if (p->n > 16 && fits<32, 2, false>(*nd, 0)) return forward_run<32, 2, false>(*nd, *p, st);
  return forward_run<32, 1, false>(*nd, *p, st);
}

template <int KM>
static hipError_t router_run(const SnapMixture &p, int S, int A, hipStream_t st) {
  const int ld = ddrl_roundup(S, 64) + 4;
  int waves = 4;
  while (waves < 16 && waves * 16 < p.G) waves *= 2;
  const size_t lds = (size_t)16 * ld * 4 + (size_t)16 * waves * KM * 12;
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_router_kernel<KM>, lds, cfg);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(snap_router_kernel<KM>, dim3((p.n + 15) / 16), dim3(waves * 64), lds, st, p, S, A, ld);
  return hipGetLastError();
}
template <int BITS, int NT, bool PACK>
static hipError_t experts_run(const SnapDesc &nd, const SnapMixture &p, hipStream_t st) {
  SnapLds m;
  const int lds = SnapShape<BITS, NT, PACK>::bytes(nd, m);
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_experts_kernel<BITS, NT, PACK>, lds, cfg);
  if (e != hipSuccess) return e;
  const int total = p.n * p.k;
  if (total <= 1024) {
    hipLaunchKernelGGL((snap_experts_kernel<BITS, NT, PACK>), dim3(total), dim3(256), lds, st, nd, m, p, 1, 0);
  } else {
    int pieces = (1024 + p.G - 1) / p.G;
    int piece = ddrl_roundup((total + pieces - 1) / pieces, 256);
    hipLaunchKernelGGL((snap_experts_kernel<BITS, NT, PACK>), dim3(p.G, (total + piece - 1) / piece), dim3(256), lds, st, nd, m, p, 0, piece);
  }
  return hipGetLastError();
}

#define SNAP_STATIC_LDS 8192         // snap_experts_kernel's list and flags
extern "C" hipError_t snap_mixture_launch(const SnapDesc *nd, const SnapMixture *p, hipStream_t st) {
  const int S = nd->d[0], A = nd->d[nd->L];
  hipError_t e = p->k == 1 ? router_run<1>(*p, S, A, st) : p->k == 2 ? router_run<2>(*p, S, A, st) : p->k <= 4 ? router_run<4>(*p, S, A, st)
                                                                                                              : router_run<8>(*p, S, A, st);
  if (e != hipSuccess) return e;
  const int total = p->n * p->k;
  if (nd->bits == 4) {
    if (total > 5 * p->G && fits<4, 1, false>(*nd, SNAP_STATIC_LDS)) return experts_run<4, 1, false>(*nd, *p, st);
    return experts_run<4, 1, true>(*nd, *p, st);
  }
  return experts_run<32, 1, false>(*nd, *p, st);
}

extern "C" hipError_t snap_grad_launch(const SnapGrad *p, hipStream_t st) {
  hipLaunchKernelGGL(snap_grad_kernel, dim3(p->G + (p->dy ? 1 : 0)), dim3(256), 0, st, *p);
  return hipGetLastError();
}
