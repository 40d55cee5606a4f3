// kernels_snap.hip -- served snapshots of a population's nets (gfx950): laying a net out in 32 or 4 bits, answering rows with
// every agent's net, a mixture of all nets behind a router, and the router's gradient.  Layout: snap_internal.h.
#include "pop_internal.h"
#include "snap_internal.h"
#include <math.h>
#include <type_traits>

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(4)));

// The kernels' first argument in the kernel-argument memory itself: a layer is one scalar load there, whatever its number
// (a run-time index into the by-value argument would make the compiler copy it to scratch memory)
typedef const __attribute__((address_space(4))) SnapDesc *DescP;
#define SNAP_DESC(nd) ((DescP)__builtin_amdgcn_kernarg_segment_ptr())
struct LayerOf { int in, out, strips, steps, act, code; unsigned off, rec; };
__device__ __forceinline__ LayerOf layer_of(DescP nd, int l) {
  const __attribute__((address_space(4))) SnapLayer *y = &nd->lay[l];
  return LayerOf{y->in, y->out, y->strips, y->steps, y->act, y->code, y->off, y->rec};
}

// linear and leaky-ReLU are max(x, slope x), ReLU is max(x, 0), with a maximum that keeps NaN
__device__ __forceinline__ float act_one(int act, float x) {
  if (act == 2) return tanhf(x);
  return __builtin_elementwise_maximum(x, act == 3 ? 0.f : act == 1 ? 0.01f * x : x);
}
__device__ __forceinline__ f32x4 act_four(int act, f32x4 x) {
  if (act == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = tanhf(x[j]);
  } else if (act == 3) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __builtin_elementwise_maximum(x[j], 0.f);
  } else if (act == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __builtin_elementwise_maximum(x[j], 0.01f * x[j]);
  }
  return x;
}

// ------------------------------------------------------------------------------------------------------------------------
// Loading.  One wave per (agent, layer, strip): lane (r, q) walks the k-steps of output r; the four lanes of an output agree
// on a block's largest magnitude.  With amax = m 2^e, m in [1, 2): amax <= 6 2^s for the least s = e - 2 (m <= 1.5) or e - 1,
// so the scale comes out of the exponent field alone, and w 2^-s is exact: the codes do not depend on any rounding of the
// machine's.  Reads 16 bytes a lane and a block of four steps at a time, and waits for them: a block is asked for when the one before
// is encoded (1024 agents of 18-400-300-6 to 4 bits: 530 MB in, 84 MB out, 170 to 197 us, 3.1 to 3.6 TB/s; a
// copy reaches 4.8).
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned snap_code(float v) {          // v = w / scale, |v| <= 6: nearest of the grid, halves to the even code
  const float a = fabsf(v);
  const unsigned c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return c | (v < 0.f && c ? 8u : 0u);
}

extern "C" __global__ void __launch_bounds__(256)
snap_load_kernel(const SnapDesc nd_, const SnapSource src, char *__restrict__ img, int all_strips) {
  const DescP nd = SNAP_DESC(nd_);
  const int wave = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if (wave >= all_strips) return;
  int l = 0, strip = wave;
  while (strip >= nd->lay[l].strips) { strip -= nd->lay[l].strips; ++l; }
  const LayerOf y = layer_of(nd, l);
  const int K = y.in, N = y.out, n = strip * 16 + r, steps = y.steps;
  const __attribute__((address_space(4))) SnapSource *from = (const __attribute__((address_space(4))) SnapSource *)(nd + 1);
  const float *w = src.w + (size_t)blockIdx.x * src.agent + from->offw[l];
  const float *b = src.w + (size_t)blockIdx.x * src.agent + from->offb[l];
  char *rec = img + (size_t)blockIdx.x * nd->stride + y.off + strip * y.rec;
  const int kp = from->kp[l];
  // inputs k .. k + 3, k a multiple of 4 (four neighbours in memory in a tile too), zeros where there are none
  auto four = [&](int k) -> f32x4 {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= N || k >= K) return v;
    const float *from = w + (src.tiled ? (size_t)ddrl_widx(n, k, kp) : (size_t)n * K + k);
    if (k + 4 <= K) return *(const f32x4u *)from;
    for (int i = 0; i < 3; ++i) if (k + i < K) v[i] = from[i];
    return v;
  };
  bool bad = false;
  if (nd->bits == 4) {
#pragma unroll 1
    for (int s0 = 0; s0 < steps; s0 += 4) {
      f32x4 v[4][2];
      u32x4 codes;
      unsigned scales = 0;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[s][h] = four(32 * (s0 + s) + 8 * q + 4 * h);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float amax = 0.f;
        bool wild = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = fabsf(v[s][i >> 2][i & 3]);
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
        for (int i = 0; i < 8; ++i) c |= (none ? 0u : snap_code(v[s][i >> 2][i & 3] * inv)) << (4 * i);
        codes[s] = c;
        scales |= (unsigned)(none ? 127 : sh + 127) << (8 * s);
      }
      if (s0 + 4 <= steps) *(u32x4 *)(rec + snap_code_off(steps, s0, lane)) = codes;
      else {
#pragma unroll
        for (int s = 0; s < 3; ++s) if (s0 + s < steps) *(unsigned *)(rec + snap_code_off(steps, s0 + s, lane)) = codes[s];
      }
      if (q == 0) *(unsigned *)(rec + snap_scale_off(y.code, s0, r)) = scales;
    }
  } else {
#pragma unroll 4
    for (int s = 0; s < steps; ++s) *(f32x4 *)(rec + s * 1024 + lane * 16) = four(16 * s + 4 * q);
  }
  if (q == 0) ((float *)(rec + y.rec - 64))[r] = n >= N ? 0.f : bad ? __uint_as_float(0x7fc00000u) : b[n];
}

extern "C" hipError_t snap_load_launch(const SnapDesc *nd, char *img, const SnapSource *src, int G, hipStream_t st) {
  int all = 0;
  for (int l = 0; l < nd->L; ++l) all += nd->lay[l].strips;
  hipLaunchKernelGGL(snap_load_kernel, dim3(G, (all + 3) / 4), dim3(256), 0, st, *nd, *src, img, all);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------------
// One net on a tile of rows, by one workgroup: D[16 outputs x 16 columns] += A (weights) B (activations) on the matrix cores, a
// wave MT strips of outputs at a time, activations in LDS between the layers (one barrier a layer).
//   32 bits: v_mfma_f32_16x16x4_f32; a single row: v_fma_f32 on the lane's own 4 weights, the lanes of an output summed at the
//            end (the matrix instruction would take 8 times as long for one column of use).
//    4 bits: v_mfma_f32_16x16x32_bf16.  A weight (2 significant bits times a power of two) is exact in bf16, decoded with its
//            scale by v_cvt_scalef32_pk_bf16_fp4, two weights an instruction; an activation x is exactly the sum of three
//            bf16 numbers (x's leading 8 bits, the next 8, the last 8), so three products with fp32 accumulation lose no more
//            than an fp32 product does, at 5 times the fp32 matrix rate.
// R rows of 16 columns: 16 (a column each; 4 bits: three products, one for each part), 4 (4 columns each) or 1 (all 16 columns).
// With 4 bits and R < 16 the columns 4 t, 4 t + 1, 4 t + 2 are the parts of row t: ONE product, summed over the columns at the
// end.  And with R < 16 every lane finishes ONE output of the tile (bias, activation, the three parts) instead of a few lanes
// finishing four: with few rows that, not the product, is most of the instructions.
// Activations lie as the B operand is read, [k-step][part][16 rows][k quarter][row] x 16 bytes: a wave's read is 1 KiB without a
// bank conflict, every one of a block of steps at a constant distance from the first.  Instructions and waits, not bytes, bound a
// net of many rows, so what is left of addresses is a scalar or such a constant (1024 agents of 18-400-300-6, 64 rows: 94 us, 540
// TFLOP/s of the three bf16 products, the vector units at work 60 % of the time, the matrix cores 28, a wave waiting 52; 147 us with
// 7 vector instructions a product and row-major inputs.  A wave of several strips or tiles at once shares more, and leaves waves
// idle where a layer ends: 110 to 196 us).  One row is bound by the layers' latency, a wave waiting 60 % of its time, and by decoding
// and the sums' ends, half of the vector units' time, before its net's bytes (84 MB of them: 21.4 us, 3.9 TB/s, out of the last-level
// cache; 26.0 out of memory).
// ------------------------------------------------------------------------------------------------------------------------
struct SnapLds { int second, image; };          // the inputs of layers 0, 2 lie in the first LDS buffer, those of 1, 3 in the second; behind them the image, where it is staged

template <int BITS, int R, int NT>
struct SnapShape {
  static_assert(BITS == 4 || R != 4, "four rows: 4 bits only");
  static constexpr int T = R * NT;                               // rows of a tile (NT > 1: R = 16)
  static constexpr int P = BITS == 4 && R == 16 ? 3 : 1;         // products a step
  static constexpr int COLS = R > 1 ? 16 : BITS == 4 ? 4 : 1;
  static constexpr int QS = COLS * 16, TS = 4 * QS, XS = P * NT * TS;   // bytes from quarter to quarter, from tile of 16 rows (or part) to the next, from step to step
  // part p of input k of row t
  __device__ static __forceinline__ int at(int t, int p, int k) {
    if (BITS == 4) return (k >> 5) * XS + (k >> 3 & 3) * QS + (k & 7) * 2 + (R == 16 ? (p * NT + (t >> 4)) * TS + (t & 15) * 16 : (4 * t + p) * 16);
    return (k >> 4) * XS + (k >> 2 & 3) * QS + (k & 3) * 4 + (t >> 4) * TS + (t & 15) * 16;
  }
  static int bytes(const SnapDesc &nd, SnapLds &m) {
    int a = 0, b = 0;
    for (int l = 0; l < nd.L; ++l) { int &w = l & 1 ? b : a; w = nd.lay[l].steps * XS > w ? nd.lay[l].steps * XS : w; }
    m.second = a;
    return m.image = a + b;
  }
};

__device__ __forceinline__ unsigned short bf_top(float x) { return (unsigned short)(__float_as_uint(x) >> 16); }
// x = p[0] + p[1] + p[2] exactly (down to 2^-133), p[j] the upper half of the word v[j]; an infinity or NaN is all in v[0]
__device__ __forceinline__ void split3(float x, float (&v)[3]) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const float r1 = fabsf(x) < __uint_as_float(0x7f800000u) ? x - hi : 0.f;
  v[0] = x; v[1] = r1;
  v[2] = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
}
// what the upper halves leave
__device__ __forceinline__ f32x4 rest4(f32x4 x) {
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = x[j] - __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u);
  return r;
}
__device__ __forceinline__ unsigned two_tops(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }

// The waves that answer a tile together: a whole workgroup, or one of several equal parts of it
struct Team { int tid, threads, wave, waves; };
__device__ __forceinline__ Team whole_team() { return {(int)threadIdx.x, (int)blockDim.x, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), (int)(blockDim.x >> 6)}; }

// `rows(t)`: where row t of the tile lies, or null; `some`: any address that can be read, so that every load is unconditional and
// BATCH are on their way at once.  All threads of the team, no barrier inside.
template <int BITS, int R, int NT, int BATCH, class Rows>
__device__ __forceinline__ void tile_in(const Team &w, int K, char *buf, const float *some, Rows rows) {
  using S = SnapShape<BITS, R, NT>;
  const int Kp = BITS == 4 ? (K + 31) & ~31 : (K + 15) & ~15;
  const int per = Kp <= 32 ? 32 : 64;                      // threads a row
  const int t0 = w.tid / per, dt = w.threads / per;
#pragma unroll 1
  for (int k = w.tid & (per - 1); k < Kp; k += per)
#pragma unroll 1
    for (int t1 = t0; t1 < S::T; t1 += BATCH * dt) {
      float v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int t = t1 + i * dt;
        const float *x = t < S::T ? rows(t) : nullptr;
        const bool ok = x && k < K;
        v[i] = *(ok ? x + k : some);
        v[i] = ok ? v[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int t = t1 + i * dt;
        if (t >= S::T) break;
        if (BITS == 4) {
          const float z = v[i] != v[i] ? __uint_as_float(0x7fc00000u) : v[i];     // (a NaN that its upper half alone would not show)
          float p[3];
          split3(z, p);
#pragma unroll
          for (int j = 0; j < 3; ++j) *(unsigned short *)(buf + S::at(t, j, k)) = bf_top(p[j]);
        } else *(float *)(buf + S::at(t, 0, k)) = v[i];
      }
    }
}

// The barrier between layers: LDS is handed over, the weights already asked for stay in flight across it
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// the value of lane L of the own quad
template <int L>
__device__ __forceinline__ float quad_lane(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), L * 0x55, 0xf, 0xf, true)); }

// What a wave works on: strips s .. s + MT - 1 of layer l; where their records start in the image (of a strip that the layer does
// not have: the last one's)
struct Item { LayerOf y; int l, s; };
template <int MT>
__device__ __forceinline__ bool next_item(Item &it, DescP nd, int wave, int waves) {
  it.s += waves * MT;
  while (it.s >= it.y.strips) {
    if (++it.l >= nd->L) return false;
    it.y = layer_of(nd, it.l);
    it.s = wave * MT;
  }
  return true;
}
template <int MT>
__device__ __forceinline__ void records(unsigned (&rec)[MT], const LayerOf &y, int s) {
#pragma unroll
  for (int i = 0; i < MT; ++i) rec[i] = y.off + (unsigned)min(s + i, y.strips - 1) * y.rec;
}

// Four k-steps of MT strips, asked for together.  32 bits: those beyond the layer's last step are whatever follows in the image.
template <int BITS, int MT> struct SnapBlock {
  using W = std::conditional_t<BITS == 4, u32x4, f32x4[4]>;
  W w[MT];
  unsigned sc[MT];
  template <bool LDS>
  __device__ __forceinline__ void load(const char *img, const unsigned (&rec)[MT], const LayerOf &y, int b, unsigned lane) {
    const bool whole = 4 * b + 4 <= y.steps;
    const unsigned mine = whole ? lane * 16 : lane * (4 * (y.steps & 3));
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (BITS == 4) {
        const char *from = img + (rec[i] + b * 1024u);
        if (LDS && whole) w[i] = *(const u32x4 *)(from + mine);
        else w[i] = *(const u32x4u *)(from + mine);
        sc[i] = *(const unsigned *)(img + (rec[i] + y.code + b * 64u) + (lane & 15) * 4);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = *(const f32x4 *)(img + (rec[i] + b * 4096u) + lane * 16 + j * 1024);
      }
    }
  }
  // Waits for the block HERE.  Left to itself the compiler waits where it is multiplied, after the next one's loads have gone
  // out under a condition it cannot count through: it would wait for those too.
  __device__ __forceinline__ void here() {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (BITS == 4) { asm volatile("" : "+v"(w[i])); asm volatile("" : "+v"(sc[i])); }
      else { _Pragma("unroll") for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(w[i][j])); }
    }
  }
};

// Step j of a block.  `x`: the block's inputs of this lane's column
template <int BITS, int R, int NT, int MT>
__device__ __forceinline__ void step_multiply(const SnapBlock<BITS, MT> &w, int j, f32x4 (&acc)[MT][NT], const char *x) {
  using S = SnapShape<BITS, R, NT>;
  if constexpr (BITS == 4) {
    bf16x8 v[NT][S::P];
#pragma unroll
    for (int p = S::P - 1; p >= 0; --p)
#pragma unroll
      for (int t = 0; t < NT; ++t) v[t][p] = *(const bf16x8 *)(x + j * S::XS + (p * NT + t) * S::TS);
    union { bf16x2 h[4]; bf16x8 v; } a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float scale = __uint_as_float((w.sc[i] >> (8 * j) & 255u) << 23);
      a[i].h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.w[i][j], scale, 0);
      a[i].h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.w[i][j], scale, 1);
      a[i].h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.w[i][j], scale, 2);
      a[i].h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w.w[i][j], scale, 3);
    }
#pragma unroll
    for (int p = S::P - 1; p >= 0; --p)             // the small parts first; products of one sum apart from each other
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i].v, v[t][p], acc[i][t], 0, 0, 0);
  } else if constexpr (R == 1) {
    const f32x4 v = *(const f32x4 *)(x + j * S::XS);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][0][k] = fmaf(w.w[i][j][k], v[k], acc[i][0][k]);
  } else {
    f32x4 v[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) v[t] = *(const f32x4 *)(x + j * S::XS + t * S::TS);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w.w[i][j][k], v[t][k], acc[i][t], 0, 0, 0);
  }
}

// The biases a lane needs.  R = 16: of its 4 outputs of every strip; R = 4: of the one of every strip; R = 1: of its one.
template <int BITS, int R, int MT> struct SnapBias {
  f32x4 v4[R == 16 ? MT : 1];
  float v1[R == 4 ? MT : 1];
  __device__ __forceinline__ void load(const char *img, const unsigned (&rec)[MT], const LayerOf &y, unsigned c, unsigned q) {
    const unsigned b = y.rec - 64;
    if constexpr (R == 16) { _Pragma("unroll") for (int i = 0; i < MT; ++i) v4[i] = *(const f32x4 *)(img + (rec[i] + b) + q * 16); }
    else if constexpr (R == 4) { _Pragma("unroll") for (int i = 0; i < MT; ++i) v1[i] = *(const float *)(img + (rec[i] + b) + (4 * q + (c & 3)) * 4); }
    else {
      const unsigned own = BITS == 4 ? (c >> 2) & (MT - 1) : q & (MT - 1), at = BITS == 4 ? 4 * q + (c & 3) : c;
      unsigned from = rec[0];
      _Pragma("unroll") for (int i = 1; i < MT; ++i) from = own == i ? rec[i] : from;
      v1[0] = *(const float *)(img + (from + b + at * 4));
    }
  }
  __device__ __forceinline__ void here() {
    if constexpr (R == 16) { _Pragma("unroll") for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(v4[i])); }
    else { _Pragma("unroll") for (int i = 0; i < (R == 4 ? MT : 1); ++i) asm volatile("" : "+v"(v1[i])); }
  }
};
// What is asked for before the inputs are there: the first block of a wave's first strips
template <int BITS, int R, int MT> struct SnapAhead { Item it; SnapBlock<BITS, MT> w; SnapBias<BITS, R, MT> bias; };
template <int BITS, int R, int MT>
__device__ __forceinline__ void ahead_load(SnapAhead<BITS, R, MT> &h, const char *img, unsigned lane) {
  unsigned rec[MT];
  records<MT>(rec, h.it.y, h.it.s);
  h.bias.load(img, rec, h.it.y, lane & 15, lane >> 4);
  h.w.template load<false>(img, rec, h.it.y, 0, lane);
}
template <int BITS, int R, int MT>
__device__ __forceinline__ void ahead_first(const Team &w, SnapAhead<BITS, R, MT> &h, DescP nd, const char *img) {
  h.it.y = layer_of(nd, 0); h.it.l = 0; h.it.s = (w.wave - w.waves) * MT;
  if (next_item<MT>(h.it, nd, w.wave, w.waves)) ahead_load(h, img, threadIdx.x & 63);
}

// All layers.  The inputs are in LDS, behind a barrier; `img`: the net's image, in memory (AHEAD: `h` comes from
// ahead_first, and whatever is next, of the next layer too, is on its way while something is multiplied) or in LDS.  Ends with a
// barrier.
template <int BITS, int R, int NT, int MT, bool AHEAD, class Out>
__device__ __forceinline__ void net_layers(const Team &w, SnapAhead<BITS, R, MT> &h, DescP nd, const SnapLds &m, const char *img, char *lds, Out out) {
  using S = SnapShape<BITS, R, NT>;
  const int lane = threadIdx.x & 63, wave = w.wave, waves = w.waves, c = lane & 15, q = lane >> 4;
  const int col = R == 16 ? c : BITS == 32 ? 0 : (R == 4 ? c & 12 : 0) + min(c & 3, 2);
  // of the strip's outputs, this lane's (R = 16: its first): where it lies as an input of the next layer
  const int at = R == 16 ? 4 * q : BITS == 4 ? 4 * q + (c & 3) : c;
  const int put = R == 16 ? (BITS == 4 ? (q >> 1) * S::QS + (q & 1) * 8 : q * S::QS) + c * 16
                  : BITS == 4 ? (at >> 3) * S::QS + (R == 4 ? c & 12 : 0) * 16 + (at & 7) * 2 : at * 4;
  LayerOf coming = layer_of(nd, 0);
  asm volatile("" : "+s"(coming.steps));                       // (here: a wait inside the loop would be one for the next layer's too)
#pragma unroll 1
  for (int l = 0; l < nd->L; ++l) {
    const LayerOf y = coming;
    coming = layer_of(nd, min(l + 1, SNAP_MAXL - 1));
    const char *xin = lds + (l & 1 ? m.second : 0) + (q * S::QS + col * 16);
    char *xout = lds + (l & 1 ? 0 : m.second) + put;
    const bool last = l == nd->L - 1;
    const int blocks = (y.steps + 3) >> 2;
#pragma unroll 1
    for (int s = wave * MT; s < y.strips; s += waves * MT) {
      f32x4 acc[MT][NT];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      unsigned rec[MT];
      records<MT>(rec, y, s);
      SnapBias<BITS, R, MT> bias;
      if (AHEAD) { h.bias.here(); bias = h.bias; }
      else bias.load(img, rec, y, c, q);
      const char *x = xin;
#pragma unroll 1
      for (int b = 0; b < blocks; ++b) {
        SnapBlock<BITS, MT> next;
        if (AHEAD) {
          h.w.here();
          if (b + 1 < blocks) next.template load<false>(img, rec, y, b + 1, lane);
        } else h.w.template load<true>(img, rec, y, b, lane);
        const int now = y.steps - 4 * b;
        if (now >= 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) step_multiply<BITS, R, NT, MT>(h.w, j, acc, x);
        } else {
#pragma unroll
          for (int j = 0; j < 3; ++j)
            if (j == 0 || j < now) step_multiply<BITS, R, NT, MT>(h.w, j, acc, x);
        }
        x += 4 * S::XS;
        if (AHEAD) h.w = next;
      }
      if (AHEAD && next_item<MT>(h.it, nd, wave, waves)) ahead_load(h, img, lane);
      const bool odd = BITS == 4 && (y.strips & 1);            // the next layer's k-steps are 32 wide: zeros behind an odd last strip
      if constexpr (R < 16) {
        const int own = R > 1 ? 0 : BITS == 4 ? (c >> 2) & (MT - 1) : q & (MT - 1);
#pragma unroll
        for (int i = 0; i < (R == 1 ? 1 : MT); ++i) {
          float v;
          int strip = s + i;
          if constexpr (R == 1 && BITS == 32) {                // the lanes (c, 0..3) hold parts of output c of every strip
            float sum[MT];
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              const f32x4 p = acc[k][0];
              sum[k] = (p[0] + p[1]) + (p[2] + p[3]);
              sum[k] += __shfl_xor(sum[k], 16); sum[k] += __shfl_xor(sum[k], 32);
            }
            v = sum[0];
#pragma unroll
            for (int k = 1; k < MT; ++k) v = own == k ? sum[k] : v;
            strip = s + own;
          } else {
            f32x4 p = acc[R == 1 ? 0 : i][0];
            if constexpr (R == 1) {
#pragma unroll
              for (int k = 1; k < MT; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = own == k ? acc[k][0][j] : p[j];
              strip = s + own;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = quad_lane<0>((quad_lane<2>(p[j]) + quad_lane<1>(p[j])) + p[j]);   // the parts lie in the lanes of a quad: smallest first
            const int j = c & 3;
            v = j & 1 ? p[1] : p[0];
            const float v2 = j & 1 ? p[3] : p[2];
            v = j & 2 ? v2 : v;
          }
          const int n = strip * 16 + at, t = R == 4 ? c >> 2 : 0;
          v = act_one(y.act, v + bias.v1[i]);
          v = n < y.out ? v : 0.f;
          const bool mine = strip < y.strips && (R == 4 || (BITS == 4 ? c < 4 * MT : q < MT));
          if (mine) {
            if (last) { if (n < y.out) out(t, n, v); }
            else if constexpr (BITS == 4) {
              float p[3];
              split3(v, p);
              char *o = xout + strip * (2 * S::QS);
#pragma unroll
              for (int k = 0; k < 3; ++k) {
                *(unsigned short *)(o + k * 16) = bf_top(p[k]);
                if (odd && strip == y.strips - 1) *(unsigned short *)(o + 2 * S::QS + k * 16) = 0;
              }
            } else *(float *)(xout + strip * S::XS) = v;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
          if (s + i < y.strips) {
            const int strip = s + i, n0 = strip * 16 + 4 * q;
            const bool end = strip == y.strips - 1;
            char *o = xout + (BITS == 4 ? (strip >> 1) * S::XS + (strip & 1) * (2 * S::QS) : strip * S::XS);
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
              const int t = 16 * tt + c;
              f32x4 a = act_four(y.act, acc[i][tt] + bias.v4[i]);
              if (end) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = n0 + j < y.out ? a[j] : 0.f;
              }
              if (last) {
#pragma unroll
                for (int j = 0; j < 4; ++j) if (n0 + j < y.out) out(t, n0 + j, a[j]);
              } else if constexpr (BITS == 4) {
                f32x4 r = rest4(a);                          // NaN where a is not finite: rare enough to look for once
                const float odd_one = __builtin_elementwise_maximum(__builtin_elementwise_maximum(r[0], r[1]), __builtin_elementwise_maximum(r[2], r[3]));
                if (__any(odd_one != odd_one)) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) r[j] = r[j] != r[j] ? 0.f : r[j];
                }
                const f32x4 lo = rest4(r);
                *(u32x2 *)(o + tt * S::TS) = u32x2{two_tops(a[0], a[1]), two_tops(a[2], a[3])};
                *(u32x2 *)(o + (NT + tt) * S::TS) = u32x2{two_tops(r[0], r[1]), two_tops(r[2], r[3])};
                *(u32x2 *)(o + (2 * NT + tt) * S::TS) = u32x2{two_tops(lo[0], lo[1]), two_tops(lo[2], lo[3])};
                if (odd && end) {
#pragma unroll
                  for (int k = 0; k < 3; ++k) *(u32x2 *)(o + (k * NT + tt) * S::TS + 2 * S::QS) = u32x2{0u, 0u};
                }
              } else *(f32x4 *)(o + tt * S::TS) = a;
            }
          }
      }
    }
    lds_barrier();
  }
}

// A net's image from memory to LDS, without a register in between: everything is asked for at once.  The caller waits.
__device__ __forceinline__ void image_in(const Team &w, const char *img, char *lds, unsigned bytes) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (unsigned i = w.wave * 1024; i < bytes; i += w.waves * 1024)
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(img + i + lane * 16),
                                     (__attribute__((address_space(3))) void *)(lds + i), 16, 0, 0);
}
__device__ __forceinline__ void image_here() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// How a workgroup comes by its net: straight from memory as it goes, or all of it staged in LDS.  net_ask before the inputs are
// brought in, net_tile after them.
template <int BITS, int R, int NT, int MT, bool STAGED> struct SnapNet {
  SnapAhead<BITS, R, MT> h;
  const char *img;
  Team w;
  __device__ __forceinline__ SnapNet(const Team &team) : w(team) {}
  __device__ __forceinline__ void stage(DescP nd, const SnapLds &m, const char *image, char *lds) {      // once for a net
    img = image;
    if (STAGED) image_in(w, image, lds + m.image, nd->stride);
  }
  __device__ __forceinline__ void ask(DescP nd) { if (!STAGED) ahead_first(w, h, nd, img); }     // for a tile
  template <class Out>
  __device__ __forceinline__ void tile(DescP nd, const SnapLds &m, char *lds, Out out) {
    if (STAGED) image_here();
    lds_barrier();
    net_layers<BITS, R, NT, MT, !STAGED>(w, h, nd, m, STAGED ? lds + m.image : img, lds, out);
  }
};

// ------------------------------------------------------------------------------------------------------------------------
// Every agent's net on its rows
// ------------------------------------------------------------------------------------------------------------------------
template <int BITS, int R, int NT, int MT, bool STAGED>
__global__ void __launch_bounds__(R == 16 && !STAGED ? 1024 : 512, BITS == 4 && R == 16 && !STAGED ? 6 : 1)     // (6 waves a SIMD: see forward_run)
snap_forward_kernel(const SnapDesc nd_, const SnapLds m, const SnapForward p) {
  extern __shared__ __align__(16) char lds[];
  using S = SnapShape<BITS, R, NT>;
  const DescP nd = SNAP_DESC(nd_);
  const int g = blockIdx.x;
  if (p.mask && !p.mask[g]) return;
  SnapNet<BITS, R, NT, MT, STAGED> net(whole_team());
  net.stage(nd, m, p.img + (size_t)g * nd->stride, lds);
  const int from = blockIdx.y * p.per, to = min(p.n, from + p.per);
#pragma unroll 1
  for (int t0 = from; t0 < to; t0 += S::T) {
    net.ask(nd);
    const float *x = p.x + g * p.x_agent + t0 * p.x_row;
    tile_in<BITS, R, NT, (R > 1 && STAGED ? 2 : 1)>(net.w, nd->lay[0].in, lds, p.x, [&](int t) { return t0 + t < to ? x + t * p.x_row : (const float *)nullptr; });
    float *o = p.out + g * p.out_agent + t0 * p.out_row;
    net.tile(nd, m, lds, [&](int t, int n, float v) { if (t0 + t < to) o[t * p.out_row + n] = v; });
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// The router.  One workgroup per 16 rows; a wave takes strips of 16 agents: logits[16 agents x 16 rows] on
// v_mfma_f64_16x16x4_f64.  Both factors are 32-bit numbers, so their products are exact and the sums are wrong by ~1e-16: two
// logits change places only where they are equal to 15 digits.  A lane holds 4 logits of one row a strip and keeps the KM best
// it has met, as keys that sort as the numbers do (NaN above all, a barred one as -infinity); the lanes of a row, then the waves, merge their
// lists.  The index decides between equal keys.  Bound by latency: one strip a wave, then the lists (256 agents, 4096 rows of 45: 9.4
// us, 10 TFLOP/s).
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

// The best of 16 lanes' (key, index), in all of them.  quad_perm and the mirrors reach every lane of a row of 16.
template <int CTRL>
__device__ __forceinline__ void best_dpp(unsigned long long &k, int &i) {
  const int hi = (int)(k >> 32), lo = (int)k;
  const unsigned oh = (unsigned)__builtin_amdgcn_update_dpp(0, hi, CTRL, 0xf, 0xf, true), ol = (unsigned)__builtin_amdgcn_update_dpp(0, lo, CTRL, 0xf, 0xf, true);
  const int oi = __builtin_amdgcn_update_dpp(0, i, CTRL, 0xf, 0xf, true);
  const unsigned long long ok = (unsigned long long)oh << 32 | ol;
  if (key_before(ok, oi, k, i)) { k = ok; i = oi; }
}
__device__ __forceinline__ void best_of_16(unsigned long long &k, int &i) {
  best_dpp<0xB1>(k, i); best_dpp<0x4E>(k, i); best_dpp<0x141>(k, i); best_dpp<0x140>(k, i);
}
// Between the rows of 16: v_permlane16_swap(a, b) is {a's even rows, b's even rows in the odd places} and the same of the odd ones,
// v_permlane32_swap the halves likewise
struct Two { unsigned x, y; };
template <bool HALVES>
__device__ __forceinline__ Two swap_rows(unsigned a, unsigned b) {
  const auto v = HALVES ? __builtin_amdgcn_permlane32_swap(a, b, false, false) : __builtin_amdgcn_permlane16_swap(a, b, false, false);
  return {v[0], v[1]};
}
template <bool HALVES>
__device__ __forceinline__ void best_swap(unsigned long long &k, int &i) {
  const Two h = swap_rows<HALVES>((unsigned)(k >> 32), (unsigned)(k >> 32)), l = swap_rows<HALVES>((unsigned)k, (unsigned)k), n = swap_rows<HALVES>((unsigned)i, (unsigned)i);
  const unsigned long long ka = (unsigned long long)h.x << 32 | l.x, kb = (unsigned long long)h.y << 32 | l.y;
  const bool a = key_before(ka, (int)n.x, kb, (int)n.y);
  k = a ? ka : kb; i = (int)(a ? n.x : n.y);
}
// the sums over the two rows (halves) of a in the even ones, of b in the odd ones
template <bool HALVES>
__device__ __forceinline__ double sum_swap(double a, double b) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(a), v = (unsigned long long)__double_as_longlong(b);
  const Two h = swap_rows<HALVES>((unsigned)(u >> 32), (unsigned)(v >> 32)), l = swap_rows<HALVES>((unsigned)u, (unsigned)v);
  return __longlong_as_double((long long)((unsigned long long)h.x << 32 | l.x)) + __longlong_as_double((long long)((unsigned long long)h.y << 32 | l.y));
}
template <int CTRL>
__device__ __forceinline__ unsigned long long most_dpp(unsigned long long k) {
  const unsigned long long o = (unsigned long long)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(k >> 32), CTRL, 0xf, 0xf, true) << 32 |
                               (unsigned)__builtin_amdgcn_update_dpp(0, (int)k, CTRL, 0xf, 0xf, true);
  return o > k ? o : k;
}
template <bool HALVES>
__device__ __forceinline__ unsigned long long most_swap(unsigned long long k) {
  const Two h = swap_rows<HALVES>((unsigned)(k >> 32), (unsigned)(k >> 32)), l = swap_rows<HALVES>((unsigned)k, (unsigned)k);
  const unsigned long long ka = (unsigned long long)h.x << 32 | l.x, kb = (unsigned long long)h.y << 32 | l.y;
  return ka > kb ? ka : kb;
}
// the largest of 64, as a scalar
__device__ __forceinline__ unsigned long long most_of_64(unsigned long long k) {
  k = most_dpp<0x140>(most_dpp<0x141>(most_dpp<0x4E>(most_dpp<0xB1>(k))));
  k = most_swap<true>(most_swap<false>(k));
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(k >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)k);
}
#define IDX_NONE 0x7fffffff
// the first of a row of 16's, in all of them
__device__ __forceinline__ int first_of_16(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x150, 0xf, 0xf, true); }
__device__ __forceinline__ float sum_of_16(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));
  return v;
}

// A lane's KM best, sorted
template <int KM> struct Best {
  unsigned long long K[KM];
  int I[KM];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < KM; ++j) { K[j] = KEY_NONE; I[j] = IDX_NONE; }
  }
  __device__ __forceinline__ void insert(unsigned long long key, int e) {     // (after all of a lower index)
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
  __device__ __forceinline__ void pop(int i) {                                 // if i is the first
    if (I[0] == i) {
#pragma unroll
      for (int j = 0; j + 1 < KM; ++j) { K[j] = K[j + 1]; I[j] = I[j + 1]; }
      K[KM - 1] = KEY_NONE; I[KM - 1] = IDX_NONE;
    }
  }
  // a list that lies in memory
  template <class Key, class Idx> __device__ __forceinline__ void read(int k, Key key, Idx idx) {
#pragma unroll
    for (int j = 0; j < KM; ++j) if (j < k) { K[j] = key(j); I[j] = idx(j); }
  }
  // the k best of 16 lanes' lists: lane j keeps the j-th
  __device__ __forceinline__ void merge_16(int lane, int k, unsigned long long &mk, int &mi) {
    mk = KEY_NONE; mi = IDX_NONE;
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
      unsigned long long bk = K[0];
      int bi = I[0];
      best_of_16(bk, bi);
      pop(bi);
      if (lane == j) { mk = bk; mi = bi; }
    }
  }
  // of 64: the largest key, then who has it, the lowest index among several (several: rare)
  __device__ __forceinline__ void merge_64(int lane, int k, unsigned long long &mk, int &mi) {
    mk = KEY_NONE; mi = IDX_NONE;
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
      const unsigned long long bk = most_of_64(K[0]);
      if (bk == KEY_NONE) break;
      int bi = IDX_NONE;
      for (unsigned long long who = __ballot(K[0] == bk); who; who &= who - 1) bi = min(bi, __builtin_amdgcn_readlane(I[0], __ffsll(who) - 1));
      pop(bi);
      if (lane == j) { mk = bk; mi = bi; }
    }
  }
};
// The softmax over the picks that 16 lanes hold.  The logits' differences are taken in fp64 and rounded once: from there on a 32-bit
// number comes out and weighs 32-bit answers, and what the rounding, expf, the sum and the division add, (|difference| + 14) 2^-24
// of it at most, is of the size of what the answers are off by themselves.
__device__ __forceinline__ float pick_prob(unsigned long long mk, int mi) {
  const unsigned long long tk = (unsigned long long)(unsigned)first_of_16((int)(mk >> 32)) << 32 | (unsigned)first_of_16((int)mk);
  const float ex = mi != IDX_NONE ? expf((float)(key_logit(mk) - key_logit(tk))) : 0.f;
  const float sum = sum_of_16(ex);
  return mi != IDX_NONE ? ex / sum : 0.f;
}

// grid (rows / 16, chunks): the rows' best among the chunk's agents; with one chunk the picks themselves
template <int KM>
__global__ void __launch_bounds__(1024)
snap_router_kernel(const SnapMixture p, int S, int A, int ld) {
  extern __shared__ __align__(16) char lds[];
  float *xs = (float *)lds;                                // [16][ld]
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  unsigned long long *ck = (unsigned long long *)(lds + 16 * ld * 4);       // [16][waves][KM]
  int *ci = (int *)(ck + 16 * waves * KM);
  const int t0 = blockIdx.x * 16;
  const int strips = (p.G + 15) >> 4, each = (strips + p.chunks - 1) / p.chunks, s_from = blockIdx.y * each, s_to = min(strips, s_from + each);
  const int Sp = (S + 15) & ~15;
  for (int t = threadIdx.x >> 5; t < 16; t += blockDim.x >> 5)
    for (int k = threadIdx.x & 31; k < Sp; k += 32) xs[t * ld + k] = t0 + t < p.n && k < S ? p.x[(t0 + t) * p.x_row + k] : 0.f;
  Best<KM> best;
  best.clear();
  const int row = min(t0 + c, p.n - 1);
  const uint8_t *al = p.allowed ? p.allowed + row * p.a_row : nullptr;
  bool first = true;
  for (int s = s_from + wave; s < s_to; s += waves) {
    const float *w = p.rw + (int64_t)min(s * 16 + c, p.G - 1) * p.r_row;
    float bias[4];
    bool ok[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = min(s * 16 + 4 * j + q, p.G - 1);
      bias[j] = p.rb ? p.rb[e] : 0.f;
      ok[j] = (!al || al[e]) && s * 16 + 4 * j + q < p.G;
    }
    f64x4 acc = {0., 0., 0., 0.};
    constexpr int U = KM > 4 ? 2 : 4;                       // 16 inputs each, asked for together
    for (int k0 = 0; k0 < S; k0 += 16 * U) {
      float a[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = k0 + 16 * u + 4 * q;
        if (k0 + 16 * u + 16 <= S) {
          const f32x4u v = *(const f32x4u *)(w + at);
          a[u][0] = v[0]; a[u][1] = v[1]; a[u][2] = v[2]; a[u][3] = v[3];
        } else if (k0 + 16 * u < S) {                       // the row's end: no lane reads beyond it
#pragma unroll
          for (int j = 0; j < 4; ++j) { const float v = w[min(at + j, S - 1)]; a[u][j] = at + j < S ? v : 0.f; }
        }
      }
      if (first) { __syncthreads(); first = false; }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + 16 * u < S) {
          const f32x4 x = *(const f32x4 *)(xs + c * ld + k0 + 16 * u + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[u][j], (double)x[j], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      best.insert(ok[j] ? logit_key(acc[j] + (double)bias[j]) : KEY_NONE, s * 16 + 4 * j + q);
    }
  }
  if (first) __syncthreads();
  // the four lanes of a row
  for (int j = 0; j < p.k; ++j) {
    unsigned long long bk = best.K[0];
    int bi = best.I[0];
    best_swap<false>(bk, bi); best_swap<true>(bk, bi);
    best.pop(bi);
    if (q == 0) { ck[(c * waves + wave) * KM + j] = bk; ci[(c * waves + wave) * KM + j] = bi; }
  }
  __syncthreads();
  // the waves: 16 lanes a row
  const int u = threadIdx.x & 15;
  for (int t = threadIdx.x >> 4; t < 16; t += blockDim.x >> 4) {
    const int tok = t0 + t;
    const bool live = tok < p.n;
    unsigned long long mk;
    int mi;
    best.clear();
    if (u < waves) best.read(p.k, [&](int j) { return ck[(t * waves + u) * KM + j]; }, [&](int j) { return ci[(t * waves + u) * KM + j]; });
    best.merge_16(u, p.k, mk, mi);
    if (live && u == 0 && blockIdx.y == 0) p.count[tok] = 0;
    if (p.chunks > 1) {                                    // the chunk's list, sorted
      if (live && u < p.k) {
        p.ckey[((int64_t)tok * p.chunks + blockIdx.y) * p.k + u] = mk;
        p.cidx[((int64_t)tok * p.chunks + blockIdx.y) * p.k + u] = mi;
      }
      continue;
    }
    const float mp = pick_prob(mk, mi);
    const bool have = mi != IDX_NONE;
    if (live && u < p.k) {
      p.idx[(int64_t)tok * p.k + u] = have ? mi : -1;
      p.prob[(int64_t)tok * p.k + u] = mp;
      if (!have) for (int a = 0; a < A; ++a) p.y[((int64_t)tok * p.k + u) * A + a] = 0.f;
    }
    if (live && first_of_16(mi) == IDX_NONE) for (int a = u; a < A; a += 16) p.out[tok * p.out_row + a] = 0.f;
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// A row's picks, for a workgroup of its own: out of the router's lists, or read.  All threads; ends with a barrier.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void row_picks(const SnapMixture &p, int row, int *picks, float *probs) {
  const int tid = threadIdx.x;
  if (p.chunks > 1) {
    if (tid < 16) {
      unsigned long long mk;
      int mi;
      const int64_t at = ((int64_t)row * p.chunks + tid) * p.k;
      Best<SNAP_MAXK> best;
      best.clear();
      if (tid < p.chunks) best.read(p.k, [&](int j) { return p.ckey[at + j]; }, [&](int j) { return p.cidx[at + j]; });
      best.merge_16(tid, p.k, mk, mi);
      const float mp = pick_prob(mk, mi);
      if (tid < p.k) { picks[tid] = mi == IDX_NONE ? -1 : mi; probs[tid] = mp; }
    }
  } else if (tid < p.k) { picks[tid] = p.idx[row * p.k + tid]; probs[tid] = p.prob[row * p.k + tid]; }
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------------------------------
// Few rows, nets that fit in LDS together: a workgroup a row, a team of its waves for each pick, so that the answers meet in LDS.
// And as long as the router's matrix is small, every workgroup works the router out for its row by itself (KM > 0), a thread an
// agent at a time, sums in fp64 as above: one launch, nothing to hand over.  Bound by the latency of what follows on what: the
// router's rows, the picks, the nets' images, the layers (16 agents of 18-100-100-6 in 32 bits, one row, top 2: 8.5 us; router and
// nets in two launches: 11.9.  1024 in 4 bits, 8 rows, top 4: 14.2 and 18.7).
// ------------------------------------------------------------------------------------------------------------------------
// inputs at .. at + 3 of a router row of S, zeros behind its end; no lane reads beyond it
__device__ __forceinline__ f32x4 row_four(const float *w, int at, int S) {
  if (S < 4) return f32x4{at < S ? w[min(at, S - 1)] : 0.f, at + 1 < S ? w[min(at + 1, S - 1)] : 0.f, at + 2 < S ? w[min(at + 2, S - 1)] : 0.f, 0.f};
  const f32x4 v = *(const f32x4u *)(w + min(at, S - 4));
  const int d = at - (S - 4);
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = d <= 0 ? v[j] : 0.f;
#pragma unroll
    for (int i = 1; j + i < 4; ++i) r[j] = d == i ? v[j + i] : r[j];
  }
  return r;
}
// xs: the row's inputs, zeros behind them up to a multiple of 16.  A wave takes 64 agents at a time, as 4 times 16 whose rows are
// read by 4 lanes each, 16 bytes a lane (a lane an agent would touch 64 lines with every read).
template <int KM>
__device__ __forceinline__ void route_row(const SnapMixture &p, int S, int row, const float *xs, char *lists, int *picks, float *probs) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6, c = lane & 15, q = lane >> 4;
  unsigned long long *ck = (unsigned long long *)lists;     // [waves][KM]
  int *ci = (int *)(ck + waves * KM);
  Best<KM> best;
  best.clear();
  const uint8_t *al = p.allowed ? p.allowed + row * p.a_row : nullptr;
  bool first = true;
#pragma unroll 1
  for (int e0 = wave * 64; e0 < p.G || first; e0 += waves * 64) {
    const int e = min(e0 + lane, p.G - 1);
    const float bias = p.rb ? p.rb[e] : 0.f;
    const bool ok = e0 + lane < p.G && (!al || al[e]);
    const float *w[4];
    double acc[4] = {0., 0., 0., 0.};
#pragma unroll
    for (int m = 0; m < 4; ++m) w[m] = p.rw + (int64_t)min(e0 + 16 * m + c, p.G - 1) * p.r_row;
#pragma unroll 1
    for (int s0 = 0; s0 < S; s0 += 32) {
      f32x4 a[4][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = s0 + 16 * u + 4 * q;
        if (s0 + 16 * u + 16 <= S) {
#pragma unroll
          for (int m = 0; m < 4; ++m) a[m][u] = *(const f32x4u *)(w[m] + at);
        } else if (s0 + 16 * u < S) {
#pragma unroll
          for (int m = 0; m < 4; ++m) a[m][u] = row_four(w[m], at, S);
        }
      }
      if (first) { __syncthreads(); first = false; }        // (the inputs have come)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (s0 + 16 * u < S) {
          const f32x4 x = *(const f32x4 *)(xs + s0 + 16 * u + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int m = 0; m < 4; ++m) acc[m] = fma((double)a[m][u][j], (double)x[j], acc[m]);
        }
    }
    const double sum = sum_swap<false>(sum_swap<true>(acc[0], acc[2]), sum_swap<true>(acc[1], acc[3]));   // lane 16 m + c: agent e0 + 16 m + c's
    best.insert(ok ? logit_key(sum + (double)bias) : KEY_NONE, e);
  }
  unsigned long long mk;
  int mi;
  best.merge_64(lane, p.k, mk, mi);
  if (p.G > 64) {
    if (lane < p.k) { ck[wave * KM + lane] = mk; ci[wave * KM + lane] = mi; }
    __syncthreads();
    if (wave == 0) {
      best.clear();
      if (lane < waves) best.read(p.k, [&](int j) { return ck[lane * KM + j]; }, [&](int j) { return ci[lane * KM + j]; });
      best.merge_64(lane, p.k, mk, mi);
    }
  }
  if (wave == 0) {
    const float mp = pick_prob(mk, mi);
    if (lane < p.k) { picks[lane] = mi == IDX_NONE ? -1 : mi; probs[lane] = mp; }
  }
  __syncthreads();
}
// where what lies in the LDS of snap_row_kernel: the row's inputs, the waves' lists, the answers, a team's part
struct SnapRow { int lists, y, teams, team, waves; };

template <int BITS, int MT, int KM>
__global__ void __launch_bounds__(1024)
snap_row_kernel(const SnapDesc nd_, const SnapLds m, const SnapMixture p, const SnapRow at) {
  extern __shared__ __align__(16) char lds[];
  __shared__ int picks[SNAP_MAXK];
  __shared__ float probs[SNAP_MAXK];
  const DescP nd = SNAP_DESC(nd_);
  const int tid = threadIdx.x, A = nd->A, S = nd->lay[0].in, row = blockIdx.x;
  float *xs = (float *)lds, *y = (float *)(lds + at.y);
  const float *x = p.x + row * p.x_row;
  for (int s = tid; s < ((S + 15) & ~15); s += blockDim.x) xs[s] = s < S ? x[s] : 0.f;
  if (KM) route_row<KM ? KM : 1>(p, S, row, xs, lds + at.lists, picks, probs);
  else row_picks(p, row, picks, probs);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = wave / at.waves;
  const int e = j < p.k ? __builtin_amdgcn_readfirstlane(picks[j]) : -1;
  // (who has no net keeps the barriers only: no strip is its own)
  const Team w = {tid - j * at.waves * 64, at.waves * 64, e >= 0 ? wave - j * at.waves : SNAP_MAXW, at.waves};
  char *own = lds + at.teams + (e >= 0 ? j : 0) * at.team;
  SnapNet<BITS, 1, 1, MT, true> net(w);
  if (e >= 0) {
    net.stage(nd, m, p.img + (size_t)e * nd->stride, own);
    tile_in<BITS, 1, 1, 1>(w, S, own, xs, [&](int) { return xs; });
  }
  if (tid < p.k && (KM || p.chunks > 1)) { p.idx[row * p.k + tid] = picks[tid]; p.prob[row * p.k + tid] = probs[tid]; }
  net.tile(nd, m, own, [&](int, int n, float v) { y[j * A + n] = v; });
  for (int a = tid; a < A; a += blockDim.x) {
    float sum = 0.f;
    for (int i = 0; i < p.k; ++i) {
      const float v = picks[i] >= 0 ? y[i * A + a] : 0.f;
      p.y[((int64_t)row * p.k + i) * A + a] = v;
      sum = picks[i] >= 0 ? fmaf(probs[i], v, sum) : sum;
    }
    p.out[row * p.out_row + a] = sum;
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// Few places of larger nets: a workgroup for each.  Whoever answers a row's last place sums the row up, in the order of its places
// whatever the order they were answered in.  The answers are stored past the XCD's own cache (agent scope); once they have arrived
// the counter may tell of them.  Nothing else passes between workgroups, so no cache has to be written back or forgotten, and
// nobody waits.  Bound by what one CU has in flight from memory (66 places of 18-400-300-6 in 32 bits, 34 MB: 15 us, 13 waves each;
// with 8 waves 17 us).
// ------------------------------------------------------------------------------------------------------------------------
template <int BITS, int MT, bool STAGED>
__global__ void __launch_bounds__(STAGED ? 512 : 1024)
snap_place_kernel(const SnapDesc nd_, const SnapLds m, const SnapMixture p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ int picks[SNAP_MAXK], last;
  __shared__ float probs[SNAP_MAXK];
  const DescP nd = SNAP_DESC(nd_);
  const int tid = threadIdx.x, A = nd->A, row = blockIdx.x / p.k, place = blockIdx.x - row * p.k;
  row_picks(p, row, picks, probs);
  const int e = __builtin_amdgcn_readfirstlane(picks[place]);
  float *y = p.y + (int64_t)blockIdx.x * A;
  if (p.chunks > 1) {
    if (tid == 0) { p.idx[blockIdx.x] = e; p.prob[blockIdx.x] = probs[place]; }
    if (e < 0) {
      for (int a = tid; a < A; a += blockDim.x) y[a] = 0.f;
      if (picks[0] < 0 && place == 0) for (int a = tid; a < A; a += blockDim.x) p.out[row * p.out_row + a] = 0.f;
    }
  }
  if (e < 0) return;
  SnapNet<BITS, 1, 1, MT, STAGED> net(whole_team());
  net.stage(nd, m, p.img + (size_t)e * nd->stride, lds);
  net.ask(nd);
  const float *x = p.x + row * p.x_row;
  tile_in<BITS, 1, 1, 1>(net.w, nd->lay[0].in, lds, p.x, [&](int) { return x; });
  net.tile(nd, m, lds, [&](int, int n, float v) { __hip_atomic_store(y + n, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int want = 0;
    for (int j = 0; j < p.k; ++j) want += picks[j] >= 0;
    last = __hip_atomic_fetch_add(p.count + row, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == want - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int a = tid; a < A; a += blockDim.x) {
    float sum = 0.f;
    for (int j = 0; j < p.k; ++j)
      if (picks[j] >= 0) sum = fmaf(probs[j], __hip_atomic_load(p.y + ((int64_t)row * p.k + j) * A + a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), sum);
    p.out[row * p.out_row + a] = sum;
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// Who picked a net, when there are many places: every 1024 places of idx sorted by the net they picked, in their order.  Lanes of a
// wave with the same net find each other bit by bit; the waves take their turns at the nets' counters, so that a place's position
// does not hang on who came first.  Places that picked nobody go to net G.  Bound by the latency of a launch, a read and a write (4.7
// us for 8192 places, 5.0 for 32768; a counter a wave instead of turns: the same).
// ------------------------------------------------------------------------------------------------------------------------
#define SORT_BLOCK 1024
__device__ __forceinline__ void sort_block(const int *__restrict__ idx, int block, int total, int G, int bits, int *__restrict__ sorted, int *__restrict__ start, char *lds) {
  int *cnt = (int *)lds;                                   // [G + 1]
  __shared__ int wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = block * SORT_BLOCK + tid;
  int e = i < total ? idx[i] : G;
  for (int j = tid; j <= G; j += 1024) cnt[j] = 0;
  e = e < 0 || e >= G ? G : e;
  unsigned long long same = __ballot(i < total);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long m = __ballot((e >> b) & 1);
    same &= (e >> b) & 1 ? m : ~m;
  }
  const unsigned long long below = (1ull << lane) - 1ull;
  const int rank = __popcll(same & below), n = __popcll(same), lead = __ffsll(same) - 1;
  int base = 0;
  for (int w = 0; w < 16; ++w) {
    __syncthreads();
    if (w == wave && i < total && lane == lead) base = atomicAdd(&cnt[e], n);
  }
  __syncthreads();
  base = __shfl(base, lead < 0 ? 0 : lead) + rank;
  // exclusive sums of the counters: a thread `per` of them, then the waves, then the block
  const int per = (G + 1 + 1023) >> 10, e0 = tid * per;
  int own = 0;
  for (int j = 0; j < per; ++j) own += e0 + j <= G ? cnt[e0 + j] : 0;
  int before = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) { const int o = __shfl_up(before, d); before += lane >= d ? o : 0; }
  if (lane == 63) wsum[wave] = before;
  __syncthreads();
  before -= own;
  for (int w = 0; w < wave; ++w) before += wsum[w];
  __syncthreads();
  for (int j = 0; j < per; ++j)
    if (e0 + j <= G) { const int c = cnt[e0 + j]; cnt[e0 + j] = before; start[(int64_t)block * (G + 1) + e0 + j] = before; before += c; }
  __syncthreads();
  if (i < total) sorted[block * SORT_BLOCK + cnt[e] + base] = i;
}
extern "C" __global__ void __launch_bounds__(1024)
snap_sort_kernel(const int *__restrict__ idx, int total, int G, int bits, int *__restrict__ sorted, int *__restrict__ start) {
  extern __shared__ __align__(16) char lds[];
  sort_block(idx, blockIdx.x, total, G, bits, sorted, start, lds);
}
// The i-th place of net e in the blocks b0 .. b0 + nb - 1 (nb <= 64), each thread of a wave its own i; `have`: how many there are.
// Lane b holds block b0 + b's.
struct Places { int from, cnt; };
__device__ __forceinline__ Places places_of(const int *start, int G, int e, int b0, int nb, int lane) {
  Places g = {0, 0};
  if (lane < nb) {
    const int *st = start + (int64_t)(b0 + lane) * (G + 1) + e;
    g.cnt = st[1] - st[0];
    g.from = (b0 + lane) * SORT_BLOCK + st[0];
  }
  return g;
}
__device__ __forceinline__ int place_at(const Places &g, int nb, int i, int &have) {
  int at = -1;
  have = 0;
  for (int b = 0; b < nb; ++b) {
    const int n = __builtin_amdgcn_readlane(g.cnt, b), f = __builtin_amdgcn_readlane(g.from, b);
    at = i >= have && i < have + n ? f + i - have : at;
    have += n;
  }
  return at;
}

// ------------------------------------------------------------------------------------------------------------------------
// The picked nets, many places: a workgroup answers, for one net, every gridDim.y-th tile of T of the places that picked it; the
// rows are summed up as above.  Bound by what follows on what in a tile (its places, their inputs, the layers, the answers' way to
// memory and back), some 8 us: 256 agents of 45-64-64-17, 4096 rows, top 2, 32 bits 20.5 us.
// ------------------------------------------------------------------------------------------------------------------------
template <int BITS, int R, int NT, int MT>
__global__ void __launch_bounds__(512)
snap_experts_kernel(const SnapDesc nd_, const SnapLds m, const SnapMixture p) {
  extern __shared__ __align__(16) char lds[];
  using S = SnapShape<BITS, R, NT>;
  __shared__ int list[S::T], picked[S::T], done[S::T], have;
  __shared__ float probs[S::T][SNAP_MAXK];
  const DescP nd = SNAP_DESC(nd_);
  const int tid = threadIdx.x, A = nd->A, threads = blockDim.x, e = blockIdx.x;
  SnapNet<BITS, R, NT, MT, false> net(whole_team());
  net.stage(nd, m, p.img + (size_t)e * nd->stride, lds);
  for (int b0 = 0; b0 < p.blocks; b0 += 64) {
    const int nb = min(64, p.blocks - b0);
    const Places places = places_of(p.start, p.G, e, b0, nb, tid & 63);
    for (int i0 = blockIdx.y * S::T; ; i0 += gridDim.y * S::T) {
      if (net.w.wave == 0) {
        int sum;
        const int at = place_at(places, nb, i0 + tid, sum);
        if (tid < S::T) list[tid] = at >= 0 ? p.sorted[at] : -1;
        if (tid == 0) have = sum;
      }
      __syncthreads();
      if (i0 >= have) break;
      net.ask(nd);
      tile_in<BITS, R, NT, (R > 1 ? 4 : 1)>(net.w, nd->lay[0].in, lds, p.x, [&](int t) { return list[t] >= 0 ? p.x + (int64_t)(list[t] / p.k) * p.x_row : (const float *)nullptr; });
      for (int i = tid; i < S::T * SNAP_MAXK; i += threads) {          // (wanted at the end)
        const int t = i / SNAP_MAXK, j = i % SNAP_MAXK, r = list[t] / p.k;
        const bool has = list[t] >= 0 && j < p.k;
        probs[t][j] = has ? p.prob[r * p.k + j] : 0.f;
        const unsigned long long who = __ballot(has && p.idx[has ? r * p.k + j : 0] >= 0);
        if (j == 0) picked[t] = (int)(who >> (i & 63)) & 255;
      }
      net.tile(nd, m, lds, [&](int t, int n, float v) {
        if (list[t] >= 0) __hip_atomic_store(p.y + (int64_t)list[t] * A + n, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      });
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid < S::T) {
        const int r = list[tid] / p.k;
        done[tid] = list[tid] >= 0 && __hip_atomic_fetch_add(p.count + r, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == __popc(picked[tid]) - 1 ? r : -1;
      }
      __syncthreads();
      for (int i = tid; i < S::T * A; i += threads) {
        const int t = i / A, a = i - t * A, r = done[t];
        if (r < 0) continue;
        float sum = 0.f;
        for (int j = 0; j < p.k; ++j)
          if (picked[t] >> j & 1) sum = fmaf(probs[t][j], __hip_atomic_load(p.y + ((int64_t)r * p.k + j) * A + a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), sum);
        p.out[r * p.out_row + a] = sum;
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// The router's gradient.  16 lanes take the dlogit of a place (a lane the outputs a, a + 16, ..).
// Few places: one launch, a workgroup per agent looks through idx itself, 256 places at once, and sums dlogit x over its own:
// thread (u, s) over the collected places u, u + parts, .. of input s, and the parts in their order.
// Many: a first launch takes all dlogits and, in other workgroups, sorts the places by agent; in a second one a workgroup per agent
// sums over the places that picked it, a wave every fourth of them, a lane an input, then the waves' sums.  Few agents: several
// workgroups each, a run of sorted blocks every one; their sums go to the workspace, and the last of them adds all.  So the order
// of a sum hangs on the sizes, never on who came first.
// Sums over rows are in fp64 (an agent may be picked by every row).  A dlogit is fp32: its dot products have as many terms as the
// nets have outputs, of answers that are fp32 sums themselves, and it is off by (outputs + top_k + 4) 2^-24 of the terms' magnitudes
// at most, once a place.  Bound by launches and latency: 16 agents of 18 inputs, 9 rows,
// top 2: 4.1 us; 1024 of 45, 4096 rows, top 4: 5.9 and 6.3 us (sums by the workgroup of an agent over unsorted idx: 65).
// ------------------------------------------------------------------------------------------------------------------------
// dlogit of a place, in all of its 16 lanes (a0 = 0 .. 15), and dy; one that picked nobody: 0
template <int KM>
__device__ __forceinline__ float dlogit_of(const SnapGrad &p, int place, int a0) {
  const int r = place / p.k, j = place - r * p.k, A = p.A;
  const float *dout = p.dout + (int64_t)r * p.dout_row, *y = p.y + (int64_t)r * p.k * A;
  float dot[KM], pr[KM];
  unsigned picked = 0;                                     // places that picked nobody may hold anything
#pragma unroll
  for (int v = 0; v < KM; ++v) {
    const int at = r * p.k + min(v, p.k - 1), ev = p.idx[at];
    pr[v] = p.prob[at];
    picked |= (v < p.k && ev >= 0 && ev < p.G) << v;
    dot[v] = 0.f;
  }
  for (int a = a0; a < A; a += 16) {
    const float d = dout[a];
#pragma unroll
    for (int v = 0; v < KM; ++v) dot[v] = fmaf(y[min(v, p.k - 1) * A + a], d, dot[v]);
  }
  float all = 0.f, own = 0.f, pj = 0.f;
#pragma unroll
  for (int v = 0; v < KM; ++v) {
    const float d = sum_of_16(dot[v]);
    all = picked >> v & 1 ? fmaf(pr[v], d, all) : all;
    if (v == j) { own = d; pj = picked >> v & 1 ? pr[v] : 0.f; }
  }
  if (p.dy) for (int a = a0; a < A; a += 16) p.dy[(int64_t)place * A + a] = picked >> j & 1 ? pj * dout[a] : 0.f;
  return picked >> j & 1 ? pj * (own - all) : 0.f;
}

template <int KM>
__global__ void __launch_bounds__(256)
snap_grad_few_kernel(const SnapGrad p) {
  __shared__ int list[256], wsum[4];
  __shared__ float dl[256];
  __shared__ double part[256];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = p.S, total = p.n * p.k;
  const int s0 = S < 256 ? S : 256, parts = 256 / s0, u = tid / s0, sx = tid - u * s0;
  double acc[4] = {0., 0., 0., 0.}, bacc = 0.;             // S <= 1024
  for (int from = 0; from < total; from += 256) {
    const int i = from + tid;
    const int v = i < total ? p.idx[i] : -1;
    // (agent 0's workgroup also looks after the places that picked nobody: their dy)
    const bool mine = i < total && (v == e || (e == 0 && p.dy && (v < 0 || v >= p.G)));
    const unsigned long long b = __ballot(mine);
    if (lane == 0) wsum[wave] = __popcll(b);
    __syncthreads();
    int at = 0;
    for (int w = 0; w < wave; ++w) at += wsum[w];
    if (mine) list[at + __popcll(b & ((1ull << lane) - 1ull))] = i;
    const int have = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
    if (!have) continue;
    for (int m = tid >> 4; m < have; m += 16) {
      const float d = dlogit_of<KM>(p, list[m], tid & 15);
      if ((tid & 15) == 0) dl[m] = d;
    }
    __syncthreads();
    if (u < parts) {
#pragma unroll 4
      for (int m = u; m < have; m += parts) {
        const float *x = p.x + (int64_t)(list[m] / p.k) * p.x_row;
        const int pick = p.idx[list[m]];
        const double d = dl[m];
        if (pick != e) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) { const int s = sx + 256 * j; if (s < S && (j == 0 || s0 == 256)) acc[j] = fma(d, (double)x[s], acc[j]); }
        if (sx == 0) bacc += d;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (256 * j >= S) break;
    part[tid] = acc[j];
    __syncthreads();
    const int s = sx + 256 * j;
    if (u == 0 && s < S) {
      double v = 0.;
      for (int i = 0; i < parts; ++i) v += part[i * s0 + sx];
      p.dw[(int64_t)e * p.dw_row + s] = (float)v;
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

// workgroups 0 .. blocks - 1 sort, the others take 64 dlogits each
template <int KM>
__global__ void __launch_bounds__(1024)
snap_grad_first_kernel(const SnapGrad p, int bits) {
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, total = p.n * p.k;
  if ((int)blockIdx.x < p.blocks) {
    if (p.sums && blockIdx.x == 0) for (int e = tid; e < p.G; e += 1024) p.done[e] = 0;
    sort_block(p.idx, blockIdx.x, total, p.G, bits, p.sorted, p.start, lds);
    return;
  }
  const int place = (blockIdx.x - p.blocks) * 64 + (tid >> 4);
  if (place >= total) return;                              // (16 lanes together)
  const float d = dlogit_of<KM>(p, place, tid & 15);
  if ((tid & 15) == 0) p.dlogit[place] = d;
}

template <int SJ>                                          // 64 SJ inputs
__global__ void __launch_bounds__(256)
snap_grad_sum_kernel(const SnapGrad p) {
  __shared__ int rows[256], last;
  __shared__ float dl[256];
  __shared__ double part[4][64];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), S = p.S;
  double acc[SJ], bacc = 0.;
#pragma unroll
  for (int j = 0; j < SJ; ++j) acc[j] = 0.;
  const int b_from = blockIdx.y * p.piece, b_to = min(p.blocks, b_from + p.piece);
  for (int b0 = b_from; b0 < b_to; b0 += 64) {
    const int nb = min(64, b_to - b0);
    const Places places = places_of(p.start, p.G, e, b0, nb, lane);
    int have = 1;
    for (int i0 = 0; i0 < have; i0 += 256) {
      const int at = place_at(places, nb, i0 + tid, have);   // (the same `have` in every wave)
      if (at >= 0) {
        const int place = p.sorted[at];
        rows[tid] = place / p.k;
        dl[tid] = p.dlogit[place];
      }
      const int now = min(256, have - i0);
      __syncthreads();
#pragma unroll 8
      for (int i = wave; i < now; i += 4) {
        const double d = dl[i];
        const float *x = p.x + (int64_t)rows[i] * p.x_row;
#pragma unroll
        for (int j = 0; j < SJ; ++j) acc[j] = fma(d, (double)x[min(64 * j + lane, S - 1)], acc[j]);
        bacc += d;
      }
      __syncthreads();
    }
  }
  double *ws = p.sums ? p.sums + ((size_t)blockIdx.y * p.G + e) * (S + 1) : nullptr;
#pragma unroll
  for (int j = 0; j < SJ + 1; ++j) {                       // the waves, in order; row SJ: the bias, column S of the workspace's rows
    if (j == SJ && !p.db) break;
    part[wave][lane] = j < SJ ? acc[j < SJ ? j : 0] : bacc;
    __syncthreads();
    const int s = j < SJ ? 64 * j + lane : S;
    if (wave == 0 && (j < SJ ? s < S : lane == 0)) {
      const double v = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
      if (ws) __hip_atomic_store(ws + s, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      else if (s < S) p.dw[(int64_t)e * p.dw_row + s] = (float)v;
      else p.db[e] = (float)v;
    }
    __syncthreads();
  }
  if (!ws) return;
  // whoever is last of an agent's workgroups adds their sums (stored past the XCD's cache, told of once arrived)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) last = __hip_atomic_fetch_add(p.done + e, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.y - 1;
  __syncthreads();
  if (!last) return;
  for (int s = tid; s < S + (p.db ? 1 : 0); s += 256) {
    double v = 0.;
#pragma unroll 8
    for (int j = 0; j < (int)gridDim.y; ++j)
      v += __hip_atomic_load(p.sums + ((size_t)j * p.G + e) * (S + 1) + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (s < S) p.dw[(int64_t)e * p.dw_row + s] = (float)v; else p.db[e] = (float)v;
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------------------------------------
static int most_strips(const SnapDesc &nd) {
  int most = 0;
  for (int l = 0; l < nd.L; ++l) most = nd.lay[l].strips > most ? nd.lay[l].strips : most;
  return most;
}
static int waves_for(const SnapDesc &nd, int mt, int most) {
  const int waves = (most_strips(nd) + mt - 1) / mt;
  return waves > most ? most : waves;
}
// the LDS of a kernel, and where in it what lies
template <int BITS, int R, int NT, bool STAGED>
static int lds_for(const SnapDesc &nd, SnapLds &m) { return SnapShape<BITS, R, NT>::bytes(nd, m) + (STAGED ? nd.stride + (BITS == 32 ? SNAP_OVER : 0) : 0); }
template <int BITS, int R, int NT, bool STAGED>
static bool fits(const SnapDesc &nd, int most) { SnapLds m; return lds_for<BITS, R, NT, STAGED>(nd, m) <= most; }

#define SNAP_HALF (SNAP_LDS / 2)      // two workgroups a CU: one computes while the other's net arrives
template <int BITS, int R, int MT, bool STAGED>
static hipError_t forward_run(const SnapDesc &nd, SnapForward p, hipStream_t st) {
  SnapLds m;
  const int lds = lds_for<BITS, R, 1, STAGED>(nd, m);
  static LdsConfig cfg;
  const auto kernel = snap_forward_kernel<BITS, R, 1, MT, STAGED>;
  hipError_t e = ddrl_set_lds(kernel, lds, cfg);
  if (e != hipSuccess) return e;
  const int tiles = (p.n + R - 1) / R;
  // 2048 workgroups where there are as many tiles (129 agents, 24-100-100-1, 250 rows: 17 us, with 1024 21 us)
  int chunks = (2048 + p.G - 1) / p.G;
  if (chunks > tiles) chunks = tiles;
  const int per = (tiles + chunks - 1) / chunks;
  p.per = per * R;
  // 8 waves; tiles of 16 rows of larger nets 12 (4 bits: two workgroups of them fit a CU's registers), where the activations leave
  // room for one workgroup a CU 16 (1024 agents, 64 rows: 18-400-300-6 with 8 waves 103 us, 12 97, 10 127, as 10 do not
  // spread evenly over the SIMDs and the second workgroup does not fit, 16 132; 18-600-500-6 with 8 275, with 16 219)
  const int most = R != 16 || STAGED ? 8 : lds > SNAP_HALF ? 16 : BITS == 4 ? 12 : 8;
  hipLaunchKernelGGL(kernel, dim3(p.G, (tiles + per - 1) / per), dim3(waves_for(nd, MT, most) * 64), lds, st, nd, m, p);
  return hipGetLastError();
}

// Rows a tile: n of 2 to 4 as 4 (4 bits; 1024 agents of 18-400-300-6, 4 rows: 23 us, in tiles of 16 28 us), more as 16.
// Staged or not: a net that lets two workgroups share a CU is staged whole (1024 agents, 18-100-100-6: 16 rows 9.6 us, unstaged
// 12.5; 1 row 7.3 and 7.7).  A larger one goes from memory to registers (18-400-300-6, all but its first layer staged: 1 row 27
// us, unstaged 22; 64 rows 147 and 105).
// Strips a wave: two share a read of the inputs but leave waves idle; with very few strips, or more than the 8 waves, one (64
// rows: 18-20-20-6 two 13.7 us, one 12.0; 24-200-200-1 67 and 57; 250 rows of 18-100-100-6: 8.7 and 10.3).
extern "C" hipError_t snap_forward_launch(const SnapDesc *nd, const SnapForward *p, hipStream_t st) {
  if (nd->bits == 4) {
    if (p->n > 4) {
      if (fits<4, 16, 1, true>(*nd, SNAP_HALF)) {
        const int strips = most_strips(*nd);
        return strips > 2 && strips <= 8 ? forward_run<4, 16, 2, true>(*nd, *p, st) : forward_run<4, 16, 1, true>(*nd, *p, st);
      }
      if (fits<4, 16, 1, false>(*nd, SNAP_LDS)) return forward_run<4, 16, 1, false>(*nd, *p, st);
    }
    if (p->n > 1) return fits<4, 4, 1, true>(*nd, SNAP_HALF) ? forward_run<4, 4, 2, true>(*nd, *p, st) : forward_run<4, 4, 1, false>(*nd, *p, st);
    return fits<4, 1, 1, true>(*nd, SNAP_HALF) ? forward_run<4, 1, 2, true>(*nd, *p, st) : forward_run<4, 1, 2, false>(*nd, *p, st);
  }
  if (p->n > 1) return fits<32, 16, 1, true>(*nd, SNAP_HALF) ? forward_run<32, 16, 2, true>(*nd, *p, st) : forward_run<32, 16, 1, false>(*nd, *p, st);
  return fits<32, 1, 1, true>(*nd, SNAP_HALF) ? forward_run<32, 1, 2, true>(*nd, *p, st) : forward_run<32, 1, 2, false>(*nd, *p, st);
}

// A launch has at most 2^32 - 1 threads along x: rows (places) that one launch of the router (of the gradient's first kernel) takes,
// of 32 (16) threads each at most
#define SNAP_AT_ONCE (1 << 26)
template <int KM>
static hipError_t router_run(const SnapMixture &p, int S, int A, hipStream_t st) {
  const int ld = ddrl_roundup(S, 64) + 4;
  const int strips = ((p.G + 15) / 16 + p.chunks - 1) / p.chunks;
  int waves = 4;
  // with enough workgroups, fewer waves with more agents each have fewer lists to merge (256 agents of 45 inputs, 16384 rows: 8
  // waves 24.6 us, 16 33.2; 4096 rows 9.6 and 9.4; 1024 agents, 512 rows 23.5 and 19.4)
  const int most = p.n >= 8192 ? 8 : 16;
  while (waves < most && waves < strips) waves *= 2;
  const size_t lds = (size_t)16 * ld * 4 + (size_t)16 * waves * KM * 12;
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_router_kernel<KM>, lds, cfg);
  if (e != hipSuccess) return e;
  for (int64_t t = 0; t < p.n && e == hipSuccess; t += SNAP_AT_ONCE) {      // (more rows than one launch takes: never in chunks)
    SnapMixture part = p;
    part.n = (int)(p.n - t < SNAP_AT_ONCE ? p.n - t : SNAP_AT_ONCE);
    part.x += t * p.x_row;
    if (p.allowed) part.allowed += t * p.a_row;
    part.out += t * p.out_row;
    part.idx += t * p.k; part.prob += t * p.k; part.y += t * p.k * A;
    part.count += t;
    hipLaunchKernelGGL(snap_router_kernel<KM>, dim3((part.n + 15) / 16, p.chunks), dim3(waves * 64), lds, st, part, S, A, ld);
    e = hipGetLastError();
  }
  return e;
}
template <int BITS, int KM>
static hipError_t row_run(const SnapDesc &nd, const SnapMixture &p, const SnapLds &m, SnapRow at, int waves, int lds, hipStream_t st) {
  static LdsConfig cfg;
  const auto kernel = snap_row_kernel<BITS, 2, KM>;
  hipError_t e = ddrl_set_lds(kernel, lds, cfg);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3(p.n), dim3(waves * 64), lds, st, nd, m, p, at);
  return hipGetLastError();
}
// the LDS of snap_row_kernel
template <int BITS>
static int row_lds(const SnapDesc &nd, int k, SnapLds &m, SnapRow &at) {
  at.waves = waves_for(nd, 2, 16 / k);
  at.lists = ddrl_roundup(nd.lay[0].in, 16) * 4;
  at.y = at.lists + 16 * SNAP_MAXK * 12;
  at.teams = at.y + ddrl_roundup(k * nd.A, 4) * 4;
  at.team = lds_for<BITS, 1, 1, true>(nd, m);
  return at.teams + k * at.team;
}
template <int BITS, int MT, bool STAGED>
static hipError_t place_run(const SnapDesc &nd, const SnapMixture &p, hipStream_t st) {
  SnapLds m;
  const int lds = lds_for<BITS, 1, 1, STAGED>(nd, m);
  static LdsConfig cfg;
  const auto kernel = snap_place_kernel<BITS, MT, STAGED>;
  hipError_t e = ddrl_set_lds(kernel, lds, cfg);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3(p.n * p.k), dim3(waves_for(nd, MT, STAGED ? 8 : 16) * 64), lds, st, nd, m, p);
  return hipGetLastError();
}
template <int BITS, int R, int NT, int MT>
static hipError_t experts_run(const SnapDesc &nd, const SnapMixture &p, hipStream_t st) {
  SnapLds m;
  const int lds = lds_for<BITS, R, NT, false>(nd, m);
  static LdsConfig cfg;
  const auto kernel = snap_experts_kernel<BITS, R, NT, MT>;
  hipError_t e = ddrl_set_lds(kernel, lds, cfg);
  if (e != hipSuccess) return e;
  int waves = waves_for(nd, MT, 8);
  waves = waves < 4 ? 4 : waves;
  // Several workgroups a net, each every share-th of its tiles: a router prefers some nets, and a net's tiles one after the other
  // are what a pass then waits for (1024 agents of 45-64-64-17, 8192 rows, top 4: 77 us with 2 workgroups a net, 60 with 4; 256
  // agents, 4096 rows, top 2: 53 with 2 and 21 with 8 or 16); a workgroup that finds no tile is over after two reads.
  const int64_t total = (int64_t)p.n * p.k, T = R * NT;
  int64_t share = (4096 + p.G - 1) / p.G;
  const int64_t tiles = (total + T - 1) / T;
  if (share > tiles) share = tiles;
  hipLaunchKernelGGL(kernel, dim3(p.G, (unsigned)share), dim3(waves * 64), lds, st, nd, m, p);
  return hipGetLastError();
}
static int sort_bits(int G) {
  int bits = 1;
  while ((1ll << bits) <= G) ++bits;
  return bits;
}
static hipError_t sort_run(const int *idx, int total, int G, int *sorted, int *start, hipStream_t st) {
  const size_t lds = (size_t)(G + 1) * 4;
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_sort_kernel, lds, cfg);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(snap_sort_kernel, dim3((total + SORT_BLOCK - 1) / SORT_BLOCK), dim3(1024), lds, st, idx, total, G, sort_bits(G), sorted, start);
  return hipGetLastError();
}

// agents x inputs up to which a row's workgroup is its own router (64-64 nets, top 2, 8 or 64 rows: 1024 agents of 45 inputs 11.6 us,
// with a router of its own 15.3; 256 of 376 15.6 and 28.7; 1024 of 128 22.0 and 17.9)
#define SNAP_ROUTE 98304
#define SNAP_STATIC_LDS 2048         // snap_experts_kernel's lists
static hipError_t router_launch(const SnapMixture &p, int S, int A, hipStream_t st) {
  return p.k == 1 ? router_run<1>(p, S, A, st) : p.k == 2 ? router_run<2>(p, S, A, st) : p.k <= 4 ? router_run<4>(p, S, A, st) : router_run<8>(p, S, A, st);
}
// A workgroup a row as long as the rows are at most two rounds of what the chip holds at once, 4 waves a SIMD: a round is 8 to 12 us,
// the three launches of many places some 20 (top 2: 500 rows of 256 agents 45-64-64-17 in 4 bits 10.7 us, in three launches
// 23.3; 2000 rows, two rounds, 20.6 and 26.7; 4000 rows 40.7 and 31.0; in 32 bits, one workgroup a CU, 500 rows 19 to 21 and
// 23.5, 1000 rows 34 and 25; 16 agents of 18-20-6, 4000 rows 15.5 and 21.5).
// It is its own router as long as that is one round (the same 256 agents: 1000 rows 14.3 us, with a router of its own 16.9; 2000
// rows 24.1 and 20.6; 1024 agents, whose router takes 16 waves: 200 rows 14.2 and 19.1, 500 rows 23.7 and 16.2).
static int rows_at_once(int waves, int lds) {
  const int by_waves = 16 / waves, by_lds = SNAP_LDS / (lds + 64);
  return 256 * (by_waves < by_lds ? by_waves : by_lds);
}
template <int BITS>
static bool mixture_rows(const SnapDesc &nd, const SnapMixture &p, hipStream_t st, hipError_t &e) {
  const int S = nd.lay[0].in;
  SnapLds m;
  SnapRow at;
  const int lds = row_lds<BITS>(nd, p.k, m, at);
  if (lds > SNAP_LDS - 1024) return false;
  const int own = p.k * at.waves, agents = p.G > 1024 ? 16 : (p.G + 63) / 64, all = own > agents ? own : agents;    // (a thread an agent)
  if ((long long)p.G * S <= SNAP_ROUTE && p.n <= rows_at_once(all, lds)) {
    e = p.k <= 4 ? row_run<BITS, 4>(nd, p, m, at, all, lds, st) : row_run<BITS, 8>(nd, p, m, at, all, lds, st);
    return true;
  }
  if (p.n > 2 * rows_at_once(own, lds)) return false;
  if ((e = router_launch(p, S, nd.A, st)) == hipSuccess) e = row_run<BITS, 0>(nd, p, m, at, own, lds, st);
  return true;
}
template <int BITS>
static hipError_t mixture_places(const SnapDesc &nd, const SnapMixture &p, hipStream_t st) {
  const hipError_t e = router_launch(p, nd.lay[0].in, nd.A, st);
  if (e != hipSuccess) return e;
  return fits<BITS, 1, 1, true>(nd, SNAP_HALF) ? place_run<BITS, 2, true>(nd, p, st) : place_run<BITS, 2, false>(nd, p, st);
}
extern "C" hipError_t snap_mixture_launch(const SnapDesc *nd, const SnapMixture *q, hipStream_t st) {
  SnapMixture p = *q;
  const int total = p.n * p.k, left = SNAP_LDS - SNAP_STATIC_LDS;
  hipError_t e = hipSuccess;
  if (nd->bits == 4 ? mixture_rows<4>(*nd, p, st, e) : mixture_rows<32>(*nd, p, st, e)) return e;
  // (64 agents of 18-400-300-6 in 32 bits, top 2: 128 rows by place 28.4 us, by net 32.8; 250 rows 45.8 and 33.2)
  if (total <= SNAP_FEW) return nd->bits == 4 ? mixture_places<4>(*nd, p, st) : mixture_places<32>(*nd, p, st);
  p.chunks = 1;                                             // (the router picks)
  if ((e = router_launch(p, nd->lay[0].in, nd->A, st)) != hipSuccess) return e;
  if ((e = sort_run(p.idx, total, p.G, p.sorted, p.start, st)) != hipSuccess) return e;
  // From memory to registers, not staged (16 agents of 18-100-100-6, 1024 rows, 32 bits: 20.7 us, staged 25.3; 256 of 45-64-64-17,
  // 4096 rows: the same).  Very many places of nets that leave two workgroups a CU go in tiles of 32 rows (256 agents of 45-64-64-17,
  // 16384 rows: 93 us, in tiles of 16 109; 4096 rows 34.0 and 35.9; 2048 rows 28.1 and 26.1; 64 of 18-400-300-6, 4096 rows 109 and 103).
  const bool many = total >= 8192;
  if (nd->bits == 4) {
    if (many && fits<4, 16, 2, false>(*nd, SNAP_HALF)) return experts_run<4, 16, 2, 1>(*nd, p, st);
    if (fits<4, 16, 1, false>(*nd, left)) return experts_run<4, 16, 1, 1>(*nd, p, st);
    return experts_run<4, 4, 1, 1>(*nd, p, st);
  }
  if (many && fits<32, 16, 2, false>(*nd, SNAP_HALF)) return experts_run<32, 16, 2, 1>(*nd, p, st);
  return experts_run<32, 16, 1, 1>(*nd, p, st);                        // (fits whatever the net: 128 KiB at most)
}

template <int KM>
static hipError_t grad_first_run(const SnapGrad &p, hipStream_t st) {
  if (!p.sorted) {
    hipLaunchKernelGGL(snap_grad_few_kernel<KM>, dim3(p.G), dim3(256), 0, st, p);
    return hipGetLastError();
  }
  const size_t lds = (size_t)(p.G + 1) * 4;
  static LdsConfig cfg;
  hipError_t e = ddrl_set_lds(snap_grad_first_kernel<KM>, lds, cfg);
  if (e != hipSuccess) return e;
  // the first launch sorts all places and takes the first of the dlogits, the others (over 2^26 places) go on; 64 rows are whole workgroups
  const int64_t rows = SNAP_AT_ONCE / p.k / 64 * 64;
  for (int64_t t = 0; t < p.n && e == hipSuccess; t += rows) {
    const int64_t now = p.n - t < rows ? p.n - t : rows;
    SnapGrad part = p;
    if (t) {
      part.blocks = 0;
      part.n = (int)now;
      part.idx += t * p.k; part.prob += t * p.k; part.y += t * p.k * p.A; part.dout += t * p.dout_row;
      if (p.dy) part.dy += t * p.k * p.A;
      part.dlogit += t * p.k;
    }
    hipLaunchKernelGGL(snap_grad_first_kernel<KM>, dim3((unsigned)(part.blocks + (now * p.k + 63) / 64)), dim3(1024), lds, st, part, sort_bits(p.G));
    e = hipGetLastError();
  }
  return e;
}
extern "C" hipError_t snap_grad_launch(const SnapGrad *q, int pieces, hipStream_t st) {
  SnapGrad p = *q;
  p.piece = (p.blocks + pieces - 1) / pieces;
  hipError_t e = p.k <= 2 ? grad_first_run<2>(p, st) : p.k <= 4 ? grad_first_run<4>(p, st) : grad_first_run<8>(p, st);
  if (e != hipSuccess || !p.sorted) return e;
  const dim3 grid(p.G, pieces);
  if (p.S <= 64) hipLaunchKernelGGL(snap_grad_sum_kernel<1>, grid, dim3(256), 0, st, p);
  else if (p.S <= 256) hipLaunchKernelGGL(snap_grad_sum_kernel<4>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(snap_grad_sum_kernel<16>, grid, dim3(256), 0, st, p);
  return hipGetLastError();
}
