// snap_internal.h -- shared between snap.hip (handles, argument checks) and kernels_snap.hip: the layout of a served snapshot.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#define SNAP_MAXL 4            // InnerProducts of a net (up to three hidden layers)
#define SNAP_MAXW 1024         // widest layer, as DDRL_WIDE_MAXW
#define SNAP_MAXK 8            // DDRL_SNAP_MAX_TOP_K
#define SNAP_LDS (160 * 1024)  // a CU's LDS

// An agent's net is one image of `stride` bytes, made for a matrix instruction whose A operand is 16 outputs (a "strip") by
// one k-step of inputs, so that a wave's load is one contiguous piece of memory in lane order (lane = 16 q + r <-> output r of
// the strip):
//   32 bits: a k-step is 16 inputs, lane (r, q) holds inputs 4q .. 4q+3 as one float4: 1 KiB a step;
//    4 bits: a k-step is 32 inputs, lane (r, q) holds inputs 8q .. 8q+7 as one dword of codes (lowest input in the lowest
//            bits); four steps lie together (lane by lane 16 bytes, 1 KiB), the last steps % 4 ones each by itself (256 bytes);
//            the scales are a byte each (E8M0: 2^(byte - 127)), [strip][step / 4][output][step % 4].
// Outputs are padded to strips and inputs to k-steps with zeros.  Biases: fp32, padded with zeros.
struct SnapDesc {
  int L, bits, hact, oact;
  int d[SNAP_MAXL + 1];
  int in[SNAP_MAXL], out[SNAP_MAXL], A;                         // of layer l; of the net
  int strips[SNAP_MAXL], steps[SNAP_MAXL];
  unsigned woff[SNAP_MAXL], soff[SNAP_MAXL], boff[SNAP_MAXL];   // byte offsets in an image: weights, scales, biases
  unsigned stride;
  int np;                                                       // parameters in the flat order
};

static inline void snap_build_desc(SnapDesc &n, int d0, const int *hidden, int nh, int dout, int hact, int oact, int bits) {
  n = SnapDesc();
  n.L = nh + 1; n.bits = bits; n.hact = hact; n.oact = oact;
  n.d[0] = d0;
  for (int i = 0; i < nh; ++i) n.d[i + 1] = hidden[i];
  n.d[nh + 1] = dout;
  unsigned off = 0;
  for (int l = 0; l < n.L; ++l) {
    const int K = n.in[l] = n.d[l], N = n.out[l] = n.d[l + 1];
    n.strips[l] = (N + 15) / 16;
    n.steps[l] = bits == 4 ? (K + 31) / 32 : (K + 15) / 16;
    n.woff[l] = off; off += (unsigned)n.strips[l] * n.steps[l] * (bits == 4 ? 256 : 1024);
    n.soff[l] = off; if (bits == 4) off += (unsigned)n.strips[l] * ((n.steps[l] + 3) / 4) * 64;
    n.boff[l] = off; off += (unsigned)n.strips[l] * 64;
    n.np += N * K + N;
  }
  n.A = dout;
  n.stride = (off + 1023) / 1024 * 1024;
}
// where the code of (output n, 32-bit piece of 8 inputs (step, q)) of a 4-bit layer lies
__host__ __device__ inline unsigned snap_code_off(int steps, int strip, int step, int lane) {
  const int full = steps & ~3;
  const unsigned at = (unsigned)strip * steps * 256;
  return step < full ? at + (step >> 2) * 1024 + lane * 16 + (step & 3) * 4 : at + step * 256 + lane * 4;
}
__host__ __device__ inline unsigned snap_scale_off(int steps, int strip, int step, int r) {
  return (unsigned)(strip * ((steps + 3) / 4) + (step >> 2)) * 64 + r * 4 + (step & 3);
}

struct SnapForward {
  int G, n, per;                      // per: rows of an agent that one workgroup answers
  const char *img;
  const float *x; int64_t x_agent, x_row;
  float *out; int64_t out_agent, out_row;
  const uint8_t *mask;
};
struct SnapMixture {
  int G, n, k;
  const char *img;
  const float *x; int64_t x_row;
  const float *rw; int64_t r_row;
  const float *rb;
  const uint8_t *allowed; int64_t a_row;
  float *out; int64_t out_row;
  int *idx; float *prob; float *y;
  int *count;                         // [n] places of a row that are answered
};
struct SnapGrad {
  int G, n, k, S, A;
  const float *x; int64_t x_row;
  const int *idx; const float *prob; const float *y;
  const float *dout; int64_t dout_row;
  float *dw; int64_t dw_row;
  float *db, *dy;
};

// where the parameters of a load come from: the tile-major nets of a population, or flat rows
struct SnapSource {
  const float *w; size_t agent;       // elements from one agent to the next (0: all the same)
  int tiled;
  int offw[SNAP_MAXL], offb[SNAP_MAXL], kp[SNAP_MAXL];
};

extern "C" {
hipError_t snap_load_launch(const SnapDesc *nd, char *img, const SnapSource *src, int G, hipStream_t st);
hipError_t snap_forward_launch(const SnapDesc *nd, const SnapForward *p, hipStream_t st);
hipError_t snap_mixture_launch(const SnapDesc *nd, const SnapMixture *p, hipStream_t st);
hipError_t snap_grad_launch(const SnapGrad *p, hipStream_t st);
}
