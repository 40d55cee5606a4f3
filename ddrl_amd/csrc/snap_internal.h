// snap_internal.h -- shared between snap.hip (handles, argument checks) and kernels_snap.hip: the layout of a served snapshot.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#define SNAP_MAXL 4            // InnerProducts of a net (up to three hidden layers)
#define SNAP_MAXW 1024         // widest layer, as DDRL_WIDE_MAXW
#define SNAP_MAXK 8            // DDRL_SNAP_MAX_TOP_K
#define SNAP_MAX_G 4194303     // agents: a launch has at most 2^32 - 1 threads along x, a workgroup of up to 1024 for each agent
#define SNAP_LDS (160 * 1024)  // a CU's LDS
#define SNAP_FEW 256           // places (rows x top_k) up to which a mixture of large nets gives every place a workgroup of its own
#define SNAP_CHUNK 256         // agents a router workgroup looks at when there are few rows
#define SNAP_CHUNK_ROWS 4096   // rows up to which a row's agents are spread over several

// An agent's net is one image of `stride` bytes: its layers one after the other, a layer a row of records, one for 16 outputs
// (a "strip"), made for a matrix instruction whose A operand is 16 outputs by one k-step of inputs, so that a wave's load is one
// contiguous piece of memory in lane order (lane = 16 q + r <-> output r of the strip):
//   32 bits: a k-step is 16 inputs, lane (r, q) holds inputs 4q .. 4q+3 as one float4: 1 KiB a step;
//    4 bits: a k-step is 32 inputs, lane (r, q) holds inputs 8q .. 8q+7 as one dword of codes (lowest input in the lowest
//            bits): 256 bytes a step.  Four steps lie together, [lane][step], 16 bytes a lane; the last steps % 4 too, with as
//            many dwords a lane.  Behind the steps the scales, a byte each (E8M0: 2^(byte - 127)), [step / 4][output][step % 4].
// A record ends with the 16 biases, fp32.  Outputs are padded to strips and inputs to k-steps with zeros.
struct SnapLayer {
  int in, out, strips, steps;
  unsigned off, rec;                          // bytes: where the layer starts, a record
  int act, code;                              // code: bytes of a record's steps
};
struct alignas(8) SnapDesc {                  // (the first argument of the kernels, which read it where it lies)
  SnapLayer lay[SNAP_MAXL];
  int L, bits, A, np;                         // layers; outputs of the net; parameters in the flat order
  unsigned stride;
};

static inline void snap_build_desc(SnapDesc &n, int d0, const int *hidden, int nh, int dout, int hact, int oact, int bits) {
  n = SnapDesc();
  n.L = nh + 1; n.bits = bits; n.A = dout;
  unsigned off = 0;
  for (int l = 0; l < n.L; ++l) {
    SnapLayer &y = n.lay[l];
    const int K = y.in = l ? hidden[l - 1] : d0, N = y.out = l < nh ? hidden[l] : dout;
    y.act = l < nh ? hact : oact;
    y.strips = (N + 15) / 16;
    y.steps = bits == 4 ? (K + 31) / 32 : (K + 15) / 16;
    y.code = y.steps * (bits == 4 ? 256 : 1024);
    y.rec = (unsigned)y.code + (bits == 4 ? (y.steps + 3) / 4 * 64 : 0) + 64;
    y.off = off; off += y.strips * y.rec;
    n.np += N * K + N;
  }
  n.stride = (off + 1023) / 1024 * 1024;
}
// where the codes of (step, lane) lie in a record
__host__ __device__ inline unsigned snap_code_off(int steps, int step, int lane) {
  const int whole = steps & ~3, in4 = step < whole ? 4 : steps & 3;
  return (step & ~3) * 256 + lane * 4 * in4 + (step & 3) * 4;
}
#define SNAP_OVER 4096         // bytes behind the last image that a 32-bit kernel may read (never use): whatever it asks for, it asks for four steps
// where the scale of (output r of a strip, step) lies in a record
__host__ __device__ inline unsigned snap_scale_off(int code, int step, int r) { return (unsigned)code + (step >> 2) * 64 + r * 4 + (step & 3); }

// how many workgroups of the router share a row's agents, where those who answer the rows or places merge the lists: as many as
// there are SNAP_CHUNKs, up to 16 (top 2: 2000 agents of 64-400-300-6, 4 rows 23.4 us, by one workgroup 48.8; 1024 of 128-64-64-6,
// 500 rows 19.8 and 37.8, 2000 rows 38.4 and 45.5)
static inline int snap_chunks(int G, int n) {
  if (n > SNAP_CHUNK_ROWS) return 1;
  const int c = (G + SNAP_CHUNK - 1) / SNAP_CHUNK;
  return c > 16 ? 16 : c;
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
  unsigned long long *ckey; int *cidx;   // [n x chunks x k] each chunk's best, where the router's agents are spread over several workgroups
  int chunks;
  int *sorted, *start, blocks;        // idx sorted by net, a block of 1024 places at a time: [blocks x 1024], [blocks x (G + 1)]
};
struct SnapGrad {
  int G, n, k, S, A;
  const float *x; int64_t x_row;
  const int *idx; const float *prob; const float *y;
  const float *dout; int64_t dout_row;
  float *dw; int64_t dw_row;
  float *db, *dy;
  int *sorted, *start, blocks;        // as in SnapMixture; null: few places, every workgroup looks through idx itself
  float *dlogit;                      // [n x k]
  double *sums;                       // [pieces x G x (S + 1)] where an agent's places are several workgroups' work
  int *done;                          // [G] those that are through
  int piece;                          // blocks of one of them
};
// places from which the gradient sorts them first (16 agents of 18 inputs: 400 places 7.7 us, sorted 8.0; 1000 places 13.9 and 8.8;
// 1024 of 45: 6.4 and 8.1, 9.7 and 8.6)
#define SNAP_SORT_FROM 512
#define SNAP_SORT_MAX_G 16383          // the sort keeps a counter a net in LDS
static inline int snap_blocks(int n, int k) { return (int)(((long long)n * k + 1023) / 1024); }
// how many workgroups an agent: a router prefers some agents, and the places of one are what a pass waits for (5 agents, 3868
// places 12.9 us, one workgroup each 21.6; 256 agents, 16000 places 12.9 and 13.5)
static inline int snap_grad_pieces(int G, int n, int k) {
  const int b = snap_blocks(n, k);
  int p = (1024 + G - 1) / G;
  return p > b ? (b < 1 ? 1 : b) : p;
}

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
hipError_t snap_grad_launch(const SnapGrad *p, int pieces, hipStream_t st);
}
