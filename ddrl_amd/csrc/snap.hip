// snap.hip -- host side of served snapshots (include/ddrl_pop.h, "Served snapshots"): handles, argument checks, staging of the
// host-buffer forms.  Kernels: kernels_snap.hip, layout: snap_internal.h.
#include "pop_host.h"
#include "snap_internal.h"

struct ddrl_snap {
  SnapDesc nd;
  int G = 0, device = 0;
  char *img = nullptr;
  hipStream_t stream = nullptr;        // the host-buffer forms
  hipEvent_t loaded = nullptr;         // the last load, for the host-buffer forms
};

namespace {
// the calling thread's current device, put back on the way out
struct OnDevice {
  int was = -1;
  hipError_t e;
  explicit OnDevice(int dev) {
    e = hipGetDevice(&was);
    if (e == hipSuccess && was != dev) e = hipSetDevice(dev); else if (e == hipSuccess) was = -1;
  }
  ~OnDevice() { if (was >= 0) (void)hipSetDevice(was); }
};
struct DevBuf {                        // temporary device memory of a host-buffer call
  char *p = nullptr;
  ~DevBuf() { if (p) (void)hipFree(p); }
  hipError_t get(size_t n) { return hipMalloc((void **)&p, std::max<size_t>(n, 16)); }
};
bool off4(const void *p) { return ((uintptr_t)p & 3) != 0; }
size_t up16(size_t n) { return (n + 15) / 16 * 16; }
struct MixSpace { size_t count, idx, prob, y, ckey, cidx, sorted, start, all; int chunks, blocks; };
MixSpace mix_space(const ddrl_snap *s, int n, int k) {
  MixSpace w;
  const size_t places = (size_t)n * k;
  w.count = 0;
  w.idx = up16((size_t)n * 4);
  w.prob = w.idx + up16(places * 4);
  w.y = w.prob + up16(places * 4);
  w.ckey = w.y + up16(places * s->nd.A * 4);
  w.chunks = snap_chunks(s->G, n);
  const size_t lists = w.chunks > 1 ? places * w.chunks : 0;
  w.cidx = w.ckey + up16(lists * 8);
  w.sorted = w.cidx + up16(lists * 4);
  w.blocks = places > SNAP_FEW ? snap_blocks(n, k) : 0;
  w.start = w.sorted + (size_t)w.blocks * 1024 * 4;
  w.all = w.start + up16((size_t)w.blocks * (s->G + 1) * 4);
  return w;
}
struct GradSpace { size_t sorted, start, dlogit, done, sums, all; int blocks, pieces; };
GradSpace grad_space(const ddrl_snap *s, int n, int k) {
  GradSpace w;
  const bool sort = (long long)n * k >= SNAP_SORT_FROM;
  w.blocks = sort ? snap_blocks(n, k) : 0;
  w.pieces = sort ? snap_grad_pieces(s->G, n, k) : 1;
  w.sorted = 0;
  w.start = (size_t)w.blocks * 1024 * 4;
  w.dlogit = w.start + up16((size_t)w.blocks * (s->G + 1) * 4);
  w.done = w.dlogit + (sort ? up16((size_t)n * k * 4) : 0);
  w.sums = w.done + (w.pieces > 1 ? up16((size_t)s->G * 4) : 0);
  w.all = w.sums + (w.pieces > 1 ? (size_t)w.pieces * s->G * (s->nd.lay[0].in + 1) * 8 : 0);
  return w;
}
int check_mix_shape(const ddrl_snap *s, int n, int k) {
  if (n < 0 || k < 1 || k > DDRL_SNAP_MAX_TOP_K || k > s->G)
    return ddrl_fail(DDRL_EINVAL, "n=%d, top_k=%d: n >= 0 and 1 <= top_k <= min(%d, %d agents)", n, k, DDRL_SNAP_MAX_TOP_K, s->G);
  if ((int64_t)n * k >= SNAP_FEW && s->G > SNAP_SORT_MAX_G)
    return ddrl_fail(DDRL_EINVAL, "n * top_k = %lld with %d agents: %d or more places are served for up to %d agents", (long long)n * k, s->G, SNAP_FEW, SNAP_SORT_MAX_G);
  if ((int64_t)n * k > (1 << 28)) return ddrl_fail(DDRL_EINVAL, "n * top_k = %lld over %d", (long long)n * k, 1 << 28);
  return DDRL_OK;
}
}  // namespace

#define ON_DEVICE(s)                                                                                \
  OnDevice on_((s)->device);                                                                        \
  if (on_.e != hipSuccess) return ddrl_fail(DDRL_EHIP, "hipSetDevice(%d): %s", (s)->device, hipGetErrorString(on_.e))

extern "C" int ddrl_snap_destroy(ddrl_snap_t *s) {
  if (!s) return DDRL_OK;
  OnDevice on(s->device);
  if (s->stream) { (void)hipStreamSynchronize(s->stream); (void)hipStreamDestroy(s->stream); }
  if (s->loaded) (void)hipEventDestroy(s->loaded);
  if (s->img) (void)hipFree(s->img);
  delete s;
  return DDRL_OK;
}

extern "C" int ddrl_snap_create(int n_agents, int in_dim, int out_dim, const int *hidden, int n_hidden, int hidden_layer_type,
                                int output_layer_type, int bits, int device, ddrl_snap_t **out) {
  if (!out || (n_hidden > 0 && !hidden)) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  *out = nullptr;
  if (n_agents < 1 || n_agents > SNAP_MAX_G) return ddrl_fail(DDRL_EINVAL, "n_agents=%d outside 1..%d", n_agents, SNAP_MAX_G);
  if (n_hidden < 0 || n_hidden > DDRL_MAX_HIDDEN) return ddrl_fail(DDRL_EINVAL, "n_hidden=%d outside 0..%d", n_hidden, DDRL_MAX_HIDDEN);
  if (in_dim < 1 || in_dim > SNAP_MAXW || out_dim < 1 || out_dim > SNAP_MAXW)
    return ddrl_fail(DDRL_EINVAL, "in_dim=%d / out_dim=%d outside 1..%d", in_dim, out_dim, SNAP_MAXW);
  for (int i = 0; i < n_hidden; ++i)
    if (hidden[i] < 1 || hidden[i] > SNAP_MAXW) return ddrl_fail(DDRL_EINVAL, "hidden[%d]=%d outside 1..%d", i, hidden[i], SNAP_MAXW);
  if (hidden_layer_type < 0 || hidden_layer_type > 3 || output_layer_type < 0 || output_layer_type > 3)
    return ddrl_fail(DDRL_EINVAL, "hidden_layer_type / output_layer_type not in 0..3");
  if (bits != 32 && bits != 4) return ddrl_fail(DDRL_EINVAL, "bits=%d: 32 or 4", bits);
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1)
    return ddrl_fail(DDRL_EHIP, "no HIP device: libddrl_pop has no CPU path");
  if (device < 0 && hipGetDevice(&device) != hipSuccess) device = 0;
  if (device >= ndev) return ddrl_fail(DDRL_EINVAL, "device %d of %d", device, ndev);
  OnDevice on(device);
  if (on.e != hipSuccess) return ddrl_fail(DDRL_EHIP, "hipSetDevice(%d): %s", device, hipGetErrorString(on.e));
  ddrl_snap *s = new (std::nothrow) ddrl_snap();
  if (!s) return ddrl_fail(DDRL_ENOMEM, "out of host memory");
  s->G = n_agents; s->device = device;
  snap_build_desc(s->nd, in_dim, hidden, n_hidden, out_dim, hidden_layer_type, output_layer_type, bits);
  const size_t bytes = (size_t)n_agents * s->nd.stride + SNAP_OVER;
  auto bail = [&](int code, const char *what, hipError_t e) {
    const int rc = ddrl_fail(code, "%s: %s", what, hipGetErrorString(e));
    ddrl_snap_destroy(s);
    return rc;
  };
  hipError_t e = hipMalloc((void **)&s->img, bytes);
  if (e != hipSuccess) { s->img = nullptr; return bail(DDRL_ENOMEM, "hipMalloc", e); }
  if ((e = hipStreamCreateWithFlags(&s->stream, hipStreamNonBlocking)) != hipSuccess) { s->stream = nullptr; return bail(DDRL_EHIP, "hipStreamCreate", e); }
  if ((e = hipEventCreateWithFlags(&s->loaded, hipEventDisableTiming)) != hipSuccess) { s->loaded = nullptr; return bail(DDRL_EHIP, "hipEventCreate", e); }
  if ((e = hipMemsetAsync(s->img, 0, bytes, s->stream)) != hipSuccess) return bail(DDRL_EHIP, "hipMemset", e);
  if ((e = hipStreamSynchronize(s->stream)) != hipSuccess) return bail(DDRL_EHIP, "hipStreamSynchronize", e);
  *out = s;
  return DDRL_OK;
}

extern "C" int ddrl_snap_create_from(ddrl_pop_t *h, int net, int bits, ddrl_snap_t **out) {
  if (!h || !out) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  *out = nullptr;
  if (bad_net(h, net)) return ddrl_fail(DDRL_EINVAL, "net %d is not one of this population", net);
  const NetDesc &n = train_net(h, net)->nd;
  int rc = ddrl_snap_create(h->G, n.d(0), n.d(n.L()), n.d_ + 1, n.L() - 1, n.hidden_act(), n.out_act(), bits, h->device, out);
  if (rc) return rc;
  rc = ddrl_snap_load(*out, h, net, (*out)->stream);
  if (!rc && hipStreamSynchronize((*out)->stream) != hipSuccess) rc = ddrl_fail(DDRL_EHIP, "hipStreamSynchronize failed");
  if (rc) { ddrl_snap_destroy(*out); *out = nullptr; }
  return rc;
}

extern "C" int ddrl_snap_shape(ddrl_snap_t *s, int *n_agents, int *in_dim, int *out_dim, int *bits, int *n_params) {
  if (!s) return ddrl_fail(DDRL_EINVAL, "NULL handle");
  if (n_agents) *n_agents = s->G;
  if (in_dim) *in_dim = s->nd.lay[0].in;
  if (out_dim) *out_dim = s->nd.A;
  if (bits) *bits = s->nd.bits;
  if (n_params) *n_params = s->nd.np;
  return DDRL_OK;
}

static int refuse_capture(hipStream_t st) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  HIPCHK(hipStreamIsCapturing(st, &cs));
  if (cs != hipStreamCaptureStatusNone) return ddrl_fail(DDRL_ESTATE, "a load cannot be captured into a graph");
  return DDRL_OK;
}

extern "C" int ddrl_snap_load(ddrl_snap_t *s, ddrl_pop_t *h, int net, void *stream) {
  if (!s || !h) return ddrl_fail(DDRL_EINVAL, "NULL handle");
  if (bad_net(h, net)) return ddrl_fail(DDRL_EINVAL, "net %d is not one of this population", net);
  const NetDesc &n = train_net(h, net)->nd;
  if (n.bn_any()) return ddrl_fail(DDRL_EINVAL, "net %d has BatchNorm towers: a snapshot holds InnerProducts only", net);
  if (h->gates_on) return ddrl_fail(DDRL_ESTATE, "developmental gates are in force: a snapshot holds the nets alone");
  bool same = h->G == s->G && n.L() == s->nd.L && h->device == s->device;
  for (int i = 0; same && i < n.L(); ++i)
    same = n.d_[i] == s->nd.lay[i].in && n.d_[i + 1] == s->nd.lay[i].out && (i < n.L() - 1 ? n.hidden_act() : n.out_act()) == s->nd.lay[i].act;
  if (!same) return ddrl_fail(DDRL_EINVAL, "the population's net has other dimensions, activations or another GPU than the snapshot");
  ON_DEVICE(s);
  const hipStream_t st = (hipStream_t)stream;
  int rc = refuse_capture(st);
  if (rc) return rc;
  DDRL_WAIT(h);
  SnapSource src = {};
  src.w = net_weights(h, net); src.agent = n.stride(); src.tiled = 1;
  for (int l = 0; l < n.L(); ++l) { src.offw[l] = n.offw_[l]; src.offb[l] = n.offb_[l]; src.kp[l] = n.kp_[l]; }
  HIPCHK(snap_load_launch(&s->nd, s->img, &src, s->G, st));
  HIPCHK(hipEventRecord(s->loaded, st));
  HIPCHK(hipStreamWaitEvent(h->stream, s->loaded, 0));
  return DDRL_OK;
}

extern "C" int ddrl_snap_load_flat_dev(ddrl_snap_t *s, const float *d_flat, int64_t ld, void *stream) {
  if (!s || !d_flat || off4(d_flat)) return ddrl_fail(DDRL_EINVAL, "NULL or misaligned argument");
  if (ld != 0 && ld < s->nd.np) return ddrl_fail(DDRL_EINVAL, "ld=%lld: 0 or at least %d parameters", (long long)ld, s->nd.np);
  ON_DEVICE(s);
  const hipStream_t st = (hipStream_t)stream;
  int rc = refuse_capture(st);
  if (rc) return rc;
  SnapSource src = {};
  src.w = d_flat; src.agent = (size_t)ld; src.tiled = 0;
  int off = 0;
  for (int l = 0; l < s->nd.L; ++l) {
    src.offw[l] = off; off += s->nd.lay[l].in * s->nd.lay[l].out;
    src.offb[l] = off; off += s->nd.lay[l].out;
  }
  HIPCHK(snap_load_launch(&s->nd, s->img, &src, s->G, st));
  HIPCHK(hipEventRecord(s->loaded, st));
  return DDRL_OK;
}

extern "C" int ddrl_snap_get_weights(ddrl_snap_t *s, double *flat) {
  if (!s || !flat) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  ON_DEVICE(s);
  HIPCHK(hipDeviceSynchronize());
  static const double grid[16] = {0., .5, 1., 1.5, 2., 3., 4., 6., -0., -.5, -1., -1.5, -2., -3., -4., -6.};
  const SnapDesc &n = s->nd;
  try {
    const size_t at_once = std::max<size_t>(1, (64u << 20) / n.stride);
    std::vector<char> img(std::min<size_t>(at_once, s->G) * n.stride);
    for (size_t g0 = 0; g0 < (size_t)s->G; g0 += at_once) {
      const size_t cnt = std::min(at_once, s->G - g0);
      HIPCHK(hipMemcpy(img.data(), s->img + g0 * n.stride, cnt * n.stride, hipMemcpyDeviceToHost));
      for (size_t g = 0; g < cnt; ++g) {
        const char *im = img.data() + g * n.stride;
        double *f = flat + (g0 + g) * n.np;
        for (int l = 0; l < n.L; ++l) {
          const SnapLayer &y = n.lay[l];
          const int K = y.in, N = y.out;
          for (int o = 0; o < N; ++o)
            for (int k = 0; k < K; ++k) {
              const char *rec = im + y.off + (size_t)(o >> 4) * y.rec;
              const int r = o & 15;
              if (n.bits == 4) {
                unsigned c;
                memcpy(&c, rec + snap_code_off(y.steps, k >> 5, ((k >> 3) & 3) * 16 + r), 4);
                const unsigned char e = (unsigned char)rec[snap_scale_off(y.code, k >> 5, r)];
                *f++ = std::ldexp(grid[(c >> (4 * (k & 7))) & 15], (int)e - 127);
              } else {
                float v;
                memcpy(&v, rec + (k >> 4) * 1024 + ((((k >> 2) & 3) * 16 + r) * 4 + (k & 3)) * 4, 4);
                *f++ = v;
              }
            }
          for (int o = 0; o < N; ++o) { float v; memcpy(&v, im + y.off + (size_t)(o >> 4) * y.rec + y.rec - 64 + (o & 15) * 4, 4); *f++ = v; }
        }
      }
    }
  } catch (const std::bad_alloc &) {
    return ddrl_fail(DDRL_ENOMEM, "out of host memory");
  }
  return DDRL_OK;
}

static int check_rows(int n) {
  if (n < 0 || n > (1 << 28)) return ddrl_fail(DDRL_EINVAL, "n=%d: 0..%d", n, 1 << 28);
  return DDRL_OK;
}
static int forward_on(ddrl_snap *s, const ddrl_snap_forward_args *a, hipStream_t st) {
  if (check_rows(a->n)) return DDRL_EINVAL;
  if (a->n == 0) return DDRL_OK;
  if (!a->x || !a->out || off4(a->x) || off4(a->out)) return ddrl_fail(DDRL_EINVAL, "x / out NULL or misaligned");
  const int64_t S = s->nd.lay[0].in, A = s->nd.A, n = a->n, G = s->G;
  SnapForward p;
  p.G = s->G; p.n = a->n; p.per = 0; p.img = s->img;
  p.x = a->x; p.out = a->out; p.mask = a->mask;
  p.x_row = a->x_row == -1 ? S : a->x_row;
  p.x_agent = a->x_agent != -1 ? a->x_agent : p.x_row ? n * p.x_row : S;           // (x_row 0: an agent has one row)
  p.out_row = a->out_row == -1 ? A : a->out_row;
  p.out_agent = a->out_agent != -1 ? a->out_agent : p.out_row ? n * p.out_row : A;
  if (p.x_row < 0 || p.x_agent < 0) return ddrl_fail(DDRL_EINVAL, "negative stride of x");
  // rows of an agent one after the other and agents apart, or the agents of a row one after the other and rows apart
  const bool rows_in = (n == 1 || p.out_row >= A) && (G == 1 || p.out_agent >= (n - 1) * p.out_row + A);
  const bool agents_in = (G == 1 || p.out_agent >= A) && (n == 1 || p.out_row >= (G - 1) * p.out_agent + A);
  if (p.out_row < 0 || p.out_agent < 0 || !(rows_in || agents_in))
    return ddrl_fail(DDRL_EINVAL, "out_row=%lld, out_agent=%lld: rows of out overlap", (long long)p.out_row, (long long)p.out_agent);
  HIPCHK(snap_forward_launch(&s->nd, &p, st));
  return DDRL_OK;
}

extern "C" int ddrl_snap_forward_dev(ddrl_snap_t *s, const ddrl_snap_forward_args *a) {
  if (!s || !a) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  ON_DEVICE(s);
  return forward_on(s, a, (hipStream_t)a->stream);
}

extern "C" int ddrl_snap_forward(ddrl_snap_t *s, int n, const float *x, float *out) {
  if (!s || (n && (!x || !out))) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  if (check_rows(n)) return DDRL_EINVAL;
  if (n == 0) return DDRL_OK;
  ON_DEVICE(s);
  const size_t nx = (size_t)s->G * n * s->nd.lay[0].in * 4, no = (size_t)s->G * n * s->nd.A * 4;
  DevBuf b;
  if (b.get(up16(nx) + no) != hipSuccess) return ddrl_fail(DDRL_ENOMEM, "hipMalloc failed");
  ddrl_snap_forward_args a = {};
  a.n = n; a.x = (const float *)b.p; a.out = (float *)(b.p + up16(nx));
  a.x_agent = a.x_row = a.out_agent = a.out_row = -1;
  HIPCHK(hipStreamWaitEvent(s->stream, s->loaded, 0));
  HIPCHK(hipMemcpyAsync(b.p, x, nx, hipMemcpyHostToDevice, s->stream));
  int rc = forward_on(s, &a, s->stream);
  hipError_t e = hipSuccess;
  if (!rc) e = hipMemcpyAsync(out, a.out, no, hipMemcpyDeviceToHost, s->stream);
  const hipError_t e2 = hipStreamSynchronize(s->stream);
  if (!rc && (e != hipSuccess || e2 != hipSuccess)) rc = ddrl_fail(DDRL_EHIP, "snap_forward: %s", hipGetErrorString(e != hipSuccess ? e : e2));
  return rc;
}

extern "C" int ddrl_snap_mixture_workspace(ddrl_snap_t *s, int n, int top_k, size_t *bytes) {
  if (!s || !bytes) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  int rc = check_mix_shape(s, n, top_k);
  if (!rc) *bytes = mix_space(s, n, top_k).all;
  return rc;
}

static int mixture_on(ddrl_snap *s, const ddrl_snap_mixture_args *a, hipStream_t st) {
  int rc = check_mix_shape(s, a->n, a->top_k);
  if (rc || a->n == 0) return rc;
  if (!a->x || !a->router_w || !a->out || off4(a->x) || off4(a->router_w) || off4(a->out) || off4(a->router_b) || off4(a->idx) ||
      off4(a->prob) || off4(a->y))
    return ddrl_fail(DDRL_EINVAL, "x, router_w or out NULL, or a misaligned pointer");
  const MixSpace w = mix_space(s, a->n, a->top_k);
  if (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < w.all)
    return ddrl_fail(DDRL_EINVAL, "workspace NULL, misaligned or under the %zu bytes of ddrl_snap_mixture_workspace", w.all);
  const int S = s->nd.lay[0].in, A = s->nd.A;
  SnapMixture p;
  p.G = s->G; p.n = a->n; p.k = a->top_k; p.img = s->img;
  p.x = a->x; p.x_row = a->x_row == -1 ? S : a->x_row;
  p.rw = a->router_w; p.r_row = a->router_row == -1 ? S : a->router_row;
  p.rb = a->router_b;
  p.allowed = a->allowed; p.a_row = a->allowed_row == -1 ? s->G : a->allowed_row;
  p.out = a->out; p.out_row = a->out_row == -1 ? A : a->out_row;
  if (p.x_row < 0 || p.r_row < 0 || p.a_row < 0) return ddrl_fail(DDRL_EINVAL, "negative stride");
  if (p.out_row < 0 || (a->n > 1 && p.out_row < A)) return ddrl_fail(DDRL_EINVAL, "out_row=%lld: rows of out overlap", (long long)p.out_row);
  char *ws = (char *)a->workspace;
  p.count = (int *)(ws + w.count);
  p.idx = a->idx ? a->idx : (int *)(ws + w.idx);
  p.prob = a->prob ? a->prob : (float *)(ws + w.prob);
  p.y = a->y ? a->y : (float *)(ws + w.y);
  p.ckey = (unsigned long long *)(ws + w.ckey); p.cidx = (int *)(ws + w.cidx); p.chunks = w.chunks;
  p.sorted = (int *)(ws + w.sorted); p.start = (int *)(ws + w.start); p.blocks = w.blocks;
  HIPCHK(snap_mixture_launch(&s->nd, &p, st));
  return DDRL_OK;
}

extern "C" int ddrl_snap_mixture_dev(ddrl_snap_t *s, const ddrl_snap_mixture_args *a) {
  if (!s || !a) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  ON_DEVICE(s);
  return mixture_on(s, a, (hipStream_t)a->stream);
}

extern "C" int ddrl_snap_mixture(ddrl_snap_t *s, int n, int top_k, const float *x, const float *router_w, const float *router_b,
                                 const uint8_t *allowed, float *out, int32_t *idx, float *prob) {
  if (!s || !router_w || (n > 0 && (!x || !out))) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  int rc = check_mix_shape(s, n, top_k);
  if (rc || n == 0) return rc;
  ON_DEVICE(s);
  const size_t S = s->nd.lay[0].in, A = s->nd.A, G = s->G, places = (size_t)n * top_k;
  const size_t sizes[8] = {n * S * 4, G * S * 4, router_b ? G * 4 : 0, allowed ? n * G : 0, n * A * 4, places * 4, places * 4, mix_space(s, n, top_k).all};
  size_t at[9] = {0};
  for (int i = 0; i < 8; ++i) at[i + 1] = at[i] + up16(sizes[i]);
  DevBuf b;
  if (b.get(at[8]) != hipSuccess) return ddrl_fail(DDRL_ENOMEM, "hipMalloc failed");
  ddrl_snap_mixture_args a = {};
  a.n = n; a.top_k = top_k;
  a.x_row = a.router_row = a.allowed_row = a.out_row = -1;
  a.x = (const float *)b.p; a.router_w = (const float *)(b.p + at[1]);
  a.router_b = router_b ? (const float *)(b.p + at[2]) : nullptr;
  a.allowed = allowed ? (const uint8_t *)(b.p + at[3]) : nullptr;
  a.out = (float *)(b.p + at[4]); a.idx = (int32_t *)(b.p + at[5]); a.prob = (float *)(b.p + at[6]);
  a.workspace = b.p + at[7]; a.workspace_bytes = sizes[7];
  const hipStream_t st = s->stream;
  HIPCHK(hipStreamWaitEvent(st, s->loaded, 0));
  hipError_t e = hipMemcpyAsync(b.p, x, sizes[0], hipMemcpyHostToDevice, st);
  if (e == hipSuccess) e = hipMemcpyAsync(b.p + at[1], router_w, sizes[1], hipMemcpyHostToDevice, st);
  if (e == hipSuccess && router_b) e = hipMemcpyAsync(b.p + at[2], router_b, sizes[2], hipMemcpyHostToDevice, st);
  if (e == hipSuccess && allowed) e = hipMemcpyAsync(b.p + at[3], allowed, sizes[3], hipMemcpyHostToDevice, st);
  if (e == hipSuccess) rc = mixture_on(s, &a, st);
  if (e == hipSuccess && !rc) e = hipMemcpyAsync(out, a.out, sizes[4], hipMemcpyDeviceToHost, st);
  if (e == hipSuccess && !rc && idx) e = hipMemcpyAsync(idx, a.idx, sizes[5], hipMemcpyDeviceToHost, st);
  if (e == hipSuccess && !rc && prob) e = hipMemcpyAsync(prob, a.prob, sizes[6], hipMemcpyDeviceToHost, st);
  const hipError_t e2 = hipStreamSynchronize(st);
  if (!rc && (e != hipSuccess || e2 != hipSuccess)) rc = ddrl_fail(DDRL_EHIP, "snap_mixture: %s", hipGetErrorString(e != hipSuccess ? e : e2));
  return rc;
}

extern "C" int ddrl_snap_mixture_grad_workspace(ddrl_snap_t *s, int n, int top_k, size_t *bytes) {
  if (!s || !bytes) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  int rc = check_mix_shape(s, n, top_k);
  if (!rc) *bytes = grad_space(s, n, top_k).all;
  return rc;
}

extern "C" int ddrl_snap_mixture_grad_dev(ddrl_snap_t *s, const ddrl_snap_mixture_grad_args *a) {
  if (!s || !a) return ddrl_fail(DDRL_EINVAL, "NULL argument");
  int rc = check_mix_shape(s, a->n, a->top_k);
  if (rc) return rc;
  if (!a->d_router_w || off4(a->d_router_w) || off4(a->d_router_b) || off4(a->dy)) return ddrl_fail(DDRL_EINVAL, "d_router_w NULL, or a misaligned pointer");
  if (a->n && (!a->x || !a->idx || !a->prob || !a->y || !a->dout || off4(a->x) || off4(a->idx) || off4(a->prob) || off4(a->y) || off4(a->dout)))
    return ddrl_fail(DDRL_EINVAL, "x, idx, prob, y or dout NULL or misaligned");
  SnapGrad p;
  p.G = s->G; p.n = a->n; p.k = a->top_k; p.S = s->nd.lay[0].in; p.A = s->nd.A;
  p.x = a->x; p.x_row = a->x_row == -1 ? p.S : a->x_row;
  p.idx = a->idx; p.prob = a->prob; p.y = a->y;
  p.dout = a->dout; p.dout_row = a->dout_row == -1 ? p.A : a->dout_row;
  p.dw = a->d_router_w; p.dw_row = a->d_router_row == -1 ? p.S : a->d_router_row;
  p.db = a->d_router_b; p.dy = a->dy;
  if (p.x_row < 0 || p.dout_row < 0) return ddrl_fail(DDRL_EINVAL, "negative stride");
  if (p.dw_row < 0 || (p.G > 1 && p.dw_row < p.S)) return ddrl_fail(DDRL_EINVAL, "d_router_row=%lld: rows of d_router_w overlap", (long long)p.dw_row);
  const GradSpace w = grad_space(s, a->n, a->top_k);
  if (w.all && (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < w.all))
    return ddrl_fail(DDRL_EINVAL, "workspace NULL, misaligned or under the %zu bytes of ddrl_snap_mixture_grad_workspace", w.all);
  char *ws = (char *)a->workspace;
  p.blocks = w.blocks;
  p.sorted = w.blocks ? (int *)(ws + w.sorted) : nullptr;
  p.start = w.blocks ? (int *)(ws + w.start) : nullptr;
  p.dlogit = w.blocks ? (float *)(ws + w.dlogit) : nullptr;
  p.done = (int *)(ws + w.done);
  p.sums = w.pieces > 1 ? (double *)(ws + w.sums) : nullptr;
  p.piece = 0;
  ON_DEVICE(s);
  HIPCHK(snap_grad_launch(&p, w.pieces, (hipStream_t)a->stream));
  return DDRL_OK;
}
