// MI355X (gfx950) kernels + C ABI of the gated linear recurrence over time.
//
//   z_t = sigmoid(gate_t), f_t = 1 - z_t = sigmoid(-gate_t)
//   h_t = f_t h_{t-1} + z_t v_t                                     t = 0 .. len - 1
// and, for a loss with gradients dh_t of the outputs and dl of the last state,
//   e_t = dh_t + p_t      p_{len-1} = dl,  p_{t-1} = f_t e_t        (backwards in time)
//   dvalue_t = z_t e_t    dgate_t = z_t f_t (v_t - h_{t-1}) e_t     dstate = p_{-1}
// The update is the GRU's (the reference's temporal cell, tempo/models/fiery_temporal.py:109)
// with gates that depend on the input alone, which makes the recurrence linear in h and lets
// time be cut into chunks.
//
// What bounds it: memory.  Forward reads gate and value and writes h; backward reads gate,
// value and dh and writes two gradients.  h is not kept for the backward pass: the forward
// stores the fp32 state in front of every kSpan-th step, and the backward recomputes a span's
// states in registers from there (less to read than h itself, and not rounded to 16 bits).
//
// Where there are too few (b, d) lanes to fill the card, time is cut into chunks.  A chunk of
// the forward maps its incoming state to  h_out = A h_in + U,  A = prod f: pass 1 computes
// (A, U) of every chunk, pass 2 scans them over the chunks, pass 3 runs each chunk from its
// incoming state.  The backward does the same with p, in the other direction.
//
// Rounding.  Everything between the loads and the stores is fp32.  With w = min(z, f) the
// step is taken as  base + w (other - base)  with base the operand of the larger weight (16-bit
// tensors: as  h + z (v - h)): z + f = 1 holds exactly, so a gate that stays nearly shut for
// thousands of steps does not drift, which f h + z v with separately rounded f and z does.  A
// chunk's A is kept as S = 1 - A while S < 1/2 for the same reason (encoded as +S, otherwise
// as -A).
//
// Values and states are taken from each other: a difference beyond fp32's range overflows.
//
// Measured (rates of a large copy on the same card: 4.8 TB/s, of a large sum 4.0 TB/s): where
// lanes fill the card, one pass each, 153600 x 4 x 32 in fp32 forward 54 us (4.8 TB/s),
// backward 73 us (5.4 TB/s).  Cut in time, the inputs are read twice: 1 x 65536 x 1024 in bf16
// 77 + 14 + 75 us (3.6 and 5.4 TB/s of what the two passes move).  One pass would need
// workgroups that wait for each other; re-reading is what it costs not to.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tempo_unproject.h"

namespace {

constexpr int kBlock = 256;
constexpr int kSpan = TEMPO_RECURRENCE_SPAN;
constexpr int kBatch = 8;          // steps loaded at a time; divides kSpan
constexpr int kScanLanes = 16;     // pass 2: lanes x segments of a workgroup
constexpr int kScanSegments = 64;

template <typename T, int V>
struct Pack {
  // element-aligned: rows of odd width start anywhere
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

struct RecurrenceArgs {
  const void *gate, *value;       // element (b, t, d) at b * sb + t * st + d
  const void* grad_h;             // backward
  void *out, *out2;               // forward: h; backward: dgate, dvalue
  const float* state;             // forward: h_{-1}; backward: dl.  [B, D] or NULL (zeros)
  const int32_t* lengths;         // [B] or NULL
  const float* ckpt_in;           // backward: [ceil(T / kSpan)][B * D] or NULL (zeros)
  float* ckpt;                    // forward: the same, or NULL
  float* last;                    // forward: last state; backward: dstate.  [B, D] or NULL
  float *weight, *carry;          // chunked: [nchunk][lanes * V]
  long long gate_sb, gate_st, value_sb, value_st, grad_sb, grad_st;
  long long out_sb, out_st, out2_sb, out2_st;
  uint32_t B, T, D, DV;           // DV = vector lanes per row
  uint32_t lanes, chunk, nchunk;  // lanes = B * DV
};

// One thread's place: V neighbouring channels of one batch row, one chunk of time.  Where V
// does not divide D, the last lane of a row moves back so that its V channels are inside the
// row, too: it shares `skip` of them with its neighbour and stores the others alone (a lane
// that loaded its few channels one by one would hold up its wave: 294 against 92 us for the
// backward pass of 13 x 4097 x 771 in fp16).
// Rows of fewer than V channels (n < V) go channel by channel.
template <int V>
struct Place {
  uint32_t lane, b, d, n, c, skip;
  bool on;
  __device__ Place(const RecurrenceArgs& a) {
    const uint32_t id = blockIdx.x * kBlock + threadIdx.x;
    on = id < a.lanes * a.nchunk;
    c = id / a.lanes;
    lane = id - c * a.lanes;
    b = lane / a.DV;
    const uint32_t first = (lane - b * a.DV) * V;
    n = min((uint32_t)V, a.D);
    d = min(first, a.D - n);
    skip = first - d;
  }
};

// V channels as they lie in memory; FULL: all of them are inside the row
template <bool FULL, int V, typename T>
__device__ __forceinline__ typename Pack<T, V>::type fetch(const T* p, uint32_t n) {
  if constexpr (FULL) return *reinterpret_cast<const typename Pack<T, V>::type*>(p);
  typename Pack<T, V>::type r;
#pragma unroll
  for (int j = 0; j < V; ++j) r[j] = (uint32_t)j < n ? p[j] : (T)0.f;
  return r;
}

template <int V>
__device__ __forceinline__ void load(const float* p, uint32_t n, float (&x)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = (uint32_t)j < n ? p[j] : 0.f;
}

template <bool FULL, int V, typename T>
__device__ __forceinline__ void put(T* p, const Place<V>& at, const float (&x)[V]) {
  if (FULL && at.skip == 0) {
    typename Pack<T, V>::type r;
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (T)x[j];
    *reinterpret_cast<typename Pack<T, V>::type*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if ((uint32_t)j >= at.skip && (uint32_t)j < at.n) p[j] = (T)x[j];
  }
}

// w = min(z, f) = e^-|g| / (1 + e^-|g|); z is the smaller one where g < 0.  A NaN stays one.
template <typename T>
__device__ __forceinline__ float small_weight(float g) {
  if constexpr (sizeof(T) == 4) {
    const float e = expf(-fabsf(g));
    const float y = 1.f + e;
    float r = __builtin_amdgcn_rcpf(y);
    r = fmaf(fmaf(-y, r, 1.f), r, r);  // one Newton step: v_rcp_f32 is good to one ulp
    return e * r;
  } else {
    const float e = __builtin_amdgcn_exp2f(-fabsf(g) * 1.44269504088896341f);
    return e * __builtin_amdgcn_rcpf(1.f + e);
  }
}

__device__ __forceinline__ float step(float w, bool shut, float h, float v) {
  const float base = shut ? h : v, other = shut ? v : h;
  return fmaf(w, other - base, base);
}

// One step's gate.  summarize: one more step of a chunk's A = k and S = 1 - A = s, each to its
// own full precision.
template <typename T>
struct Gate;
template <>
struct Gate<float> {
  float w;
  bool shut;
  __device__ __forceinline__ explicit Gate(float g) : w(small_weight<float>(g)), shut(g < 0.f) {}
  __device__ __forceinline__ float step(float h, float v) const {
    const float base = shut ? h : v, other = shut ? v : h;
    return fmaf(w, other - base, base);
  }
  __device__ __forceinline__ float back(float x) const {
    const float wx = w * x;
    return shut ? x - wx : wx;
  }
  __device__ __forceinline__ void summarize(float* s, float* k) const {
    const float rest = 1.f - w;
    *s = fmaf(shut ? w : rest, *k, *s);
    *k *= shut ? rest : w;
  }
};
// 16-bit tensors: z and f from one exponential, no choice between them (backward summary of
// 8 x 2048 x 1024: 20.4 -> 15.6 us).  h + z (v - h) does not drift either; what it gives up is
// an open gate's exactness to the last of 24 bits.
template <typename T>
struct Gate {
  float z, f;
  __device__ __forceinline__ explicit Gate(float g) {
    float a = 1.44269504088896341f * g;
    a = a > 126.f ? 126.f : a;  // z below: no infinity times 0; a NaN passes
    const float e = __builtin_amdgcn_exp2f(a);
    f = __builtin_amdgcn_rcpf(1.f + e);
    z = e * f;  // 0 where the gate is shut for good: the value may be the type's largest there
  }
  __device__ __forceinline__ float step(float h, float v) const { return fmaf(z, v - h, h); }
  __device__ __forceinline__ float back(float x) const { return f * x; }
  __device__ __forceinline__ void summarize(float* s, float* k) const {
    *s = fmaf(z, *k, *s);
    *k *= f;
  }
};

// h_out of a chunk (or of several) from its incoming state
__device__ __forceinline__ float apply(float weight, float u, float h) {
  return (__float_as_uint(weight) >> 31) ? fmaf(-weight, h, u) : fmaf(-weight, h, h) + u;
}

__device__ __forceinline__ float kept(float weight) {  // A
  return (__float_as_uint(weight) >> 31) ? -weight : 1.f - weight;
}

// first `one`, then `two`
__device__ __forceinline__ float chain(float one, float two) {
  if (!((__float_as_uint(one) | __float_as_uint(two)) >> 31)) {
    const float s = fmaf(two, 1.f - one, one);
    return s < 0.5f ? s : -(1.f - s);
  }
  return -(kept(one) * kept(two));
}

__device__ __forceinline__ uint32_t length_of(const RecurrenceArgs& a, uint32_t b) {
  if (!a.lengths) return a.T;
  const int32_t n = a.lengths[b];
  return n < 0 ? 0u : min((uint32_t)n, a.T);
}

template <int V>
__device__ __forceinline__ void load_state(const float* p, const RecurrenceArgs& a, uint32_t b,
                                           uint32_t d, uint32_t n, float (&x)[V]) {
  if (p) {
    load<V>(p + (size_t)b * a.D + d, n, x);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = 0.f;
  }
}

// ------------------------------------------------------------------------------- forward

// kBatch steps of two streams.  (Loading a batch ahead changed nothing: other waves fill the
// gaps.)  Steps missing from a chunk's last batch are left out in 16 bits (31164 x 1 x 1072: 127
// us, 169 with the last step loaded in their place); in fp32, where one step is more of the time
// (102 against 106), that costs registers and with them a third of the waves (8 x 8192 x 1024: 345
// against 333), so there they are the last step again.
template <typename T, int V>
struct Batch {
  typename Pack<T, V>::type a[kBatch], b[kBatch];
  template <bool FULL>
  __device__ __forceinline__ void load(const T* pa, long long sa, const T* pb, long long sb,
                                       uint32_t i, uint32_t steps, uint32_t n) {
    pa += i * sa;
    pb += i * sb;
    if (i + kBatch <= steps) {
#pragma unroll
      for (int q = 0; q < kBatch; ++q, pa += sa, pb += sb) {
        a[q] = fetch<FULL, V>(pa, n);
        b[q] = fetch<FULL, V>(pb, n);
      }
    } else {
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        if (sizeof(T) == 2 && i + q >= steps) break;
        const uint32_t t = min((uint32_t)q, steps - 1 - i);
        a[q] = fetch<FULL, V>(pa + t * sa, n);
        b[q] = fetch<FULL, V>(pb + t * sb, n);
      }
    }
  }
};

template <bool FULL, typename T, int V>
__device__ __forceinline__ void forward_summary(const RecurrenceArgs& a, const Place<V>& at) {
  const uint32_t begin = at.c * a.chunk;
  const uint32_t end = min(begin + a.chunk, length_of(a, at.b));
  const uint32_t steps = end > begin ? end - begin : 0;
  const T* pg = (const T*)a.gate + (at.b * a.gate_sb + begin * a.gate_st + at.d);
  const T* pv = (const T*)a.value + (at.b * a.value_sb + begin * a.value_st + at.d);
  float s[V], k[V], u[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = u[j] = 0.f, k[j] = 1.f;
  for (uint32_t i = 0; i < steps; i += kBatch) {
    Batch<T, V> x;
    x.template load<FULL>(pg, a.gate_st, pv, a.value_st, i, steps, at.n);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (i + q < steps) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const Gate<T> gate((float)x.a[q][j]);
          u[j] = gate.step(u[j], (float)x.b[q][j]);
          gate.summarize(&s[j], &k[j]);
        }
      }
    }
  }
  const size_t o = ((size_t)at.c * a.lanes + at.lane) * V;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.weight[o + j] = s[j] < 0.5f ? s[j] : -k[j];
    a.carry[o + j] = u[j];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void forward_summary_kernel(const RecurrenceArgs a) {
  const Place<V> at(a);
  if (!at.on) return;
  if (at.n == V) forward_summary<true, T, V>(a, at);
  else forward_summary<false, T, V>(a, at);
}

// Pass 2 of both directions: chunk summaries -> every chunk's incoming value (over `carry`)
// and the value behind the last one.  A workgroup holds kScanLanes lanes and cuts their
// chunks into kScanSegments runs: fold each run, chain the runs, walk each run again.
template <bool REVERSE, int V>
__global__ __launch_bounds__(kScanLanes* kScanSegments) void scan_kernel(const RecurrenceArgs a) {
  __shared__ float s_weight[kScanSegments][kScanLanes], s_u[kScanSegments][kScanLanes];
  const uint32_t l = threadIdx.x % kScanLanes, seg = threadIdx.x / kScanLanes;
  const uint32_t width = a.lanes * V;
  const uint32_t q = blockIdx.x * kScanLanes + l;
  const uint32_t lane = q / V, b = lane / a.DV, d0 = (lane - b * a.DV) * V;
  const uint32_t moved = d0 - min(d0, a.D - min((uint32_t)V, a.D));  // see Place
  const uint32_t d = d0 - moved + q % V;
  const bool on = q < width && q % V >= moved && d < a.D;
  const uint32_t run = (a.nchunk + kScanSegments - 1) / kScanSegments;
  const uint32_t first = min(seg * run, a.nchunk), stop = min(first + run, a.nchunk);
  float weight = 0.f, u = 0.f;
  float h = on && a.state ? a.state[(size_t)b * a.D + d] : 0.f;
  if (on) {
#pragma unroll 8
    for (uint32_t i = first; i < stop; ++i) {
      const size_t o = (size_t)(REVERSE ? a.nchunk - 1 - i : i) * width + q;
      const float w = a.weight[o], c = a.carry[o];
      weight = chain(weight, w);
      u = apply(w, c, u);
    }
  }
  s_weight[seg][l] = weight;
  s_u[seg][l] = u;
  __syncthreads();
  if (!on) return;
#pragma unroll 8
  for (uint32_t i = 0; i < seg; ++i) h = apply(s_weight[i][l], s_u[i][l], h);
#pragma unroll 8
  for (uint32_t i = first; i < stop; ++i) {
    const size_t o = (size_t)(REVERSE ? a.nchunk - 1 - i : i) * width + q;
    const float w = a.weight[o], c = a.carry[o];
    a.carry[o] = h;
    h = apply(w, c, h);
  }
  if (seg == kScanSegments - 1 && a.last) a.last[(size_t)b * a.D + d] = h;
}

template <bool FULL, typename T, int V>
__device__ __forceinline__ void forward_chunk(const RecurrenceArgs& a, const Place<V>& at) {
  const uint32_t begin = at.c * a.chunk, stop = min(begin + a.chunk, a.T);
  const uint32_t end = max(begin, min(stop, length_of(a, at.b)));
  const uint32_t steps = end - begin, all = stop - begin;
  const T* pg = (const T*)a.gate + (at.b * a.gate_sb + begin * a.gate_st + at.d);
  const T* pv = (const T*)a.value + (at.b * a.value_sb + begin * a.value_st + at.d);
  T* ph = (T*)a.out + (at.b * a.out_sb + begin * a.out_st + at.d);
  const size_t row = (size_t)at.b * a.D + at.d, width = (size_t)a.B * a.D;
  float* ckpt = a.ckpt ? a.ckpt + (begin / kSpan) * width + row : nullptr;
  float h[V];
  if (a.nchunk > 1)
    load<V>(a.carry + ((size_t)at.c * a.lanes + at.lane) * V, V, h);
  else
    load_state<V>(a.state, a, at.b, at.d, at.n, h);
  for (uint32_t i = 0; i < steps; i += kBatch) {
    Batch<T, V> x;
    x.template load<FULL>(pg, a.gate_st, pv, a.value_st, i, steps, at.n);
    if (ckpt && i % kSpan == 0) {
      put<FULL, V>(ckpt, at, h);
      ckpt += width;
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (i + q < steps) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[j] = Gate<T>((float)x.a[q][j]).step(h[j], (float)x.b[q][j]);
        }
        put<FULL, V>(ph + (i + q) * a.out_st, at, h);
      }
    }
  }
  if (a.nchunk == 1 && a.last) put<FULL, V>(a.last + row, at, h);
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = 0.f;
  for (uint32_t i = steps; i < all; ++i) put<FULL, V>(ph + i * a.out_st, at, h);
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void forward_kernel(const RecurrenceArgs a) {
  const Place<V> at(a);
  if (!at.on) return;
  if (at.n == V) forward_chunk<true, T, V>(a, at);
  else forward_chunk<false, T, V>(a, at);
}

// ------------------------------------------------------------------------------ backward

template <bool FULL, typename T, int V>
__device__ __forceinline__ void backward_summary(const RecurrenceArgs& a, const Place<V>& at) {
  const uint32_t begin = at.c * a.chunk;
  const uint32_t end = max(begin, min(begin + a.chunk, length_of(a, at.b)));
  const uint32_t steps = end - begin;
  // from the last step of the chunk back
  const long long from = (long long)end - 1;
  const T* pg = (const T*)a.gate + (at.b * a.gate_sb + from * a.gate_st + at.d);
  const T* pe = (const T*)a.grad_h + (at.b * a.grad_sb + from * a.grad_st + at.d);
  float s[V], k[V], p[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = p[j] = 0.f, k[j] = 1.f;
  for (uint32_t i = 0; i < steps; i += kBatch) {
    Batch<T, V> x;
    x.template load<FULL>(pg, -a.gate_st, pe, -a.grad_st, i, steps, at.n);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (i + q < steps) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const Gate<T> gate((float)x.a[q][j]);
          p[j] = gate.back((float)x.b[q][j] + p[j]);
          gate.summarize(&s[j], &k[j]);
        }
      }
    }
  }
  const size_t o = ((size_t)at.c * a.lanes + at.lane) * V;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.weight[o + j] = s[j] < 0.5f ? s[j] : -k[j];
    a.carry[o + j] = p[j];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void backward_summary_kernel(const RecurrenceArgs a) {
  const Place<V> at(a);
  if (!at.on) return;
  if (at.n == V) backward_summary<true, T, V>(a, at);
  else backward_summary<false, T, V>(a, at);
}

// A span of C steps: recompute its states from the checkpoint, keep per step w (negative
// where the gate is open) and z f (v - h); then walk it back.
template <bool FULL, bool WHOLE, typename T, int V, int C>
__device__ __forceinline__ void backward_span(const RecurrenceArgs& a, const Place<V>& at,
                                              uint32_t t0, uint32_t steps, const T* pg,
                                              const T* pv, const T* pe, T* pdg, T* pdv,
                                              float (&p)[V]) {
  typename Pack<T, V>::type g[C], v[C], e[C];
  const uint32_t last = WHOLE ? C - 1 : steps - 1;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const uint32_t t = WHOLE ? k : min((uint32_t)k, last);
    g[k] = fetch<FULL, V>(pg + t * a.gate_st, at.n);
    v[k] = fetch<FULL, V>(pv + t * a.value_st, at.n);
  }
  float w[C][V], r[C][V], h[V];
  if (a.ckpt_in) {
    const size_t row = (size_t)at.b * a.D + at.d, width = (size_t)a.B * a.D;
    load<V>(a.ckpt_in + (t0 / kSpan) * width + row, at.n, h);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const uint32_t t = WHOLE ? k : min((uint32_t)k, last);
    e[k] = fetch<FULL, V>(pe + t * a.grad_st, at.n);
  }
#pragma unroll
  for (int k = 0; k < C; ++k) {
    if (WHOLE || (uint32_t)k < steps) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float y = (float)g[k][j], x = small_weight<T>(y), z = (float)v[k][j];
        const bool shut = y < 0.f;
        w[k][j] = shut ? x : -x;
        r[k][j] = (x - x * x) * (z - h[j]);
        h[j] = step(x, shut, h[j], z);
      }
    }
  }
#pragma unroll
  for (int k = C - 1; k >= 0; --k) {
    if (WHOLE || (uint32_t)k < steps) {
      float dg[V], dv[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = (float)e[k][j] + p[j], wx = fabsf(w[k][j]) * x;
        const bool shut = !(__float_as_uint(w[k][j]) >> 31);
        dg[j] = r[k][j] * x;
        dv[j] = shut ? wx : x - wx;
        p[j] = shut ? x - wx : wx;
      }
      put<FULL, V>(pdg + k * a.out_st, at, dg);
      put<FULL, V>(pdv + k * a.out2_st, at, dv);
    }
  }
}

template <bool FULL, typename T, int V, int C>
__device__ __forceinline__ void backward_chunk(const RecurrenceArgs& a, const Place<V>& at) {
  const uint32_t begin = at.c * a.chunk, stop = min(begin + a.chunk, a.T);
  const uint32_t end = max(begin, min(stop, length_of(a, at.b)));
  const T* pg = (const T*)a.gate + (at.b * a.gate_sb + begin * a.gate_st + at.d);
  const T* pv = (const T*)a.value + (at.b * a.value_sb + begin * a.value_st + at.d);
  const T* pe = (const T*)a.grad_h + (at.b * a.grad_sb + begin * a.grad_st + at.d);
  T* pdg = (T*)a.out + (at.b * a.out_sb + begin * a.out_st + at.d);
  T* pdv = (T*)a.out2 + (at.b * a.out2_sb + begin * a.out2_st + at.d);
  float p[V];
#pragma unroll
  for (int j = 0; j < V; ++j) p[j] = 0.f;
  for (uint32_t i = end - begin; i < stop - begin; ++i) {
    put<FULL, V>(pdg + i * a.out_st, at, p);
    put<FULL, V>(pdv + i * a.out2_st, at, p);
  }
  if (a.nchunk > 1)
    load<V>(a.carry + ((size_t)at.c * a.lanes + at.lane) * V, V, p);
  else
    load_state<V>(a.state, a, at.b, at.d, at.n, p);
  const uint32_t steps = end - begin, rest = steps % C;
  uint32_t i = steps - rest;
  if (rest)
    backward_span<FULL, false, T, V, C>(a, at, begin + i, rest, pg + i * a.gate_st,
                                        pv + i * a.value_st, pe + i * a.grad_st,
                                        pdg + i * a.out_st, pdv + i * a.out2_st, p);
  while (i > 0) {
    i -= C;
    backward_span<FULL, true, T, V, C>(a, at, begin + i, C, pg + i * a.gate_st,
                                       pv + i * a.value_st, pe + i * a.grad_st,
                                       pdg + i * a.out_st, pdv + i * a.out2_st, p);
  }
  if (a.nchunk == 1 && a.last) put<FULL, V>(a.last + (size_t)at.b * a.D + at.d, at, p);
}

template <typename T, int V, int C>
__global__ __launch_bounds__(kBlock) void backward_kernel(const RecurrenceArgs a) {
  const Place<V> at(a);
  if (!at.on) return;
  if (at.n == V) backward_chunk<true, T, V, C>(a, at);
  else backward_chunk<false, T, V, C>(a, at);
}

// --------------------------------------------------------------------------------- host

struct Plan {
  int vec;
  uint32_t lanes, DV, chunk, nchunk;
};

// Threads hold 4 channels; the backward beyond 4 steps 2, for its registers hold a span of
// fp32 values (8 x 2048 x 1024 in bf16: 34 us against 42 with 4, 256 registers).  Time is cut
// only where the (b, d) lanes alone are fewer than kFill threads: 16 waves for each of the 256
// compute units, 4 for each of their SIMDs.  Sums of the kernels' times with a quarter of that,
// half, as it is and twice, in us: 8 x 2048 x 1024 in bf16 trained 140, 112, 109, 110; forward of
// 1 x 65536 x 1024 187, 154, 164, 162.
constexpr uint32_t kFill = 1u << 18;
constexpr uint32_t kMinChunk = 2 * kSpan;

bool make_plan(long long B, int T, int D, bool backward, Plan* p) {
  p->vec = backward && T > 4 ? 2 : 4;
  p->DV = (uint32_t)((D + p->vec - 1) / p->vec);
  const long long lanes = B * p->DV;
  if (lanes > 0x7fffffffLL) return false;
  p->lanes = (uint32_t)lanes;
  uint32_t want = kFill / p->lanes;
  const uint32_t most = ((uint32_t)T + kMinChunk - 1) / kMinChunk;
  if (want > most) want = most;
  if (want < 2) {
    p->chunk = (uint32_t)T;
    p->nchunk = 1;
    return true;
  }
  const uint32_t chunk = ((uint32_t)T + want - 1) / want;
  p->chunk = (chunk + kSpan - 1) / kSpan * kSpan;
  p->nchunk = ((uint32_t)T + p->chunk - 1) / p->chunk;
  return true;
}

long long plan_bytes(const Plan& p) {
  return p.nchunk < 2 ? 0 : 2ll * p.nchunk * p.lanes * p.vec * 4;
}

int check_sizes(long long B, int T, int D, int dtype) {
  if (B <= 0 || T <= 0 || D <= 0) return TEMPO_E_DIM;
  if (dtype != TEMPO_DTYPE_F32 && dtype != TEMPO_DTYPE_F16 && dtype != TEMPO_DTYPE_BF16)
    return TEMPO_E_ARG;
  if (B > 0x7fffffffLL || D > 0x3fffffff || T > 0x3fffffff) return TEMPO_E_SIZE;
  return TEMPO_OK;
}

bool misaligned(const void* p, int dtype) {
  return ((uintptr_t)p & (dtype == TEMPO_DTYPE_F32 ? 3 : 1)) != 0;
}

template <typename T, int V>
int launch_forward(const RecurrenceArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(((unsigned long long)a.lanes * a.nchunk + kBlock - 1) / kBlock));
  if (a.nchunk > 1) {
    hipLaunchKernelGGL((forward_summary_kernel<T, V>), grid, dim3(kBlock), 0, stream, a);
    const dim3 scan((a.lanes * V + kScanLanes - 1) / kScanLanes);
    hipLaunchKernelGGL((scan_kernel<false, V>), scan, dim3(kScanLanes * kScanSegments), 0, stream,
                       a);
  }
  hipLaunchKernelGGL((forward_kernel<T, V>), grid, dim3(kBlock), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T, int V, int C>
int launch_backward(const RecurrenceArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(((unsigned long long)a.lanes * a.nchunk + kBlock - 1) / kBlock));
  if (a.nchunk > 1) {
    hipLaunchKernelGGL((backward_summary_kernel<T, V>), grid, dim3(kBlock), 0, stream, a);
    const dim3 scan((a.lanes * V + kScanLanes - 1) / kScanLanes);
    hipLaunchKernelGGL((scan_kernel<true, V>), scan, dim3(kScanLanes * kScanSegments), 0, stream,
                       a);
  }
  hipLaunchKernelGGL((backward_kernel<T, V, C>), grid, dim3(kBlock), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T>
int launch_backward_for(const RecurrenceArgs& a, int vec, hipStream_t stream) {
  if (vec == 4) return launch_backward<T, 4, 4>(a, stream);
  return launch_backward<T, 2, kSpan>(a, stream);
}

}  // namespace

extern "C" {

long long tempo_recurrence_workspace(long long B, int T, int D, int dtype, int backward) {
  const int rc = check_sizes(B, T, D, dtype);
  if (rc != TEMPO_OK) return rc;
  Plan p;
  if (!make_plan(B, T, D, backward != 0, &p)) return TEMPO_E_SIZE;
  return plan_bytes(p);
}

int tempo_recurrence(const void* gate, long long gate_sb, long long gate_st, const void* value,
                     long long value_sb, long long value_st, const float* state,
                     const int32_t* lengths, void* h, long long h_sb, long long h_st, float* last,
                     float* ckpt, long long B, int T, int D, int dtype, void* workspace,
                     long long workspace_bytes, void* stream) {
  if (!gate || !value || !h) return TEMPO_E_NULL;
  const int rc = check_sizes(B, T, D, dtype);
  if (rc != TEMPO_OK) return rc;
  Plan p;
  if (!make_plan(B, T, D, false, &p)) return TEMPO_E_SIZE;
  if (misaligned(gate, dtype) || misaligned(value, dtype) || misaligned(h, dtype))
    return TEMPO_E_ARG;
  const long long need = plan_bytes(p);
  if (need > 0 && !workspace) return TEMPO_E_NULL;
  if (need > workspace_bytes) return TEMPO_E_SIZE;
  if (((uintptr_t)workspace & 3) || ((uintptr_t)state & 3) || ((uintptr_t)last & 3) ||
      ((uintptr_t)ckpt & 3) || ((uintptr_t)lengths & 3))
    return TEMPO_E_ARG;
  RecurrenceArgs a = {};
  a.gate = gate; a.value = value; a.out = h; a.state = state; a.lengths = lengths;
  a.last = last; a.ckpt = ckpt;
  a.weight = (float*)workspace; a.carry = a.weight + (size_t)p.nchunk * p.lanes * p.vec;
  a.gate_sb = gate_sb; a.gate_st = gate_st; a.value_sb = value_sb; a.value_st = value_st;
  a.out_sb = h_sb; a.out_st = h_st;
  a.B = (uint32_t)B; a.T = (uint32_t)T; a.D = (uint32_t)D; a.DV = p.DV;
  a.lanes = p.lanes; a.chunk = p.chunk; a.nchunk = p.nchunk;
  if (dtype == TEMPO_DTYPE_F32) return launch_forward<float, 4>(a, (hipStream_t)stream);
  if (dtype == TEMPO_DTYPE_F16) return launch_forward<_Float16, 4>(a, (hipStream_t)stream);
  return launch_forward<__bf16, 4>(a, (hipStream_t)stream);
}

int tempo_recurrence_backward(const void* gate, long long gate_sb, long long gate_st,
                              const void* value, long long value_sb, long long value_st,
                              const void* grad_h, long long grad_sb, long long grad_st,
                              const float* grad_last, const int32_t* lengths, const float* ckpt,
                              void* grad_gate, long long dgate_sb, long long dgate_st,
                              void* grad_value, long long dvalue_sb, long long dvalue_st,
                              float* grad_state, long long B, int T, int D, int dtype,
                              void* workspace, long long workspace_bytes, void* stream) {
  if (!gate || !value || !grad_h || !grad_gate || !grad_value) return TEMPO_E_NULL;
  const int rc = check_sizes(B, T, D, dtype);
  if (rc != TEMPO_OK) return rc;
  if (!ckpt && T > kSpan) return TEMPO_E_NULL;
  Plan p;
  if (!make_plan(B, T, D, true, &p)) return TEMPO_E_SIZE;
  if (misaligned(gate, dtype) || misaligned(value, dtype) || misaligned(grad_h, dtype) ||
      misaligned(grad_gate, dtype) || misaligned(grad_value, dtype))
    return TEMPO_E_ARG;
  const long long need = plan_bytes(p);
  if (need > 0 && !workspace) return TEMPO_E_NULL;
  if (need > workspace_bytes) return TEMPO_E_SIZE;
  if (((uintptr_t)workspace & 3) || ((uintptr_t)grad_last & 3) || ((uintptr_t)ckpt & 3) ||
      ((uintptr_t)grad_state & 3) || ((uintptr_t)lengths & 3))
    return TEMPO_E_ARG;
  RecurrenceArgs a = {};
  a.gate = gate; a.value = value; a.grad_h = grad_h; a.out = grad_gate; a.out2 = grad_value;
  a.state = grad_last; a.lengths = lengths; a.ckpt_in = ckpt; a.last = grad_state;
  a.weight = (float*)workspace; a.carry = a.weight + (size_t)p.nchunk * p.lanes * p.vec;
  a.gate_sb = gate_sb; a.gate_st = gate_st; a.value_sb = value_sb; a.value_st = value_st;
  a.grad_sb = grad_sb; a.grad_st = grad_st;
  a.out_sb = dgate_sb; a.out_st = dgate_st; a.out2_sb = dvalue_sb; a.out2_st = dvalue_st;
  a.B = (uint32_t)B; a.T = (uint32_t)T; a.D = (uint32_t)D; a.DV = p.DV;
  a.lanes = p.lanes; a.chunk = p.chunk; a.nchunk = p.nchunk;
  if (dtype == TEMPO_DTYPE_F32) return launch_backward_for<float>(a, p.vec, (hipStream_t)stream);
  if (dtype == TEMPO_DTYPE_F16)
    return launch_backward_for<_Float16>(a, p.vec, (hipStream_t)stream);
  return launch_backward_for<__bf16>(a, p.vec, (hipStream_t)stream);
}

}  // extern "C"
