// MI355X (gfx950) kernels + C ABI of the fused linear layer and its gradients.
//
//   forward   z = x W^T + b          y = act(z) + r
//   backward  dz = g * act'(z)       dx = dz W    dW = dz^T x    db = sum over rows of dz
// x [M, K], W [N, K] (a 1x1 convolution's weight), y, r, g [M, N].
//
// All three products run through one tile kernel, C[i, j] = sum_k A(i, k) B(j, k), whose
// operands lie in memory either with k adjacent (K_ADJACENT: x and W in the forward, dz in
// dx) or with their own rows' index adjacent (ROW_ADJACENT: W in dx, both in dW).  Nothing is
// transposed in memory: 16-bit ROW_ADJACENT tiles are turned by the LDS's transposing read
// (ds_read_b64_tr_b16), fp32 tiles are read one k at a time, which v_mfma_f32_32x32x2_f32
// wants anyway.
//
// Rounding.  Products and sums are fp32 (fp32 inputs: fp32 matrix instructions, no split or
// shortened operands).  The epilogue is fp32 and rounds y once.  Two choices round to the
// tensors' type in between: z is kept for the backward pass in that type, and dz is an operand
// of two products in that type; both are half a step of a value that the products average
// over, no more than the rounding of their outputs (in fp16 a dz below 2^-25 becomes 0, like any
// gradient of that type: losses are scaled).  db is summed from unrounded dz.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/tempo_unproject.h"
#include "linear_plan.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

template <typename T, int V>
struct Pack {  // element-aligned: rows of odd width start anywhere
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// ---------------------------------------------------------------------------- activations

enum { NONE = TEMPO_ACT_NONE, RELU = TEMPO_ACT_RELU, SILU = TEMPO_ACT_SILU,
       GELU = TEMPO_ACT_GELU, SIGMOID = TEMPO_ACT_SIGMOID, TANH = TEMPO_ACT_TANH };

__device__ __forceinline__ float fast_exp(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504088896341f);
}

template <bool FULL>
__device__ __forceinline__ float sigmoid(float z) {
  const float e = FULL ? expf(-fabsf(z)) : fast_exp(-fabsf(z));
  const float r = FULL ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e);
  return z < 0.f ? e * r : (z != z ? z : r);
}

// Phi(z), the normal distribution.  16-bit results: erfc(x) = e^(-x^2) t P(t), t = 1 / (1 + p x),
// P and p fitted to the least relative error over 0 <= x <= 9.6, which is 4e-6 = 2^-18: far down
// gelu's tail, too, nothing beside the result's own rounding (an approximation good to an absolute
// 1.5e-7 is off by 14 % at z = -5.5).  The derivative needs e^(-z^2 / 2), too.
template <bool FULL>
__device__ __forceinline__ float normal_cdf(float z, float* density) {
  const float c = 0.3989422804014327f;  // 1 / sqrt(2 pi)
  if constexpr (FULL) {
    *density = c * expf(-0.5f * z * z);
    return 0.5f * erfcf(-0.7071067811865476f * z);
  } else {
    const float x = 0.7071067811865476f * fabsf(z);
    const float e = fast_exp(-x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.435207337f, x, 1.f));
    float p = fmaf(-0.151495814f, t, 0.382373691f);
    p = fmaf(p, t, 0.011490942f);
    p = fmaf(p, t, 0.274320513f);
    p = fmaf(p, t, 0.237244785f);
    p = fmaf(p, t, 0.246062174f);
    const float half = 0.5f * p * t * e;
    *density = c * e;
    return z < 0.f ? half : 1.f - half;
  }
}

template <bool FULL>
__device__ __forceinline__ float tanh_of(float z) {
  if constexpr (FULL) return tanhf(z);
  const float a = fabsf(z);
  const float e = fast_exp(-2.f * a);
  // next to 0 the quotient cancels: the series' error is 2/15 z^5 there
  const float t = a < 0.03f ? fmaf(-0.33333333f * a * a, a, a)
                            : (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
  return copysignf(t, z);
}

template <bool FULL>
__device__ __forceinline__ float activate(float z, int act) {
  float density;
  switch (act) {
    case RELU: return z < 0.f ? 0.f : z;  // a NaN passes
    case SILU: return z * sigmoid<FULL>(z);
    case GELU: return z * normal_cdf<FULL>(z, &density);
    case SIGMOID: return sigmoid<FULL>(z);
    case TANH: return tanh_of<FULL>(z);
    default: return z;
  }
}

template <bool FULL>
__device__ __forceinline__ float slope(float z, int act) {
  float density;
  switch (act) {
    case RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case SILU: {
      const float s = sigmoid<FULL>(z), n = sigmoid<FULL>(-z);
      return fmaf(z * s, n, s);
    }
    case GELU: {
      const float p = normal_cdf<FULL>(z, &density);
      return fmaf(z, density, p);
    }
    case SIGMOID: return sigmoid<FULL>(z) * sigmoid<FULL>(-z);
    case TANH: {  // 1 - tanh^2 = 4 sigmoid(2z) sigmoid(-2z), which does not cancel
      return 4.f * sigmoid<FULL>(2.f * z) * sigmoid<FULL>(-2.f * z);
    }
    default: return 1.f;
  }
}

// z in the tensors' type for the backward pass.  relu asks for its sign, which an fp16 underflow
// would lose; silu and gelu for a finite z to stay finite, for their slopes at an infinity are
// infinity times 0.  Beyond the type's range they are what they are at its end.
template <typename T>
__device__ __forceinline__ T keep_z(float z) {
  if constexpr (sizeof(T) == 2) {
    const float most = std::is_same<T, _Float16>::value ? 65504.f : 0x1.fep127f;
    const float inside = __builtin_amdgcn_fmed3f(z, -most, most);
    const T r = (T)(fabsf(z) <= 0x1.fffffep127f ? inside : z);  // infinities and NaN stay
    if (z > 0.f && (float)r == 0.f) {
      T least;
      const uint16_t one = 1;
      __builtin_memcpy(&least, &one, 2);
      return least;
    }
    return r;
  }
  return (T)z;
}

// ------------------------------------------------------------------------------ tile kernel

struct Epilogue {
  const void *bias, *residual;  // of the output's type, or NULL
  void *out, *pre;              // pre: z, or NULL
  float* partial;               // not NULL: raw sums [split][I][J] instead of the above
  long long ldr, ldo, ldp;
  int act;
};

struct TileArgs {
  const void *a, *b;
  long long lda, ldb;  // elements between rows (K_ADJACENT) or between k (ROW_ADJACENT)
  long long I, J, K;
  uint32_t ti, tj;     // tiles
  uint32_t split;      // parts of K, each k_part long (a multiple of the step)
  long long k_part;
  Epilogue e;
};

template <typename T>
struct Mfma;
template <>
struct Mfma<float> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c,
                                               0, 0, 0);
    return c;
  }
};
template <>
struct Mfma<_Float16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma<__bf16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// E elements at p, of which those at or beyond `left` are not in memory and count as 0
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p, long long left) {
  constexpr int E = 16 / sizeof(T);
  if (left >= E) {
    const typename Pack<T, E>::type r = *reinterpret_cast<const typename Pack<T, E>::type*>(p);
    return __builtin_bit_cast(u32x4, r);
  }
  T r[E];
#pragma unroll
  for (int j = 0; j < E; ++j) r[j] = j < left ? p[j] : (T)0.f;
  u32x4 out;
  __builtin_memcpy(&out, r, 16);
  return out;
}

// One operand's tile in LDS: ROWS rows x BYTES of k.  16-byte chunks are permuted within their
// row so that the 16 lanes which the LDS serves at a time hit every bank once:
//   K_ADJACENT    [row][k], 128 bytes: chunk c of row r at c ^ (r / 2 % 8), for two rows are all
//                 banks (c ^ (r % 8): half of the LDS's cycles were conflicts);  64 bytes: four
//                 rows are, c ^ (r / 4 % 4)
//   ROW_ADJACENT  [k][row], 16 bit: chunk c of line k at c ^ 4 (k % 4) (64 rows: two lines are all
//                 banks, c ^ 4 (k / 2 % 2);  32: four are, as it is);  fp32: as it is
template <typename T, int LAYOUT, int ROWS, int BYTES = 128>
struct Tile {
  static constexpr int E = 16 / sizeof(T);
  static constexpr int kDepth = BYTES / sizeof(T);
  static constexpr int kSteps = BYTES / 32;
  static constexpr int kLine = LAYOUT == K_ADJACENT ? BYTES / 16 : ROWS / E;  // chunks per line
  static constexpr int kBytes = ROWS * BYTES;
  static constexpr int kPerThread = ROWS * 8 / kThreads;

  static __device__ __forceinline__ uint32_t swap(uint32_t line, uint32_t c) {
    if constexpr (LAYOUT == K_ADJACENT)
      return BYTES == 128 ? c ^ (line / 2 & 7) : c ^ (line / 4 & 3);
    else if constexpr (sizeof(T) == 2 && ROWS >= 128)
      return c ^ (4 * (line & 3));
    else if constexpr (sizeof(T) == 2 && ROWS == 64)
      return c ^ (4 * (line / 2 & 1));
    else
      return c;
  }
  static __device__ __forceinline__ uint32_t place(uint32_t line, uint32_t c) {
    return (line * kLine + swap(line, c)) * 16;
  }

  static __device__ __forceinline__ void fetch(const T* p, long long ld, long long row0,
                                               long long rows, long long k0, long long k_end,
                                               u32x4 (&r)[kPerThread]) {
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
      const uint32_t q = n * kThreads + threadIdx.x;
      const uint32_t line = q / kLine, c = q % kLine;
      if constexpr (LAYOUT == K_ADJACENT) {
        const long long row = row0 + line, k = k0 + c * E;
        r[n] = load16<T>(p + row * ld + k, row < rows ? k_end - k : 0);
      } else {
        const long long row = row0 + c * E, k = k0 + line;
        r[n] = load16<T>(p + k * ld + row, k < k_end ? rows - row : 0);
      }
    }
  }

  static __device__ __forceinline__ void put(char* lds, const u32x4 (&r)[kPerThread]) {
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
      const uint32_t q = n * kThreads + threadIdx.x;
      *reinterpret_cast<u32x4*>(lds + place(q / kLine, q % kLine)) = r[n];
    }
  }

  // rows row0 .. row0 + 31 (lane % 32) x the k of step s: lanes 0..31 hold its first half,
  // 32..63 its second
  static __device__ __forceinline__ u32x4 fragment(const char* lds, uint32_t row0, uint32_t s,
                                                   uint32_t lane) {
    if constexpr (LAYOUT == K_ADJACENT) {
      return *reinterpret_cast<const u32x4*>(lds + place(row0 + lane % 32, 2 * s + lane / 32));
    } else if constexpr (sizeof(T) == 2) {
      // 16 lanes read 4 lines of 16 rows; lane i of them gets row i of the 4 lines
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      const uint32_t line = 16 * s + 8 * (lane / 32) + lane % 16 / 4;
      const uint32_t row = row0 + lane / 16 % 2 * 16 + lane % 4 * 4;
      const uint32_t low = (row * 2) & 8;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_i16x4*)(lds + place(line, row / 8) + low));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_i16x4*)(lds + place(line + 4, row / 8) + low));
      u32x4 out;
      __builtin_memcpy(&out, &lo, 8);
      __builtin_memcpy(reinterpret_cast<char*>(&out) + 8, &hi, 8);
      return out;
    } else {
      u32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = *reinterpret_cast<const uint32_t*>(
            lds + ((8 * s + 4 * (lane / 32) + j) * ROWS + row0 + lane % 32) * 4);
      return out;
    }
  }
};

// Tiles go to the 8 XCDs (workgroups are dealt to them in turn) in contiguous runs, and within
// a run 8 tile rows at a time, so that one L2 sees few different rows of both operands.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t ti, uint32_t tj, uint32_t* i,
                                        uint32_t* j) {
  const uint32_t n = ti * tj, per = n / 8, rest = n % 8, x = id % 8;
  const uint32_t t = x * per + min(x, rest) + id / 8;
  const uint32_t group = t / (8 * tj), first = group * 8, high = min(8u, ti - first);
  const uint32_t in = t - group * 8 * tj;
  *i = first + in % high;
  *j = in / high;
}

template <bool FULL, int ROWS>
__device__ __forceinline__ void activate_rows(f32x4 (&z)[ROWS], int act) {
  switch (act) {  // one branch for all of them
#define TEMPO_EACH(name)                                                              \
  case name:                                                                          \
    _Pragma("unroll") for (int r = 0; r < ROWS; ++r) _Pragma("unroll") for (int q = 0; q < 4; ++q) \
        z[r][q] = activate<FULL>(z[r][q], name);                                      \
    break;
    TEMPO_EACH(RELU)
    TEMPO_EACH(SILU)
    TEMPO_EACH(GELU)
    TEMPO_EACH(SIGMOID)
    TEMPO_EACH(TANH)
#undef TEMPO_EACH
    default: break;
  }
}

// The epilogue of ROWS quads of one column group, rows `apart` from each other, those from
// `stop` on left out; n of the 4 columns are inside the matrix.  The residuals of all of them
// are on their way before the first one is needed: one at a time, their latency took longer
// than four rows' (16384 x 4096 x 4096 with residual: 590 us against 544).
template <typename T, int ROWS>
__device__ __forceinline__ void finish(const Epilogue& e, long long i, uint32_t apart,
                                       long long stop, long long j, int n, f32x4 (&z)[ROWS]) {
  constexpr bool FULL = sizeof(T) == 4;
  typedef typename Pack<T, 4>::type V4;
  V4 residual[ROWS];
  if (e.residual) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const T* p = (const T*)e.residual + min(i + r * apart, stop - 1) * e.ldr + j;
      if (n == 4) {
        residual[r] = *reinterpret_cast<const V4*>(p);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) residual[r][q] = q < n ? p[q] : (T)0.f;
      }
    }
  }
  if (e.bias) {
    const T* p = (const T*)e.bias + j;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float b = (float)p[min(q, n - 1)];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) z[r][q] += b;
    }
  }
  if (e.pre) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (i + r * apart >= stop) continue;
      T* p = (T*)e.pre + (i + r * apart) * e.ldp + j;
      V4 kept;
#pragma unroll
      for (int q = 0; q < 4; ++q) kept[q] = keep_z<T>(z[r][q]);
      if (n == 4) {
        *reinterpret_cast<V4*>(p) = kept;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < n) p[q] = kept[q];
      }
    }
  }
  activate_rows<FULL, ROWS>(z, e.act);
  if (e.residual) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int q = 0; q < 4; ++q) z[r][q] += (float)residual[r][q];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (i + r * apart >= stop) continue;
    T* p = (T*)e.out + (i + r * apart) * e.ldo + j;
    V4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = (T)z[r][q];
    if (n == 4) {
      *reinterpret_cast<V4*>(p) = o;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < n) p[q] = o[q];
    }
  }
}

constexpr int kTogether = 4;  // rows of an epilogue that are under way at a time

// A slab of sums in LDS to memory: rows row0 .. row0 + high - 1 of C, threads side by side along
// a row.  16-byte chunk c of row i lies at c ^ (i % 32), i % 16 where a row has 16.
template <typename T, uint32_t QUADS, uint32_t THREADS>
__device__ __forceinline__ void write_slab(const TileArgs& a, const char* lds, long long row0,
                                           uint32_t high, long long j0) {
  const uint32_t c = threadIdx.x % QUADS;
  constexpr uint32_t kApart = THREADS / QUADS, kMask = QUADS < 32 ? QUADS - 1 : 31;
  const long long j = j0 + c * 4;
  if (j >= a.J) return;
  const int n = (int)min(4ll, a.J - j);
#pragma unroll 1
  for (uint32_t i = threadIdx.x / QUADS; i < high; i += kTogether * kApart) {
    f32x4 v[kTogether];
#pragma unroll
    for (int r = 0; r < kTogether; ++r) {
      const uint32_t row = min(i + r * kApart, high - 1);
      v[r] = *reinterpret_cast<const f32x4*>(lds + (row * QUADS + (c ^ (row & kMask))) * 16);
    }
    if (a.e.partial) {
#pragma unroll
      for (int r = 0; r < kTogether; ++r) {
        if (i + r * kApart >= high) continue;
        float* p = a.e.partial +
                   ((long long)blockIdx.y * a.I + row0 + i + r * kApart) * a.J + j;
        if (n == 4) {
          *reinterpret_cast<Pack<float, 4>::type*>(p) = v[r];
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q < n) p[q] = v[r][q];
        }
      }
    } else {
      finish<T, kTogether>(a.e, row0 + i, kApart, row0 + high, j, n, v);
    }
  }
}

// 16 bytes moved down by n elements, zeros from above
template <typename T>
__device__ __forceinline__ u32x4 shift_down(u32x4 r, uint32_t n) {
  const uint32_t bits = n * 8 * sizeof(T);
  uint64_t lo = (uint64_t)r[1] << 32 | r[0], hi = (uint64_t)r[3] << 32 | r[2];
  if (bits >= 128) lo = hi = 0;
  else if (bits >= 64) lo = hi >> (bits - 64), hi = 0;
  else if (bits) lo = lo >> bits | hi << (64 - bits), hi >>= bits;
  const u32x4 out = {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  return out;
}

// One operand's way to LDS through registers, for rows at any alignment.  Every load is whole
// and inside the operand, without a branch: a chunk across the end of its row is loaded so that
// it ends there and moved down afterwards, rows and k beyond the end are loaded from the last
// ones, k beyond the end then set to 0.  Needs 16 bytes in the adjacent direction.
template <typename T, int LAYOUT, int ROWS>
struct Gather {
  typedef Tile<T, LAYOUT, ROWS> Shape;
  static constexpr int E = Shape::E, kCount = Shape::kPerThread;
  const T* at[kCount];
  long long ld;
  uint32_t first[kCount];  // K_ADJACENT: a chunk's first k in its step; ROW_ADJACENT: its line
  uint32_t move[kCount];   // ROW_ADJACENT: elements
  bool edge;               // ROW_ADJACENT: some chunk needs to be moved

  __device__ __forceinline__ Gather(const void* p, long long ld_, long long row0, long long rows) {
    ld = ld_;
    edge = LAYOUT == ROW_ADJACENT && row0 + ROWS > rows;
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const uint32_t q = n * kThreads + threadIdx.x;
      const uint32_t line = q / Shape::kLine, c = q % Shape::kLine;
      if constexpr (LAYOUT == K_ADJACENT) {
        at[n] = (const T*)p + min(row0 + line, rows - 1) * ld;
        first[n] = c * E;
        move[n] = 0;
      } else {
        const long long row = row0 + c * E, inside = min(row, rows - E);
        at[n] = (const T*)p + inside;
        first[n] = line;
        move[n] = (uint32_t)(row - inside);
      }
    }
  }

  __device__ __forceinline__ void fetch(uint32_t k0, uint32_t K, u32x4 (&r)[kCount]) const {
    typedef typename Pack<T, E>::type Chunk;
    if (k0 + Shape::kDepth <= K) {
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const T* p = LAYOUT == K_ADJACENT ? at[n] + (k0 + first[n])
                                          : at[n] + (k0 + first[n]) * ld;
        r[n] = __builtin_bit_cast(u32x4, *reinterpret_cast<const Chunk*>(p));
      }
    } else {
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const uint32_t k = k0 + first[n];
        const T* p = LAYOUT == K_ADJACENT ? at[n] + min(k, K - E) : at[n] + min(k, K - 1) * ld;
        r[n] = __builtin_bit_cast(u32x4, *reinterpret_cast<const Chunk*>(p));
      }
#pragma unroll
      for (int n = 0; n < kCount; ++n) {
        const uint32_t k = k0 + first[n];
        if constexpr (LAYOUT == K_ADJACENT) {
          r[n] = shift_down<T>(r[n], k - min(k, K - E));
        } else if (k >= K) {
          r[n] = u32x4{0, 0, 0, 0};
        }
      }
    }
  }

  __device__ __forceinline__ void put(char* lds, u32x4 (&r)[kCount]) const {
    if (edge) {
#pragma unroll
      for (int n = 0; n < kCount; ++n) r[n] = shift_down<T>(r[n], move[n]);
    }
    Shape::put(lds, r);
  }
};

// The same for operands shorter than that, element by element
template <typename T, int LAYOUT, int ROWS>
struct TinyGather {
  typedef Tile<T, LAYOUT, ROWS> Shape;
  const T* p;
  long long ld, row0, rows;
  __device__ __forceinline__ TinyGather(const void* p_, long long ld_, long long row0_,
                                        long long rows_)
      : p((const T*)p_), ld(ld_), row0(row0_), rows(rows_) {}
  __device__ __forceinline__ void fetch(uint32_t k0, uint32_t K,
                                        u32x4 (&r)[Shape::kPerThread]) const {
    Shape::fetch(p, ld, row0, rows, k0, K, r);
  }
  __device__ __forceinline__ void put(char* lds, u32x4 (&r)[Shape::kPerThread]) const {
    Shape::put(lds, r);
  }
};

// 64 XI x 64 XJ of C per workgroup, 4 waves of a quarter each; loads of the next 128 bytes of k
// fly under the products of the present ones.  4999 x 515 x 1021 in fp16 and its gradients: 33,
// 23 and 22 us (0.16 to 0.24 PFLOP/s; a third of that time is loads through registers, most of the
// rest the latency of few steps in few tiles) and 7 us where parts of k are joined.
template <typename T, int AL, int BL, int XI, int XJ, bool TINY>
__global__ __launch_bounds__(kThreads) void tile_kernel(const TileArgs a) {
  constexpr int kRows = 64 * XI, kCols = 64 * XJ;
  typedef Tile<T, AL, kRows> TA;
  typedef Tile<T, BL, kCols> TB;
  __shared__ __attribute__((aligned(16))) char lds[2][TA::kBytes + TB::kBytes];
  uint32_t i_tile, j_tile;
  tile_of(blockIdx.x, a.ti, a.tj, &i_tile, &j_tile);
  const long long i0 = (long long)i_tile * kRows, j0 = (long long)j_tile * kCols;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t wi = wave / 2 * (32 * XI), wj = wave % 2 * (32 * XJ);
  const uint32_t k_begin = blockIdx.y * (uint32_t)a.k_part, K = (uint32_t)a.K;
  const uint32_t k_end = min(K, k_begin + (uint32_t)a.k_part);
  typedef typename std::conditional<TINY, TinyGather<T, AL, kRows>, Gather<T, AL, kRows>>::type GA;
  typedef typename std::conditional<TINY, TinyGather<T, BL, kCols>, Gather<T, BL, kCols>>::type GB;
  const GA ga(a.a, a.lda, i0, a.I);
  const GB gb(a.b, a.ldb, j0, a.J);

  f32x16 acc[XI][XJ];
#pragma unroll
  for (int x = 0; x < XI; ++x)
#pragma unroll
    for (int y = 0; y < XJ; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;

  u32x4 ra[TA::kPerThread], rb[TB::kPerThread];
  ga.fetch(k_begin, K, ra);
  gb.fetch(k_begin, K, rb);
  ga.put(lds[0], ra);
  gb.put(lds[0] + TA::kBytes, rb);
  __syncthreads();
  int now = 0;
  for (uint32_t k = k_begin; k < k_end; k += TA::kDepth, now ^= 1) {
    const bool more = k + TA::kDepth < k_end;
    if (more) {
      ga.fetch(k + TA::kDepth, K, ra);
      gb.fetch(k + TA::kDepth, K, rb);
    }
    const char* la = lds[now];
    const char* lb = la + TA::kBytes;
    u32x4 fa[2][XI], fb[2][XJ];
#pragma unroll
    for (int x = 0; x < XI; ++x) fa[0][x] = TA::fragment(la, wi + 32 * x, 0, lane);
#pragma unroll
    for (int y = 0; y < XJ; ++y) fb[0][y] = TB::fragment(lb, wj + 32 * y, 0, lane);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
#pragma unroll
      for (int x = 0; x < XI; ++x) {
        if (s < 3) {  // the next step's operands arrive under this one's products
          fa[s + 1 & 1][x] = TA::fragment(la, wi + 32 * x, s + 1, lane);
#pragma unroll
          for (int y = x * XJ / XI; y < (x + 1) * XJ / XI; ++y)
            fb[s + 1 & 1][y] = TB::fragment(lb, wj + 32 * y, s + 1, lane);
        }
#pragma unroll
        for (int y = 0; y < XJ; ++y)  // C^T: a lane holds 4 neighbouring j of one i
          acc[x][y] = Mfma<T>::run(fb[s & 1][y], fa[s & 1][x], acc[x][y]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) {
      ga.put(lds[now ^ 1], ra);
      gb.put(lds[now ^ 1] + TA::kBytes, rb);
    }
    __syncthreads();
  }

  // The tile's sums pass through LDS (the operands are done with): a wave holds columns
  // of rows, memory wants rows.  See write_slab for where they lie.
  char* lc = lds[0];
  constexpr uint32_t kQuads = kCols / 4, kMask = kQuads < 32 ? kQuads - 1 : 31;
  static_assert(sizeof(lds) >= kRows * kCols * 4, "the tile's sums fit");
#pragma unroll
  for (int x = 0; x < XI; ++x) {
#pragma unroll
    for (int y = 0; y < XJ; ++y) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t i = wi + 32 * x + lane % 32, c = (wj + 32 * y + 8 * g) / 4 + lane / 32;
        const f32x4 v = {acc[x][y][4 * g], acc[x][y][4 * g + 1], acc[x][y][4 * g + 2],
                         acc[x][y][4 * g + 3]};
        *reinterpret_cast<f32x4*>(lc + (i * kQuads + (c ^ (i & kMask))) * 16) = v;
      }
    }
  }
  __syncthreads();
  write_slab<T, kQuads, kThreads>(a, lc, i0, (uint32_t)min((long long)kRows, a.I - i0), j0);
}

// ---------------------------------------------------- tile kernel on aligned operands
//
// The same product where every 16-byte chunk of both operands is aligned and wholly inside or
// outside of its row: tiles go from memory straight to LDS (buffer_load ... lds), so no
// register holds data in flight and a workgroup can be 256 x 256, which halves what each
// product reads from LDS.  16384 x 4096 x 4096 in bf16: 464 us bare (1.18 PFLOP/s; the library's
// product 354 us), 523 us with a residual; what bounds it is the way from L2 to LDS -- on loads
// that all miss memory the same loop runs at 2.1 PFLOP/s, on loads that hit L2 at 1.42 -- and at
// short k the epilogue, which nothing overlaps (8192 x 4096 x 1024: 75 us bare, 119 with gelu and
// the values kept for the backward pass).  128 x 256 tiles, two workgroups a compute unit, do
// overlap it and lose more in the loop (600 us).  Chunks outside an operand carry an offset beyond the buffer's
// range, for which the hardware writes zeros.  A chunk's place in LDS follows from its lane
// (base + 16 lane), hence the lane picks the chunk that belongs to its place.

constexpr uint32_t kOutside = 0x80000000u;

__device__ __forceinline__ u32x4 buffer_of(const void* p, uint32_t bytes) {
  const uint64_t at = (uint64_t)p;
  u32x4 r = {(uint32_t)at, (uint32_t)(at >> 32), bytes, 0x00020000u};
#pragma unroll
  for (int q = 0; q < 4; ++q) r[q] = __builtin_amdgcn_readfirstlane(r[q]);
  return r;
}

// 64 chunks to LDS bytes lds .. lds + 1023; the caller waits (vmcnt) before anyone reads them
__device__ __forceinline__ void chunks_to_lds(uint32_t lds, uint32_t offset, u32x4 buffer,
                                              uint32_t scalar_offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds),
      "v"(offset), "s"(buffer), "s"(scalar_offset)
      : "memory");
}

// One operand's way to LDS: kLoads instructions per wave and step
template <typename T, int LAYOUT, int ROWS, int BYTES, int WAVES>
struct Stream {
  typedef Tile<T, LAYOUT, ROWS, BYTES> Shape;
  static constexpr int E = Shape::E;
  static constexpr int kLoads = Shape::kBytes / (WAVES * 1024);
  static_assert(kLoads * WAVES * 1024 == Shape::kBytes, "whole instructions");
  const T* base;
  long long ld;
  uint32_t offset[kLoads], chunk_k[kLoads];
  uint32_t extent;  // K_ADJACENT: bytes from the tile's first to its last element
  uint32_t rows;    // ROW_ADJACENT: of the operand from the tile's first on

  __device__ __forceinline__ Stream(const void* p, long long ld_, long long row0, long long I,
                                    long long K, uint32_t wave, uint32_t lane) {
    ld = ld_;
    const uint32_t high = (uint32_t)min((long long)ROWS, I - row0);
    rows = high;
    if constexpr (LAYOUT == K_ADJACENT) {
      base = (const T*)p + row0 * ld;
      extent = (uint32_t)(((high - 1) * ld + K) * sizeof(T));
    } else {
      base = (const T*)p + row0;
      extent = 0;
    }
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const uint32_t q = (n * WAVES + wave) * 64 + lane;
      const uint32_t line = q / Shape::kLine, slot = q % Shape::kLine;
      if constexpr (LAYOUT == K_ADJACENT) {
        const uint32_t c = Shape::swap(line, slot);
        chunk_k[n] = c * E;
        offset[n] = line < high ? (uint32_t)(line * ld * sizeof(T)) + c * 16 : kOutside;
      } else {
        const uint32_t c = Shape::swap(line, slot);
        offset[n] = c * E < high ? (uint32_t)(line * ld * sizeof(T)) + c * 16 : kOutside;
      }
    }
  }

  // One stage: k .. k + kDepth - 1; what lies at or beyond K becomes zeros, all of it where
  // k >= K, so that every step issues the same loads and can count them.
  struct Stage {
    u32x4 buffer;
    uint32_t at, left, lds;
  };
  __device__ __forceinline__ Stage stage(uint32_t lds, uint32_t k, uint32_t K) const {
    Stage s;
    s.lds = lds;
    s.left = k < K ? K - k : 0;
    if constexpr (LAYOUT == K_ADJACENT) {
      s.buffer = buffer_of(base, extent);
      s.at = __builtin_amdgcn_readfirstlane(s.left ? (uint32_t)(k * sizeof(T)) : 0u);
    } else {
      const uint32_t lines = min((uint32_t)Shape::kDepth, s.left);
      s.buffer = buffer_of(base + (s.left ? k * ld : 0),
                           lines ? (uint32_t)(((lines - 1) * ld + rows) * sizeof(T)) : 0u);
      s.at = 0;
    }
    return s;
  }
  __device__ __forceinline__ void load(const Stage& s, int n, uint32_t wave) const {
    const uint32_t o =
        LAYOUT == ROW_ADJACENT || chunk_k[n] < s.left ? offset[n] : kOutside;
    chunks_to_lds(s.lds + (n * WAVES + wave) * 1024, o, s.buffer, s.at);
  }
};

template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N of the wave's loads are under way
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// WI x WJ waves of XI x XJ blocks of 32 x 32; STAGES tiles of BYTES of k in LDS, of which one
// is read while the others arrive.
template <typename T, int AL, int BL, int WI, int WJ, int XI, int XJ, int BYTES, int STAGES>
__global__ __launch_bounds__(WI* WJ * 64, 2) void stream_kernel(const TileArgs a) {
  constexpr int kWaves = WI * WJ, kRows = WI * XI * 32, kCols = WJ * XJ * 32;
  typedef Tile<T, AL, kRows, BYTES> TA;
  typedef Tile<T, BL, kCols, BYTES> TB;
  constexpr int kStage = TA::kBytes + TB::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[STAGES * kStage];
  uint32_t i_tile, j_tile;
  tile_of(blockIdx.x, a.ti, a.tj, &i_tile, &j_tile);
  const long long i0 = (long long)i_tile * kRows, j0 = (long long)j_tile * kCols;
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wi = wave / WJ * XI * 32, wj = wave % WJ * XJ * 32;
  const uint32_t k_begin = blockIdx.y * (uint32_t)a.k_part;
  const uint32_t k_end = min((uint32_t)a.K, k_begin + (uint32_t)a.k_part);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  typedef Stream<T, AL, kRows, BYTES, kWaves> SA;
  typedef Stream<T, BL, kCols, BYTES, kWaves> SB;
  const SA sa(a.a, a.lda, i0, a.I, a.K, wave, lane);
  const SB sb(a.b, a.ldb, j0, a.J, a.K, wave, lane);

  f32x16 acc[XI][XJ];
#pragma unroll
  for (int x = 0; x < XI; ++x)
#pragma unroll
    for (int y = 0; y < XJ; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;

  // Loads, LDS reads and products are dealt out evenly: issued in a burst behind the barrier,
  // a stage's loads keep the compute unit's address path, and with it every wave, busy for
  // longer than its products take.  A stage's loads are cut into kSteps portions: the first
  // goes out behind the barrier that frees the stage's place, the others in the next round.
  constexpr int kLoads = SA::kLoads + SB::kLoads;
  constexpr int kPortion = (kLoads + TA::kSteps - 1) / TA::kSteps;
  constexpr int kReads = XI + XJ;
  u32x4 fa[2][XI], fb[2][XJ];  // one set feeds the products while the other one arrives
  typename SA::Stage ga;
  typename SB::Stage gb;
  auto refill = [&](uint32_t place, uint32_t k) {
    ga = sa.stage(lds0 + place, k, k_end);
    gb = sb.stage(lds0 + place + TA::kBytes, k, k_end);
  };
  auto load = [&](int n) {
    if (n < SA::kLoads) sa.load(ga, n, wave);
    else if (n < kLoads) sb.load(gb, n - SA::kLoads, wave);
  };
  auto read = [&](int set, uint32_t place, int step, int n) {
    if (n < XJ) fb[set][n] = TB::fragment(lds + place + TA::kBytes, wj + 32 * n, step, lane);
    else fa[set][n - XJ] = TA::fragment(lds + place, wi + 32 * (n - XJ), step, lane);
  };
  // products of one set, reads of the other, one portion of loads
  auto phase = [&](int set, uint32_t place, int step, int portion) {
#pragma unroll
    for (int x = 0; x < XI; ++x) {
#pragma unroll
      for (int n = x * kReads / XI; n < (x + 1) * kReads / XI; ++n) read(set ^ 1, place, step, n);
#pragma unroll
      for (int y = 0; y < XJ; ++y)
        acc[x][y] = Mfma<T>::run(fb[set][y], fa[set][x], acc[x][y]);
#pragma unroll
      for (int n = x * kPortion / XI; n < (x + 1) * kPortion / XI; ++n)
        load(portion * kPortion + n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int n = 0; n < STAGES; ++n) {
    refill(n * kStage, k_begin + n * TA::kDepth);
#pragma unroll
    for (int l = 0; l < (n < STAGES - 1 ? kLoads : kPortion); ++l) load(l);
  }
  wait_loads<(STAGES - 2) * kLoads + kPortion>();
  __syncthreads();
  uint32_t now = 0;
#pragma unroll
  for (int n = 0; n < kReads; ++n) read(0, 0, 0, n);
  for (uint32_t k = k_begin; k < k_end; k += TA::kDepth) {
    const uint32_t next = now + kStage < STAGES * kStage ? now + kStage : 0;
#pragma unroll
    for (int step = 0; step < TA::kSteps - 1; ++step) phase(step & 1, now, step + 1, step + 1);
    // The next stage has arrived (the STAGES - 2 behind it may still be under way) and everyone
    // has read this one: refill it, and begin on the next under the last products of this one.
    wait_loads<(STAGES - 2) * kLoads>();
    __syncthreads();
    refill(now, k + STAGES * TA::kDepth);
    phase(1, next, 0, 0);
    now = next;
  }
  wait_loads<0>();  // zeros on their way to stages behind the end
  __syncthreads();

  // sums through LDS as above, kSlab rows at a time
  constexpr uint32_t kFit = STAGES * kStage / (kCols * 4) / (XI * 32) * (XI * 32);
  constexpr uint32_t kSlab = kFit < kRows ? kFit : kRows, kQuads = kCols / 4;
  constexpr uint32_t kMask = kQuads < 32 ? kQuads - 1 : 31;
  static_assert(kSlab > 0, "a wave's rows fit in LDS");
#pragma unroll
  for (uint32_t slab = 0; slab < kRows; slab += kSlab) {
    if (slab) __syncthreads();
    if (wi >= slab && wi < slab + kSlab) {
#pragma unroll
      for (int x = 0; x < XI; ++x) {
#pragma unroll
        for (int y = 0; y < XJ; ++y) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t i = wi - slab + 32 * x + lane % 32;
            const uint32_t q = (wj + 32 * y + 8 * g) / 4 + lane / 32;
            const f32x4 v = {acc[x][y][4 * g], acc[x][y][4 * g + 1], acc[x][y][4 * g + 2],
                             acc[x][y][4 * g + 3]};
            *reinterpret_cast<f32x4*>(lds + (i * kQuads + (q ^ (i & kMask))) * 16) = v;
          }
        }
      }
    }
    __syncthreads();
    const long long left = a.I - i0 - slab;
    const uint32_t high = left < 0 ? 0u : (uint32_t)min((long long)kSlab, left);
    write_slab<T, kQuads, kWaves * 64>(a, lds, i0 + slab, high, j0);
  }
}

// The parts of a K that was split, then the epilogue.  GROUPS threads share an output quad:
// each adds a run of parts, in order, and the first one adds the runs, in order.
template <typename T, int GROUPS>
__global__ __launch_bounds__(kThreads) void join_kernel(const float* partial, uint32_t split,
                                                        long long I, long long J, Epilogue e) {
  constexpr int kWide = kThreads / GROUPS;
  __shared__ f32x4 s_sum[GROUPS][kWide];
  const uint32_t x = threadIdx.x % kWide, group = threadIdx.x / kWide;
  const long long quads = (J + 3) / 4;
  const long long id = (long long)blockIdx.x * kWide + x;
  const bool on = id < I * quads;
  const long long i = id / quads, j = (id - i * quads) * 4;
  const int n = (int)min(4ll, J - j);
  const uint32_t run = (split + GROUPS - 1) / GROUPS;
  const uint32_t first = min(group * run, split), stop = min(first + run, split);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    const float* p = partial + ((long long)first * I + i) * J + j;
#pragma unroll 8
    for (uint32_t s = first; s < stop; ++s, p += I * J) {
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] += p[min(q, n - 1)];
    }
  }
  if constexpr (GROUPS > 1) {
    s_sum[group][x] = sum;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) sum += s_sum[g][x];
  }
  if (on) {
    f32x4 z[1] = {sum};
    finish<T, 1>(e, i, 0, i + 1, j, n, z);
  }
}

// ------------------------------------------------------------------------ many rows, few columns
//
// J <= 32, B small enough to stay in LDS: a workgroup lays B out in fragment order once and
// its waves stream rows of A, 32 at a time, from memory right into the matrix units' operand
// registers, the next kChunk steps ahead of the products.  Nothing but A's rows and the
// result moves, at any alignment: memory bounds it: 614400 x 32 x 256 in bf16 71 us
// (5.0 TB/s), 153600 x 32 x 256 in fp32 38 us (4.7 TB/s).
constexpr int kChunk = 8;  // steps in flight per wave: 32 rows x 256 bytes

template <typename T>
struct ThinArgs {
  TileArgs t;
  uint32_t blocks, steps;  // row blocks of 32; steps of k
  int b_layout;
};

template <typename T>
__global__ __launch_bounds__(kThreads, 3) void thin_kernel(const ThinArgs<T> args) {
  constexpr int E = 16 / sizeof(T), kStep = 2 * E;
  constexpr uint32_t kQuads = 8;
  constexpr int kThinTogether = 2;  // rows of the epilogue under way at a time
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const TileArgs& a = args.t;
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const T* pb = (const T*)a.b;
  for (uint32_t q = threadIdx.x; q < args.steps * 64; q += kThreads) {
    const uint32_t l = q % 64, s = q / 64;
    const long long j = l % 32, k = (long long)s * kStep + l / 32 * E;
    u32x4 v = {0, 0, 0, 0};
    if (j < a.J) {
      if (args.b_layout == K_ADJACENT) {
        v = load16<T>(pb + j * a.ldb + k, a.K - k);
      } else {
        T r[E];
#pragma unroll
        for (int n = 0; n < E; ++n) r[n] = k + n < a.K ? pb[(k + n) * a.ldb + j] : (T)0.f;
        __builtin_memcpy(&v, r, 16);
      }
    }
    *reinterpret_cast<u32x4*>(lds + (size_t)q * 16) = v;
  }
  __syncthreads();
  char* turn = lds + (size_t)args.steps * 1024 + wave * 4096;

  const uint32_t chunks = (args.steps + kChunk - 1) / kChunk;
  const uint32_t stride = gridDim.x * (kThreads / 64);
  uint32_t block = blockIdx.x * (kThreads / 64) + wave, chunk = 0;
  if (block >= args.blocks) return;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;

  auto fetch = [&](u32x4(&f)[kChunk], uint32_t blk, uint32_t chk) {
    const long long i = min((long long)blk * 32 + lane % 32, a.I - 1);
    const T* p = (const T*)a.a + i * a.lda + (lane / 32 * E + chk * (kChunk * kStep));
    const long long left = a.K - (long long)chk * (kChunk * kStep);
    if (left >= kChunk * kStep) {
#pragma unroll
      for (int s = 0; s < kChunk; ++s) f[s] = load16<T>(p + s * kStep, E);
    } else {
      const long long mine = left - lane / 32 * E;
#pragma unroll
      for (int s = 0; s < kChunk; ++s) {
        if (s * kStep < left) f[s] = load16<T>(p + s * kStep, mine - s * kStep);
      }
    }
  };
  auto use = [&](const u32x4(&f)[kChunk], uint32_t blk, uint32_t chk) {
    const uint32_t s0 = chk * kChunk;
    const char* pf = lds + (size_t)(s0 * 64 + lane) * 16;
#pragma unroll
    for (int s = 0; s < kChunk; ++s) {
      if (s0 + s < args.steps) {
        const u32x4 fb = *reinterpret_cast<const u32x4*>(pf + (size_t)s * 1024);
        acc = Mfma<T>::run(fb, f[s], acc);
      }
    }
    if (chk + 1 < chunks) return;
    const long long left = a.I - (long long)blk * 32;
    const uint32_t high = (uint32_t)min(32ll, left);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t i = lane % 32, q = 2 * g + lane / 32;
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = acc[4 * g + r];
        acc[4 * g + r] = 0.f;
      }
      *reinterpret_cast<f32x4*>(turn + (i * kQuads + (q ^ (i % kQuads))) * 16) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const uint32_t q = lane % kQuads;
    const long long j = q * 4;
    const int n = (int)min(4ll, a.J - j);
    if (n > 0) {
      constexpr uint32_t kApart = 64 / kQuads;
#pragma unroll 1
      for (uint32_t i = lane / kQuads; i < high; i += kThinTogether * kApart) {
        f32x4 v[kThinTogether];
#pragma unroll
        for (int r = 0; r < kThinTogether; ++r) {
          const uint32_t row = i + r * kApart;  // < 32, the block's rows
          v[r] = *reinterpret_cast<const f32x4*>(
              turn + (row * kQuads + (q ^ (row % kQuads))) * 16);
        }
        finish<T, kThinTogether>(a.e, (long long)blk * 32 + i, kApart, a.I, j, n, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };

  u32x4 one[kChunk], two[kChunk];
  fetch(one, block, chunk);
  while (true) {
    uint32_t block2 = block, chunk2 = chunk + 1;
    if (chunk2 == chunks) chunk2 = 0, block2 += stride;
    if (block2 < args.blocks) fetch(two, block2, chunk2);
    use(one, block, chunk);
    if (block2 >= args.blocks) break;
    block = block2, chunk = chunk2 + 1;
    if (chunk == chunks) chunk = 0, block += stride;
    if (block < args.blocks) fetch(one, block, chunk);
    use(two, block2, chunk2);
    if (block >= args.blocks) break;
  }
}

// ------------------------------------------------------------------------ few rows, any weight
//
// I <= 16 NI: what counts is reading B, once and by the whole card (8 x 4096 x 4096 in fp16:
// 11 us = 3.0 TB/s).  A workgroup takes 16 rows
// of B; its waves share out k, each streaming its part of the 16 rows into the matrix units'
// operands, and their sums meet in LDS.  One launch, no scratch memory.
template <typename T>
struct SmallMfma;
template <>
struct SmallMfma<float> {
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0,
                                               0, 0);
    return c;
  }
};
template <>
struct SmallMfma<_Float16> {
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct SmallMfma<__bf16> {
  static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

constexpr int kFewWaves = 16;

template <typename T, int NI>
__global__ __launch_bounds__(kFewWaves * 64) void few_kernel(const TileArgs a) {
  constexpr int E = 16 / sizeof(T), kStep = 4 * E, kAhead = 4;
  __shared__ f32x4 s_sum[kFewWaves][NI][64];
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t waves = blockDim.x / 64;
  const long long j0 = (long long)blockIdx.x * 16;
  const long long row = min(j0 + lane % 16, a.J - 1);
  const T* pb = (const T*)a.b + row * a.ldb + lane / 16 * E;
  const T* pa[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x)
    pa[x] = (const T*)a.a + min((long long)x * 16 + lane % 16, a.I - 1) * a.lda + lane / 16 * E;
  const uint32_t steps = (uint32_t)((a.K + kStep - 1) / kStep);
  f32x4 acc[NI];
#pragma unroll
  for (int x = 0; x < NI; ++x) acc[x] = {0.f, 0.f, 0.f, 0.f};
  // waves take neighbouring steps: together they read whole rows
  for (uint32_t s0 = wave; s0 < steps; s0 += waves * kAhead) {
    u32x4 fb[kAhead], fa[kAhead][NI];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const uint32_t s = s0 + n * waves;
      if (s < steps) {
        const long long k = (long long)s * kStep, left = a.K - k - lane / 16 * E;
        fb[n] = load16<T>(pb + k, left);
#pragma unroll
        for (int x = 0; x < NI; ++x) fa[n][x] = load16<T>(pa[x] + k, left);
      }
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (s0 + n * waves < steps) {
#pragma unroll
        for (int x = 0; x < NI; ++x) acc[x] = SmallMfma<T>::run(fb[n], fa[n][x], acc[x]);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < NI; ++x) s_sum[wave][x][lane] = acc[x];
  __syncthreads();
  if (wave >= NI) return;
  f32x4 sum = s_sum[0][wave][lane];
  for (uint32_t w = 1; w < waves; ++w) sum += s_sum[w][wave][lane];
  // lane: row 16 x + lane % 16 of A, 4 neighbouring rows of B
  const long long i = wave * 16 + lane % 16, j = j0 + lane / 16 * 4;
  if (i < a.I && j < a.J) {
    f32x4 z[1] = {sum};
    finish<T, 1>(a.e, i, 0, i + 1, j, (int)min(4ll, a.J - j), z);
  }
}

// --------------------------------------------------------------- gradient of z, bias gradient


template <bool FULL, int V, typename Chunk>
__device__ __forceinline__ void slopes(const Chunk& z, float (&d)[V], int act) {
  switch (act) {  // one branch for all of them
#define TEMPO_EACH(name)                                                            \
  case name:                                                                        \
    _Pragma("unroll") for (int q = 0; q < V; ++q) d[q] = slope<FULL>((float)z[q], name); \
    break;
    TEMPO_EACH(RELU)
    TEMPO_EACH(SILU)
    TEMPO_EACH(GELU)
    TEMPO_EACH(SIGMOID)
    TEMPO_EACH(TANH)
#undef TEMPO_EACH
    default: break;
  }
}

// dz = g * act'(z) in the tensors' type (unless dz is NULL) and the sums of the unrounded
// values over the workgroup's rows (right into db where one workgroup holds them all).  A thread
// owns 16 bytes of columns, WIDE threads side by side, four rows of each under way at a time: 8192
// x 4096 in bf16 42 us, 4.8 TB/s.
template <typename T, int WIDE>
__global__ __launch_bounds__(kThreads) void grad_z_kernel(const T* g, long long ldg, const T* pre,
                                                          T* dz, float* sums, T* db, long long M,
                                                          int N, int act, int rows) {
  constexpr bool FULL = sizeof(T) == 4;
  constexpr int V = 16 / sizeof(T), kWide = WIDE * V, kHigh = kThreads / WIDE, kRows = 4;
  typedef typename Pack<T, V>::type Chunk;
  __shared__ float s_sum[kWide][kHigh + 1];
  const int j = blockIdx.y * kWide + threadIdx.x % WIDE * V;
  const int r = threadIdx.x / WIDE;
  const long long first = (long long)blockIdx.x * rows;
  const long long stop = min(M, first + rows);
  const int n = max(0, min(V, N - j));
  float sum[V];
#pragma unroll
  for (int q = 0; q < V; ++q) sum[q] = 0.f;
  if (n > 0) {
    for (long long i0 = first + r; i0 < stop; i0 += kHigh * kRows) {
      Chunk gv[kRows], zv[kRows];
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        const long long i = min(i0 + kHigh * x, stop - 1);
        if (n == V) {
          gv[x] = *reinterpret_cast<const Chunk*>(g + i * ldg + j);
          if (pre) zv[x] = *reinterpret_cast<const Chunk*>(pre + i * N + j);
        } else {
#pragma unroll
          for (int q = 0; q < V; ++q) {
            gv[x][q] = q < n ? g[i * ldg + j + q] : (T)0.f;
            if (pre) zv[x][q] = q < n ? pre[i * N + j + q] : (T)0.f;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        const long long i = i0 + kHigh * x;
        if (i >= stop) continue;
        float d[V];
        if (pre) slopes<FULL, V>(zv[x], d, act);
        Chunk out;
#pragma unroll
        for (int q = 0; q < V; ++q) {
          d[q] = (float)gv[x][q] * (pre ? d[q] : 1.f);
          sum[q] += d[q];
          out[q] = (T)d[q];
        }
        if (!dz) continue;
        if (n == V) {
          *reinterpret_cast<Chunk*>(dz + i * N + j) = out;
        } else {
#pragma unroll
          for (int q = 0; q < V; ++q)
            if (q < n) dz[i * N + j + q] = out[q];
        }
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int q = 0; q < V; ++q) s_sum[threadIdx.x % WIDE * V + q][r] = sum[q];
  __syncthreads();
  for (int c = threadIdx.x; c < kWide; c += kThreads) {
    float total = 0.f;
    for (int k = 0; k < kHigh; ++k) total += s_sum[c][k];
    const int col = blockIdx.y * kWide + c;
    if (col < N && gridDim.x == 1) db[col] = (T)total;
    else if (col < N) sums[(long long)blockIdx.x * N + col] = total;
  }
}

// bias gradient from the row blocks' sums: a workgroup owns 8 columns
template <typename T>
__global__ __launch_bounds__(kThreads) void grad_bias_kernel(const float* sums, long long blocks,
                                                             int N, T* out) {
  __shared__ float s_sum[32][9];
  const int col = blockIdx.x * 8 + threadIdx.x % 8, r = threadIdx.x / 8;
  float sum = 0.f;
  if (col < N) {
#pragma unroll 8
    for (long long b = r; b < blocks; b += 32) sum += sums[b * N + col];
  }
  s_sum[r][threadIdx.x % 8] = sum;
  __syncthreads();
  if (threadIdx.x < 8 && col < N) {
    float total = 0.f;
    for (int k = 0; k < 32; ++k) total += s_sum[k][threadIdx.x];
    out[col] = (T)total;
  }
}

// ------------------------------------------------------------------------------------- host

template <typename T>
int run_few(const TileArgs& t, hipStream_t stream) {
  const dim3 grid((unsigned)((t.J + 15) / 16));
  const long long steps = (t.K * (long long)sizeof(T) + 63) / 64;
  const dim3 block((unsigned)(steps < kFewWaves ? (steps < 4 ? 4 : steps) : kFewWaves) * 64);
  if (t.I <= 16)
    hipLaunchKernelGGL((few_kernel<T, 1>), grid, block, 0, stream, t);
  else if (t.I <= 32)
    hipLaunchKernelGGL((few_kernel<T, 2>), grid, block, 0, stream, t);
  else
    hipLaunchKernelGGL((few_kernel<T, 4>), grid, block, 0, stream, t);
  return (int)hipGetLastError();
}

template <typename T>
int run_thin(const TileArgs& t, int b_layout, hipStream_t stream) {
  ThinArgs<T> a = {};
  a.t = t;
  a.blocks = (uint32_t)((t.I + 31) / 32);
  a.steps = (uint32_t)((t.K * (long long)sizeof(T) + 31) / 32);
  a.b_layout = b_layout;
  const uint32_t groups = (a.blocks + 3) / 4;
  const dim3 grid(groups < 3 * kUnits ? groups : 3 * kUnits);
  hipLaunchKernelGGL((thin_kernel<T>), grid, dim3(kThreads), thin_lds(t.K, sizeof(T)), stream, a);
  return (int)hipGetLastError();
}

template <typename T, int AL, int BL, int XI, int XJ>
void launch_tile(const Product& p, const TileArgs& t, bool tiny, hipStream_t stream) {
  const dim3 grid(p.ti * p.tj, p.split);
  if (p.kernel == STREAM)
    hipLaunchKernelGGL((stream_kernel<T, AL, BL, 2, 2, XI, XJ, 64, 4>), grid, dim3(256), 0, stream,
                       t);
  else if (tiny)
    hipLaunchKernelGGL((tile_kernel<T, AL, BL, XI, XJ, true>), grid, dim3(kThreads), 0, stream, t);
  else
    hipLaunchKernelGGL((tile_kernel<T, AL, BL, XI, XJ, false>), grid, dim3(kThreads), 0, stream,
                       t);
}

template <typename T, int AL, int BL>
int run_product(const void* a, long long lda, const void* b, long long ldb, long long I,
                long long J, long long K, const Epilogue& e, float* scratch,
                hipStream_t stream) {
  constexpr int dtype = sizeof(T) == 4 ? TEMPO_DTYPE_F32 : TEMPO_DTYPE_F16;
  Product p;
  plan_product(I, J, K, AL, BL, dtype,
               streamable(a, lda, AL, I, K, sizeof(T)) && streamable(b, ldb, BL, J, K, sizeof(T)),
               &p);
  TileArgs t = {};
  t.a = a; t.b = b; t.lda = lda; t.ldb = ldb; t.I = I; t.J = J; t.K = K;
  t.ti = p.ti; t.tj = p.tj; t.split = p.split; t.k_part = p.k_part;
  t.e = e;
  t.e.partial = p.split > 1 ? scratch : nullptr;
  const dim3 grid(p.ti * p.tj, p.split);
  if constexpr (AL == K_ADJACENT && BL == K_ADJACENT) {
    if (p.kernel == FEW) return run_few<T>(t, stream);
  }
  if constexpr (AL == K_ADJACENT) {
    if (p.kernel == THIN) return run_thin<T>(t, BL, stream);
  }
  if (p.kernel == TILE || p.kernel == STREAM) {
    constexpr int e = 16 / sizeof(T);
    const bool tiny = (AL == K_ADJACENT ? K : I) < e || (BL == K_ADJACENT ? K : J) < e;
    if (p.xi == 2 && p.xj == 2) launch_tile<T, AL, BL, 2, 2>(p, t, tiny, stream);
    else if (p.xi == 2) launch_tile<T, AL, BL, 2, 1>(p, t, tiny, stream);
    else if (p.xj == 2) launch_tile<T, AL, BL, 1, 2>(p, t, tiny, stream);
    else launch_tile<T, AL, BL, 1, 1>(p, t, tiny, stream);
  }
  if constexpr (AL == ROW_ADJACENT) {
    if (p.kernel == STREAM_32x256)
      hipLaunchKernelGGL((stream_kernel<T, AL, BL, 1, 4, 1, 2, 128, 2>), grid, dim3(256), 0, stream, t);
  }
  if constexpr (sizeof(T) == 2) {
    if (p.kernel == STREAM_256)
      hipLaunchKernelGGL((stream_kernel<T, AL, BL, 2, 4, 4, 2, 64, 4>), grid, dim3(512), 0, stream, t);
  }
  if (p.split > 1) {
    const long long quads = I * ((J + 3) / 4);
    if (p.split >= 16)
      hipLaunchKernelGGL((join_kernel<T, 16>), dim3((unsigned)((quads + 15) / 16)),
                         dim3(kThreads), 0, stream, scratch, p.split, I, J, e);
    else
      hipLaunchKernelGGL((join_kernel<T, 1>), dim3((unsigned)((quads + kThreads - 1) / kThreads)),
                         dim3(kThreads), 0, stream, scratch, p.split, I, J, e);
  }
  return (int)hipGetLastError();
}

struct BackwardPlan {
  int wide, rows;  // threads along a row and rows of grad_z_kernel's workgroups
  long long dz_bytes, sum_bytes, scratch_bytes;
  long long total() const { return dz_bytes + sum_bytes + scratch_bytes; }
};

long long up16(long long n) { return (n + 15) / 16 * 16; }

bool plan_backward(long long M, int N, int K, int dtype, int act, BackwardPlan* p) {
  long long x, w;
  if (!product_bytes(M, K, N, K_ADJACENT, ROW_ADJACENT, dtype, &x) ||
      !product_bytes(N, K, M, ROW_ADJACENT, ROW_ADJACENT, dtype, &w)) return false;
  p->dz_bytes = act == NONE ? 0 : up16(M * N * (dtype == TEMPO_DTYPE_F32 ? 4 : 2));
  // A row's pieces that end inside a 128-byte line are written to memory twice, so a workgroup
  // holds whole rows where it can (325353 x 280 in bf16: 126 us with 64 threads a row, 172 with
  // 32, 207 with 8), but no idle threads where pieces end with lines (200000 x 96 in fp32: 64 us
  // with 32, 55 with 8).  Beyond 64 threads a row, 32: 8192 x 4096 in bf16 40 us, 48 with 8, 44
  // with 64.
  const int size = dtype == TEMPO_DTYPE_F32 ? 4 : 2;
  const int chunks = (N * size + 15) / 16;
  p->wide = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 || chunks > 64 ? 32 : 64;
  while (N * size % 128 == 0 && chunks % p->wide) p->wide /= 2;
  // one workgroup for all rows needs no second launch (64 x 4096 in fp16: 4 us against 7)
  if (M <= 128) p->wide = 8;
  // few sums to add up, but four workgroups for each compute unit where the matrix allows it
  // (5000 x 515 in fp16: 31 us with 128 rows each, 13 with 32)
  const long long groups = (chunks + p->wide - 1) / p->wide;
  p->rows = 512;
  while (p->rows > 1024 / p->wide && (M + p->rows - 1) / p->rows * groups < 4 * kUnits)
    p->rows /= 2;
  p->sum_bytes = up16((M + p->rows - 1) / p->rows * N * 4);
  p->scratch_bytes = up16(x > w ? x : w);
  return true;
}

int check_sizes(long long M, int N, int K, int dtype, int act) {
  if (M <= 0 || N <= 0 || K <= 0) return TEMPO_E_DIM;
  if (dtype != TEMPO_DTYPE_F32 && dtype != TEMPO_DTYPE_F16 && dtype != TEMPO_DTYPE_BF16)
    return TEMPO_E_ARG;
  if (act < NONE || act > TANH) return TEMPO_E_ARG;
  if (M > 0x7fffffffLL || N > (1 << 20) || K > (1 << 20)) return TEMPO_E_SIZE;
  return TEMPO_OK;
}

bool misaligned(const void* p, int dtype) {
  return ((uintptr_t)p & (dtype == TEMPO_DTYPE_F32 ? 3 : 1)) != 0;
}

template <typename T>
int backward_for(const BackwardPlan& p, const void* g, long long ldg, const void* pre,
                 const void* x, long long ldx, const void* w, long long ldw, void* dx,
                 long long lddx, void* dw, void* db, long long M, int N, int K, int act,
                 char* ws, hipStream_t stream) {
  T* dz = act == NONE ? nullptr : (T*)ws;
  float* sums = db ? (float*)(ws + p.dz_bytes) : nullptr;
  float* scratch = (float*)(ws + p.dz_bytes + p.sum_bytes);
  const long long blocks = (M + p.rows - 1) / p.rows;
  if (dz || db) {
    constexpr int V = 16 / sizeof(T);
    auto kernel = p.wide == 8    ? grad_z_kernel<T, 8>
                  : p.wide == 16 ? grad_z_kernel<T, 16>
                  : p.wide == 32 ? grad_z_kernel<T, 32>
                                 : grad_z_kernel<T, 64>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (N + p.wide * V - 1) / (p.wide * V)),
                       dim3(kThreads), 0, stream, (const T*)g, ldg, (const T*)pre, dz, sums,
                       (T*)db, M, N, act, p.rows);
    if (db && blocks > 1)
      hipLaunchKernelGGL((grad_bias_kernel<T>), dim3((N + 7) / 8), dim3(kThreads), 0, stream,
                         sums, blocks, N, (T*)db);
  }
  const void* z = dz ? (const void*)dz : g;
  const long long ldz = dz ? N : ldg;
  Epilogue e = {};
  int rc = (int)hipGetLastError();
  if (rc == 0 && dx) {
    e.out = dx; e.ldo = lddx;
    rc = run_product<T, K_ADJACENT, ROW_ADJACENT>(z, ldz, w, ldw, M, K, N, e, scratch, stream);
  }
  if (rc == 0 && dw) {
    e.out = dw; e.ldo = K;
    rc = run_product<T, ROW_ADJACENT, ROW_ADJACENT>(z, ldz, x, ldx, N, K, M, e, scratch, stream);
  }
  return rc;
}

}  // namespace

extern "C" {

long long tempo_linear_workspace(long long M, int N, int K, int dtype, int activation,
                                 int backward) {
  const int rc = check_sizes(M, N, K, dtype, activation);
  if (rc != TEMPO_OK) return rc;
  if (backward) {
    BackwardPlan p;
    return plan_backward(M, N, K, dtype, activation, &p) ? p.total() : TEMPO_E_SIZE;
  }
  long long bytes;
  return product_bytes(M, N, K, K_ADJACENT, K_ADJACENT, dtype, &bytes) ? bytes : TEMPO_E_SIZE;
}

int tempo_linear(const void* x, long long ldx, const void* weight, long long ldw,
                 const void* bias, const void* residual, long long ldr, void* y, long long ldy,
                 void* pre, long long M, int N, int K, int dtype, int activation,
                 void* workspace, long long workspace_bytes, void* stream) {
  if (!x || !weight || !y) return TEMPO_E_NULL;
  const int rc = check_sizes(M, N, K, dtype, activation);
  if (rc != TEMPO_OK) return rc;
  long long need;
  if (!product_bytes(M, N, K, K_ADJACENT, K_ADJACENT, dtype, &need)) return TEMPO_E_SIZE;
  if (ldx < 0 || ldw < 0 || ldr < 0 || (M > 1 && ldy < N)) return TEMPO_E_ARG;
  if (misaligned(x, dtype) || misaligned(weight, dtype) || misaligned(y, dtype) ||
      misaligned(bias, dtype) || misaligned(residual, dtype) || misaligned(pre, dtype))
    return TEMPO_E_ARG;
  if (need > 0 && !workspace) return TEMPO_E_NULL;
  if (need > workspace_bytes) return TEMPO_E_SIZE;
  if ((uintptr_t)workspace & 15) return TEMPO_E_ARG;
  Epilogue e = {};
  e.bias = bias; e.residual = residual; e.out = y; e.pre = pre;
  e.ldr = ldr; e.ldo = ldy; e.ldp = N; e.act = activation;
  float* scratch = (float*)workspace;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TEMPO_DTYPE_F32)
    return run_product<float, K_ADJACENT, K_ADJACENT>(x, ldx, weight, ldw, M, N, K, e, scratch, s);
  if (dtype == TEMPO_DTYPE_F16)
    return run_product<_Float16, K_ADJACENT, K_ADJACENT>(x, ldx, weight, ldw, M, N, K, e, scratch,
                                                         s);
  return run_product<__bf16, K_ADJACENT, K_ADJACENT>(x, ldx, weight, ldw, M, N, K, e, scratch, s);
}

int tempo_linear_backward(const void* grad_y, long long ldg, const void* pre, const void* x,
                          long long ldx, const void* weight, long long ldw, void* grad_x,
                          long long lddx, void* grad_weight, void* grad_bias, long long M, int N,
                          int K, int dtype, int activation, void* workspace,
                          long long workspace_bytes, void* stream) {
  if (!grad_y || (grad_x && !weight) || (grad_weight && !x)) return TEMPO_E_NULL;
  const int rc = check_sizes(M, N, K, dtype, activation);
  if (rc != TEMPO_OK) return rc;
  if (activation != NONE && !pre) return TEMPO_E_NULL;
  BackwardPlan p;
  if (!plan_backward(M, N, K, dtype, activation, &p)) return TEMPO_E_SIZE;
  if (ldg < 0 || ldx < 0 || ldw < 0 || (grad_x && M > 1 && lddx < K)) return TEMPO_E_ARG;
  if (misaligned(grad_y, dtype) || misaligned(pre, dtype) || misaligned(x, dtype) ||
      misaligned(weight, dtype) || misaligned(grad_x, dtype) || misaligned(grad_weight, dtype) ||
      misaligned(grad_bias, dtype))
    return TEMPO_E_ARG;
  if (!workspace) return TEMPO_E_NULL;
  if (p.total() > workspace_bytes) return TEMPO_E_SIZE;
  if ((uintptr_t)workspace & 15) return TEMPO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  const void* z = activation == NONE ? nullptr : pre;
  if (dtype == TEMPO_DTYPE_F32)
    return backward_for<float>(p, grad_y, ldg, z, x, ldx, weight, ldw, grad_x, lddx, grad_weight,
                               grad_bias, M, N, K, activation, ws, s);
  if (dtype == TEMPO_DTYPE_F16)
    return backward_for<_Float16>(p, grad_y, ldg, z, x, ldx, weight, ldw, grad_x, lddx,
                                  grad_weight, grad_bias, M, N, K, activation, ws, s);
  return backward_for<__bf16>(p, grad_y, ldg, z, x, ldx, weight, ldw, grad_x, lddx, grad_weight,
                              grad_bias, M, N, K, activation, ws, s);
}

}  // extern "C"
