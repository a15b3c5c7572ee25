// Packed dense layer with bias, activation and residual in the epilogue
// (ops.nn.linear_act), forward and backward.
//
//   z = x_g W_g^T + b_g,   y_g = r_g + act(z)              (forward, NT)
//   dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz
//
// Three GEMMs from one kernel template.  They differ in which operands are
// stored with the reduction axis contiguous:
//
//   forward  A = x  [M][K] k-contiguous   B = W  [N][K] k-contiguous
//   dgrad    A = dz [M][N] k-contiguous   B = W  [N][K] k-strided (k = N)
//   wgrad    A = dz [M][N] k-strided      B = x  [M][K] k-strided (k = M)
//
// Operands are staged global -> registers -> LDS.  A k-strided operand is
// transposed on the way: a thread loads 8 k-rows of V neighbouring columns and
// writes V chunks of 8 consecutive k, so the LDS image, the fragments and the
// MFMA loop are the same for all three.
//
// Precision.  A bf16 operand is one plane; its products are exact in the fp32
// accumulators of v_mfma_f32_16x16x32_bf16.  An fp32 operand is split when it
// is staged into three bf16 planes p0 + p1 + p2, each the rounding of what the
// ones before it leave: together its 24 bits.  The product runs as the six
// terms p_i q_j with i + j <= 2, smallest first; what is dropped is below
// 2^-24 of |x||w| a term, so the result is that of an fp32 product (measured
// against 64 bits: as near as the library's) at 6/16 of the time of fp32 MFMA.
// In bf16 mode dz = dy * act'(z) has more than 8 bits: it is kept in fp32 and
// enters dW, an fp32 tensor, as DZ_PLANES planes and dx, a bf16 one, as DX_PLANES.  A non-finite fp32 factor gives a non-finite result,
// NaN where a single fp32 product would give an infinity; |x| above 3.39e38
// rounds to infinity.
#include <atomic>
#include <math.h>

#include "common.h"
#include "nodes_api.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
// element-aligned vectors: odd row lengths keep wide loads (gfx950 takes any
// element alignment for global accesses)
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32_a1 __attribute__((aligned(1)));

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_RELU6 = 6, ACT_GELU = 7, ACT_GELU_TANH = 8, ACT_SILU = 9 };
enum { EPI_FWD = 0, EPI_T = 1, EPI_F32 = 2 };

static inline bool act_known(int a) {
  return a == ACT_NONE || a == ACT_RELU || a == ACT_RELU6 || (a >= ACT_GELU && a <= ACT_SILU);
}
__host__ __device__ static inline bool act_smooth(int a) { return a >= ACT_GELU; }

// 1 / (1 + e), 0 <= e <= 1: the hardware's reciprocal and one Newton step
__device__ __forceinline__ float rcp1p(float e) {
  const float x = 1.f + e, r = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, r, 1.f), r, r);
}

// Polynomials of the normal distribution, coefficients from the constant up: least
// squares reweighted until the largest relative error of Phi stops falling (4 000
// and 8 000 points, in 64 bits).
//   |z| <= 1.5: (Phi(z) - 1/2) / z in z^2, to 2^-30
//   1.5 <= a:   Phi(-a) exp(a^2 / 2) in 1 / (a + 1.5), to 2^-25
__device__ __forceinline__ float phi_mid(float z2) {
  float p = 4.0268761836159683e-07f;
  p = fmaf(p, z2, -8.652973519929219e-06f);
  p = fmaf(p, z2, 1.1417106e-04f);
  p = fmaf(p, z2, -1.1862358e-03f);
  p = fmaf(p, z2, 9.9730734e-03f);
  p = fmaf(p, z2, -6.6490285e-02f);
  return fmaf(p, z2, 3.9894226e-01f);
}

__device__ __forceinline__ float phi_tail(float a) {
  const float t = __builtin_amdgcn_rcpf(a + 1.5f);
  float p = -6.780151844024658f;
  p = fmaf(p, t, 11.185012817382812f);
  p = fmaf(p, t, -6.108560085296631f);
  p = fmaf(p, t, 0.24226641654968262f);
  p = fmaf(p, t, 0.4250870943069458f);
  p = fmaf(p, t, 0.6031176447868347f);
  p = fmaf(p, t, 0.39877673983573914f);
  return fmaf(p, t, 2.4561902591813123e-06f);
}

// act(z), and act'(z) in d.  NaN passes through every branch (comparisons with
// NaN are false), unlike fmaxf.  The smooth ones are as near to 64 bits as erf, tanh
// and exp in fp32 (standard normal z: gelu 3.6e-8, its derivative 3.7e-8), and keep
// their relative error far below zero: nothing is left of 1 by subtraction.
__device__ __forceinline__ float act_fwd(float z, int act, float& d) {
  if (act == ACT_NONE) {
    d = 1.f;
    return z;
  }
  if (act == ACT_RELU) {
    d = z > 0.f ? 1.f : 0.f;
    return z <= 0.f ? 0.f : z;
  }
  if (act == ACT_RELU6) {
    d = (z > 0.f && z < 6.f) ? 1.f : 0.f;
    return z <= 0.f ? 0.f : (z >= 6.f ? 6.f : z);
  }
  const float a = fabsf(z);
  // beyond the float range of exp the limits, not inf * 0
  if (a > 1e4f) {
    d = z < 0.f ? 0.f : 1.f;
    return z < 0.f ? 0.f : z;
  }
  if (act == ACT_GELU) {
    const float z2 = z * z, e = expf(-0.5f * z2);
    const float tail = phi_tail(a) * e;
    const float cdf = a < 1.5f ? fmaf(z, phi_mid(z2), 0.5f) : z < 0.f ? tail : 1.f - tail;
    d = fmaf(z * 0.39894228040143268f, e, cdf);
    return z * cdf;
  }
  if (act == ACT_GELU_TANH) {
    const float c = 0.79788456080286536f;
    const float u = c * z * fmaf(0.044715f * z, z, 1.f);
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u)), and q = (1 - tanh u) / 2
    const float e = expf(-2.f * fabsf(u)), r = rcp1p(e), er = e * r;
    const float s = z < 0.f ? er : r, q = z < 0.f ? r : er;
    d = fmaf(2.f * z * s * q, c * fmaf(0.134145f * z, z, 1.f), s);
    return z * s;
  }
  // silu
  const float e = expf(-a), r = rcp1p(e), er = e * r;
  const float s = z < 0.f ? er : r, q = z < 0.f ? r : er;
  d = s * fmaf(z, q, 1.f);
  return z * s;
}

struct GemmP {
  const void* a;        // A + g * a_gs, leading dimension lda (elements)
  const void* b;
  int64_t lda, ldb, a_gs, b_gs;
  int m, n, k, G;
  void* c;              // out + g * c_gs + row * ldc + col
  int64_t ldc, c_gs;
  const void* bias;     // EPI_FWD: + g * bias_gs + col (or null)
  int64_t bias_gs;
  const void* res;      // EPI_FWD: residual (or null), config stride = c_gs
  int64_t ldr;
  void* d;              // EPI_FWD: act'(z) out (or null): fp32, or u8 for relu / relu6
  int act;
  float* part;          // split-K partials [split][g][m][n] (splits > 1)
  int splits, steps;    // k steps per split
  int tm, tn;           // tiles
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return bf2f(v); }

// 4 consecutive outputs of one row, the last `nv` < 4 of a ragged edge
template <typename T>
__device__ __forceinline__ void st4(T* p, const float* v, int nv) {
  if (nv >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_a4*>(p) = f32x4_a4{v[0], v[1], v[2], v[3]};
    } else {
      *reinterpret_cast<u32x2_a2*>(p) = u32x2_a2{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < nv) st1(p + i, v[i]);
  }
}

template <typename T>
__device__ __forceinline__ void ld4(const T* p, float* v, int nv) {
  if (nv >= 4) {
    if constexpr (sizeof(T) == 4) {
      const f32x4_a4 u = *reinterpret_cast<const f32x4_a4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = u[i];
    } else {
      const u32x2_a2 u = *reinterpret_cast<const u32x2_a2*>(p);
      v[0] = __uint_as_float(u.x << 16);
      v[1] = __uint_as_float(u.x & 0xffff0000u);
      v[2] = __uint_as_float(u.y << 16);
      v[3] = __uint_as_float(u.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < nv ? ld1(p + i) : 0.f;
  }
}

// bias and residual of columns col .. col + nv - 1 (at most 4) of config g
template <typename T>
__device__ __forceinline__ void ld_bias(const GemmP& P, int g, int col, int nv, float* b) {
  if (P.bias) ld4(reinterpret_cast<const T*>(P.bias) + g * P.bias_gs + col, b, nv);
  else b[0] = b[1] = b[2] = b[3] = 0.f;
}

template <typename T>
__device__ __forceinline__ const T* at_res(const GemmP& P, int g, int row, int col) {
  return reinterpret_cast<const T*>(P.res) + g * P.c_gs + (int64_t)row * P.ldr + col;
}

// finished sums of row `row`, those columns; EPI_FWD: with their bias and, if there
// is one, residual
template <int EPI, typename T>
__device__ __forceinline__ void epilogue(const GemmP& P, int g, int row, int col, int nv, float* z,
                                         const float* b, const float* r) {
  const int64_t o = (int64_t)g * P.c_gs + (int64_t)row * P.ldc + col;
  if constexpr (EPI == EPI_FWD) {
    if (P.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] += b[i];
    }
    float d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = act_fwd(z[i], P.act, d[i]);
    if (P.d) {
      if (act_smooth(P.act)) {
        st4(reinterpret_cast<float*>(P.d) + o, d, nv);
      } else {
        uint8_t* p = reinterpret_cast<uint8_t*>(P.d) + o;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (d[i] != 0.f ? 1u : 0u) << (8 * i);
        if (nv >= 4) {
          *reinterpret_cast<u32_a1*>(p) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 3; ++i)
            if (i < nv) p[i] = (uint8_t)(w >> (8 * i));
        }
      }
    }
    if (P.res) {
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] += r[i];
    }
    st4(reinterpret_cast<T*>(P.c) + o, z, nv);
  } else if constexpr (EPI == EPI_T) {
    st4(reinterpret_cast<T*>(P.c) + o, z, nv);
  } else {
    st4(reinterpret_cast<float*>(P.c) + o, z, nv);
  }
}

template <int EPI, typename T>
__device__ __forceinline__ void epilogue(const GemmP& P, int g, int row, int col, int nv,
                                         float* z) {
  float b[4] = {}, r[4] = {};
  if constexpr (EPI == EPI_FWD) {
    ld_bias<T>(P, g, col, nv, b);
    if (P.res) ld4(at_res<T>(P, g, row, col), r, nv);
  }
  epilogue<EPI, T>(P, g, row, col, nv, z, b, r);
}

// ---------------------------------------------------------------------------
// operand staging: rows R x BK of one operand per step, T threads; every
// thread moves V = R * BK / (8 T) chunks of 8 k
// ---------------------------------------------------------------------------
template <int BK>
__device__ __forceinline__ int lds_off(int row, int chunk) {
  // 16-B chunks are XOR-swizzled by row.  A wave's 16-B LDS access goes 16 lanes
  // at a time, 256 B; in a fragment read those are 16 neighbouring rows at one
  // chunk, or 8 of them at that chunk and 8 at its neighbour (c ^ 1): the
  // patterns below give 16 different places either way.  The transposing
  // writes (rows V apart) keep two lanes to a place.
  if constexpr (BK == 64) {
    return row * 128 + ((chunk ^ (((row >> 1) ^ (row >> 4)) & 7)) << 4);
  } else {
    const int i = row >> 2;
    return row * 64 + ((chunk ^ ((i ^ ((i & 1) << 1)) & 3)) << 4);
  }
}

template <typename S, bool KS, int R, int BK, int T, int PL>
struct Stage {
  static constexpr int V = R * BK / (8 * T);
  static_assert(V >= 1 && V * 8 * T == R * BK, "one unit per thread");
  static constexpr int CH = BK / 8;
  static constexpr bool F32 = sizeof(S) == 4;
  static constexpr int NR = F32 ? 8 * V : (KS ? 8 * (V > 1 ? V / 2 : 1) : 4 * V);
  static constexpr int BYTES = PL * R * BK * 2;
  struct Regs {
    uint32_t r[NR];
  };
  uint32_t off[KS ? 1 : V];   // byte offsets inside a step's tile
  const char* base;           // uniform: tile origin
  int64_t step_bytes;         // uniform: bytes from one step to the next
  uint32_t ldb;               // row pitch in bytes
  int row0, rows, kc;         // tile origin, operand extent; this thread's k chunk
  // k-strided operands, V > 1 columns a load.  Where no tile fits in the columns a
  // vector that crosses the last one is loaded V columns back from it and shifted
  // into place (a bf16 training pass of 8192 x 101 x 8192: 877 -> 600 us).  Not in
  // the tile of BK 64, where the code of it alone spills 40 registers instead of 2:
  // with 66 the bf16 dgrad of 8192 x 4096 x 4096 took 440 us, with 48 298, with 2
  // 290.  bf16 rows that start inside a dword are loaded as they lie; taking them
  // from their dwords by shifts costs 219 us against 207 at 2047^3.
  static constexpr bool SHIFT = KS && V > 1 && BK == 32;
  bool aligned;               // no vector of the tile crosses
  bool single;                // element by element

  __device__ __forceinline__ void init(const void* src, int64_t ld, int r0, int nrows, int k,
                                       int tid) {
    rows = nrows;
    row0 = r0;
    ldb = (uint32_t)(ld * sizeof(S));
    if constexpr (KS) {
      // V columns before the tile: offsets of vectors that start there stay
      // positive
      base = reinterpret_cast<const char*>(src) + ((int64_t)r0 - V) * (int)sizeof(S);
      step_bytes = (int64_t)BK * ld * sizeof(S);
      kc = tid / (R / V);
      int c = (tid % (R / V)) * V;
      aligned = r0 + R <= nrows || nrows % V == 0;
      single = nrows < V || (!SHIFT && !aligned);
      if (r0 + c + V > nrows) c = nrows - V - r0;       // wholly outside: any columns
      off[0] = (uint32_t)(kc * 8) * ldb + (uint32_t)((c + V) * (int)sizeof(S));
    } else {
      base = reinterpret_cast<const char*>(src) + (int64_t)r0 * ld * sizeof(S);
      step_bytes = (int64_t)BK * sizeof(S);
      kc = tid % CH;
      aligned = true;
      single = k < 8;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        int row = tid / CH + i * (T / CH);
        if (r0 + row >= nrows) row = nrows - 1 - r0;           // discarded rows: any row
        off[i] = (uint32_t)row * ldb + (uint32_t)(kc * 8 * (int)sizeof(S));
      }
    }
  }

  // chunk i of a row-strided operand: 8 k from p
  __device__ __forceinline__ void chunk(uint32_t* r, int i, const char* p) const {
    if constexpr (F32) {
      const f32x4_a4 a = *reinterpret_cast<const f32x4_a4*>(p);
      const f32x4_a4 b = *reinterpret_cast<const f32x4_a4*>(p + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[8 * i + e] = __float_as_uint(a[e]);
        r[8 * i + 4 + e] = __float_as_uint(b[e]);
      }
    } else {
      const u32x4_a2 a = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[4 * i + e] = a[e];
    }
  }

  // k number e of a k-strided operand: V columns from p
  __device__ __forceinline__ void vec(uint32_t* r, int e, const char* p) const {
    if constexpr (F32) {
      if constexpr (V == 1) {
        r[e] = *reinterpret_cast<const uint32_t*>(p);
      } else if constexpr (V == 2) {
        const f32x2_a4 a = *reinterpret_cast<const f32x2_a4*>(p);
        r[2 * e] = __float_as_uint(a.x);
        r[2 * e + 1] = __float_as_uint(a.y);
      } else {
        const f32x4_a4 a = *reinterpret_cast<const f32x4_a4*>(p);
#pragma unroll
        for (int v = 0; v < 4; ++v) r[4 * e + v] = __float_as_uint(a[v]);
      }
    } else {
      if constexpr (V == 1) {
        r[e] = *reinterpret_cast<const bf16_t*>(p);
      } else if constexpr (V == 2) {
        r[e] = *reinterpret_cast<const u32_a2*>(p);
      } else {
        const u32x2_a2 a = *reinterpret_cast<const u32x2_a2*>(p);
        r[2 * e] = a.x;
        r[2 * e + 1] = a.y;
      }
    }
  }

  __device__ __forceinline__ void load_full(Regs& q_, int step) const {
    uint32_t* r = q_.r;
    const char* p = base + step * step_bytes;
    if constexpr (!KS) {
#pragma unroll
      for (int i = 0; i < V; ++i) chunk(r, i, p + off[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) vec(r, e, p + (uint64_t)e * ldb + off[0]);
    }
  }

  // the last step, with kleft < BK: zeros behind.  A chunk that crosses the last k
  // is loaded from the 8 k that end there and shifted; k behind the last one are
  // loaded from it and dropped.  (bf16 forward of 2048 x 2047 x 2048: 44.3 us,
  // element by element 48.7; of 8192 x 4095 x 4096: 334 and 354.)
  __device__ __forceinline__ void load_tail(Regs& q_, int step, int kleft) const {
    uint32_t* r = q_.r;
    const char* p = base + step * step_bytes;
    if constexpr (!KS) {
      const int back = max(0, kc * 8 + 8 - kleft);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        chunk(r, i, p + off[i] - (int64_t)back * (int)sizeof(S));
        constexpr int D = F32 ? 8 : 4;                // dwords of a chunk
        uint32_t* c = r + D * i;
        if constexpr (!F32) {
#pragma unroll
          for (int d = 0; d < D; ++d)
            c[d] = back & 1 ? __builtin_amdgcn_alignbit(d + 1 < D ? c[d + 1] : 0, c[d], 16) : c[d];
        }
#pragma unroll
        for (int b = 1; b < D; b <<= 1) {
          const bool on = back & (F32 ? b : 2 * b);
#pragma unroll
          for (int d = 0; d < D; ++d) c[d] = on ? (d + b < D ? c[d + b] : 0) : c[d];
        }
#pragma unroll
        for (int d = 0; d < D; ++d) c[d] = back < 8 ? c[d] : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int over = max(0, kc * 8 + e - (kleft - 1));
        vec(r, e, p + (int64_t)(e - over) * ldb + off[0]);
        constexpr int D = NR / 8;                     // dwords of a vector
#pragma unroll
        for (int d = 0; d < D; ++d) r[D * e + d] = over ? 0 : r[D * e + d];
      }
    }
  }

  __device__ __forceinline__ uint32_t elem(const char* p) const {
    if constexpr (F32) return *reinterpret_cast<const uint32_t*>(p);
    else return *reinterpret_cast<const bf16_t*>(p);
  }

  // element by element; those outside are zero
  __device__ __forceinline__ void load_single(Regs& q_, int step, int kleft, int tid) const {
    uint32_t* r = q_.r;
    const char* p = base + step * step_bytes;
#pragma unroll
    for (int i = 0; i < NR; ++i) r[i] = 0;
    if constexpr (!KS) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t v = 0;
          if (kc * 8 + e < kleft) v = elem(p + off[i] + e * sizeof(S));
          if constexpr (F32) r[8 * i + e] = v;
          else r[4 * i + e / 2] |= v << (16 * (e & 1));
        }
      }
    } else {
      const int c = (tid % (R / V)) * V;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const char* q = p + (uint64_t)(kc * 8 + e) * ldb + (c + V) * (int)sizeof(S);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          uint32_t w = 0;
          if (kc * 8 + e < kleft && row0 + c + v < rows) w = elem(q + v * sizeof(S));
          if constexpr (F32) r[V * e + v] = w;
          else if constexpr (V == 1) r[e] = w;
          else r[(V / 2) * e + v / 2] |= w << (16 * (v & 1));
        }
      }
    }
  }

  // moves the vectors that cross the last column into place
  __device__ __forceinline__ void shift(Regs& q_, int tid) const {
    uint32_t* r = q_.r;
    const int over = row0 + (tid % (R / V)) * V + V - rows;
    const int sh = over > 0 && over < V ? over : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (F32) {
#pragma unroll
        for (int b = 1; b < V; b <<= 1)
#pragma unroll
          for (int v = 0; v + b < V; ++v) r[V * e + v] = sh & b ? r[V * e + v + b] : r[V * e + v];
      } else if constexpr (V == 2) {
        r[e] >>= 16 * sh;
      } else if constexpr (V == 4) {
        uint64_t w = ((uint64_t)r[2 * e + 1] << 32) | r[2 * e];
        w >>= 16 * sh;
        r[2 * e] = (uint32_t)w;
        r[2 * e + 1] = (uint32_t)(w >> 32);
      }
    }
  }

  // a step that load_full alone serves
  __device__ __forceinline__ bool plain(int step, int k) const {
    return k - step * BK >= BK && aligned && !single;
  }

  __device__ __forceinline__ void load(Regs& q_, int step, int k, int tid) const {
    const int kleft = k - step * BK;
    if (single) {
      load_single(q_, step, kleft, tid);
      return;
    }
    if (kleft < BK) load_tail(q_, step, kleft);
    else load_full(q_, step);
    if constexpr (SHIFT) {
      if (!aligned) shift(q_, tid);
    }
  }

  // the 8 k of chunk i as PL bf16 planes into LDS
  __device__ __forceinline__ void store(const Regs& q_, char* lds, int tid) const {
    const uint32_t* r = q_.r;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int row = KS ? (tid % (R / V)) * V + i : tid / CH + i * (T / CH);
      const int o = lds_off<BK>(row, kc);
      uint32_t h[4];
      if constexpr (F32) {
        float a[4], b[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          a[q] = __uint_as_float(KS ? r[V * (2 * q) + i] : r[8 * i + 2 * q]);
          b[q] = __uint_as_float(KS ? r[V * (2 * q + 1) + i] : r[8 * i + 2 * q + 1]);
        }
#pragma unroll
        for (int p = 0; p < PL; ++p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            h[q] = cvt_pk_bf16(a[q], b[q]);
            a[q] -= __uint_as_float(h[q] << 16);
            b[q] -= __uint_as_float(h[q] & 0xffff0000u);
          }
          *reinterpret_cast<uint4*>(lds + p * (R * BK * 2) + o) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        continue;
      } else if constexpr (KS) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (V == 1) {
            h[q] = r[2 * q] | (r[2 * q + 1] << 16);
          } else {
            const uint32_t a = r[(V / 2) * (2 * q) + i / 2], b = r[(V / 2) * (2 * q + 1) + i / 2];
            h[q] = (i & 1) ? __builtin_amdgcn_perm(b, a, 0x07060302u)
                           : __builtin_amdgcn_perm(b, a, 0x05040100u);
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) h[q] = r[4 * i + q];
      }
      *reinterpret_cast<uint4*>(lds + o) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
};

// ---------------------------------------------------------------------------
// C tile BM x BN per block; WM x WN waves; LDS double buffered: while step t is
// multiplied, the tile of step t + 1 goes from registers to LDS and that of step
// t + 1 + PF is requested; one barrier per step.  PF tiles wait in registers.
// ---------------------------------------------------------------------------
template <typename SA, typename SB, int PA, int PB, bool KA, bool KB, int BM, int BN, int BK,
          int WM, int WN, int PF, int EPI, typename TO>
__global__ __launch_bounds__(WM * WN * 64, 2) void dense_gemm(const GemmP P) {
  constexpr int T = WM * WN * 64;
  constexpr int IM = BM / WM / 16, JN = BN / WN / 16;
  typedef Stage<SA, KA, BM, BK, T, PA> StA;
  typedef Stage<SB, KB, BN, BK, T, PB> StB;
  constexpr int BUF = StA::BYTES + StB::BYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // Blocks go to the 8 XCDs round robin: give each XCD a contiguous range of
  // the work, so neighbouring tiles share its L2
  const int nblk = gridDim.x;
  int w = blockIdx.x;
  {
    const int per = nblk >> 3, cut = per << 3;
    if (w < cut) w = (w & 7) * per + (w >> 3);
  }
  const int per_split = P.G * P.tm * P.tn;
  const int split = w / per_split;
  w -= split * per_split;
  const int g = w / (P.tm * P.tn);
  w -= g * P.tm * P.tn;
  // bands of 4 tile rows: consecutive blocks reuse 4 A panels and one B panel
  const int band = w / (4 * P.tn), in = w - band * 4 * P.tn;
  const int bh = min(4, P.tm - band * 4);
  const int tm = band * 4 + in % bh, tn = in / bh;
  // The last tile of a k-strided operand whose extent is no multiple of the vector
  // is moved back to end with it: whole loads, and the rows or columns it shares
  // with its neighbour get the same sums from both.  With single elements for
  // these tiles a bf16 training pass of 2047^3 takes 313 us, so 175, 2048^3 155.
  int m0 = tm * BM, n0 = tn * BN;
  if (KA && P.m >= BM && P.m % StA::V) m0 = min(m0, P.m - BM);
  if (KB && P.n >= BN && P.n % StB::V) n0 = min(n0, P.n - BN);

  StA sa;
  StB sb;
  sa.init(reinterpret_cast<const SA*>(P.a) + g * P.a_gs, P.lda, m0, P.m, P.k, tid);
  sb.init(reinterpret_cast<const SB*>(P.b) + g * P.b_gs, P.ldb, n0, P.n, P.k, tid);

  const int total = (P.k + BK - 1) / BK;
  const int s0 = split * P.steps;
  const int s1 = min(total, s0 + P.steps);

  f32x4 acc[IM][JN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < JN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  const int fr = lane & 15, fc = lane >> 4;

  auto mma = [&](const char* cur, int kk) {
    bf16x8 bf[JN][PB];
#pragma unroll
    for (int j = 0; j < JN; ++j)
#pragma unroll
      for (int p = 0; p < PB; ++p)
        bf[j][p] = *reinterpret_cast<const bf16x8*>(cur + StA::BYTES + p * (BN * BK * 2) +
                                                    lds_off<BK>(wn + j * 16 + fr, kk * 4 + fc));
#pragma unroll
    for (int i = 0; i < IM; ++i) {
      bf16x8 af[PA];
#pragma unroll
      for (int p = 0; p < PA; ++p)
        af[p] = *reinterpret_cast<const bf16x8*>(cur + p * (BM * BK * 2) +
                                                 lds_off<BK>(wm + i * 16 + fr, kk * 4 + fc));
      // operands swapped: a lane ends with 4 neighbouring columns of a row
#pragma unroll
      for (int t = 2; t >= 0; --t)
#pragma unroll
        for (int p = PA - 1; p >= 0; --p) {
          if (t - p < 0 || t - p >= PB) continue;
#pragma unroll
          for (int j = 0; j < JN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[j][t - p], af[p], acc[i][j], 0,
                                                                0, 0);
        }
    }
  };

  typename StA::Regs ra[PF];
  typename StB::Regs rb[PF];
  auto load = [&](int q, int s) {
    sa.load(ra[q], s, P.k, tid);
    sb.load(rb[q], s, P.k, tid);
  };
  auto store = [&](int q, char* buf) {
    sa.store(ra[q], buf, tid);
    sb.store(rb[q], buf + StA::BYTES, tid);
  };
  if (s0 < s1) {
    // tile s0 + i waits in registers i % PF
    load(0, s0);
    store(0, smem);
#pragma unroll
    for (int i = 1; i <= PF; ++i)
      if (s0 + i < s1) load(i % PF, s0 + i);
    __syncthreads();
    int s = s0;
    char *cur = smem, *nxt = smem + BUF;
    // steps whose requests stay inside both operands: no branch between the
    // multiplications, the stores and the requests
    for (; s + 2 * PF < s1 && sa.plain(s + 2 * PF, P.k) && sb.plain(s + 2 * PF, P.k); s += PF) {
#pragma unroll
      for (int u = 0; u < PF; ++u) {
        mma(cur, 0);
        store((u + 1) % PF, nxt);
        sa.load_full(ra[(u + 1) % PF], s + u + 1 + PF);
        sb.load_full(rb[(u + 1) % PF], s + u + 1 + PF);
#pragma unroll
        for (int kk = 1; kk < BK / 32; ++kk) mma(cur, kk);
        // Spread the step's other work between its multiplications: 4 MFMAs, a
        // fragment read, some of the splitting and addressing, then the writes
        // and the requests one by one.  Left alone the compiler runs them in a
        // piece, in which the matrix cores wait (8192 x 4096 x 4096 bf16: NT 307
        // -> 257 us, wgrad 300 -> 259 us; the bf16 dgrad is better left alone,
        // 242 us against 261 us)
        if constexpr (!(PA + PB == 2 && !KA && KB)) {
          constexpr int TERMS = PA * PB == 9 ? 6 : PA * PB, PRE = JN * PB + PA;
          constexpr int NM = IM * JN * TERMS * (BK / 32);
          constexpr int NR = (IM * PA + JN * PB) * (BK / 32) - PRE;
          constexpr int NW = StA::V * PA + StB::V * PB;
          __builtin_amdgcn_sched_group_barrier(0x100, PRE, 0);          // LDS reads
#pragma unroll
          for (int q = 0; q < NM / 4; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);          // MFMA
            if (q < NR) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, KA ? 4 : 8, 0); // VALU
            if (q >= 2 && q < 2 + NW) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
            if (q >= 2 + NW) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);           // request
          }
        }
        __syncthreads();
        char* t = cur;
        cur = nxt;
        nxt = t;
      }
    }
    for (; s < s1; s += PF) {
#pragma unroll
      for (int u = 0; u < PF; ++u) {
        if (s + u < s1) {
          if (s + u + 1 < s1) {
            store((u + 1) % PF, nxt);
            if (s + u + 1 + PF < s1) load((u + 1) % PF, s + u + 1 + PF);
          }
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk) mma(cur, kk);
          __syncthreads();
          char* t = cur;
          cur = nxt;
          nxt = t;
        }
      }
    }
  }

  // Each wave turns its tile through LDS, 16 * ER rows at a time, so that its 64
  // lanes finish and store whole row segments; the loop keeps the epilogue's
  // code (activation, residual) short.  A turn's residual is requested a turn
  // ahead and waits in LDS: loads in the loop, which stay behind its stores, would
  // be waited for one by one (bf16 8192 x 4096 x 4096 with gelu and act': 384 -> 355
  // us; 376 us since gelu is exact to fp32).
  constexpr int WC = BN / WN, PITCH = WC + 4, ER = IM < 2 ? 1 : 2;
  constexpr int LC = WC / 4, RS = 64 / LC, SN = 16 * ER / RS;   // lanes a row, rows a step, steps
  static_assert(IM % ER == 0, "rows of a turn");
  float* turn = reinterpret_cast<float*>(smem) + wave * (16 * ER * PITCH);
  typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(TO))));   // 4 elements
  Raw* wait = reinterpret_cast<Raw*>(smem + WM * WN * 16 * ER * PITCH * 4) + wave * SN * 64 + lane;
  const int col = n0 + wn + (lane % LC) * 4, row1 = m0 + wm + lane / LC;
  const bool have = EPI == EPI_FWD && P.res && P.splits == 1 && col < P.n;
  float bias[4] = {};
  Raw ahead[SN];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int s = 0; s < SN; ++s) {
      const TO* p = at_res<TO>(P, g, min(row1 + i0 * 16 + s * RS, P.m - 1), col);
      if (col + 4 <= P.n) {
        __builtin_memcpy(&ahead[s], p, sizeof(Raw));
      } else {
        TO v[4] = {};
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (col + i < P.n) v[i] = p[i];
        __builtin_memcpy(&ahead[s], v, sizeof(Raw));
      }
    }
  };
  if constexpr (EPI == EPI_FWD) {
    if (col < P.n && P.splits == 1) ld_bias<TO>(P, g, col, P.n - col, bias);
    if (have) fetch(0);
  }
#pragma unroll
  for (int i0 = 0; i0 < IM; i0 += ER) {
#pragma unroll
    for (int i = 0; i < ER; ++i)
#pragma unroll
      for (int j = 0; j < JN; ++j)
        *reinterpret_cast<f32x4*>(turn + (i * 16 + fr) * PITCH + j * 16 + fc * 4) = acc[i0 + i][j];
    if constexpr (EPI == EPI_FWD) {
      if (have) {
#pragma unroll
        for (int s = 0; s < SN; ++s) wait[s * 64] = ahead[s];
        if (i0 + ER < IM) fetch(i0 + ER);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (col < P.n) {
#pragma unroll 2
      for (int s = 0; s < SN; ++s) {
        const int row = row1 + i0 * 16 + s * RS;
        if (row >= P.m) break;
        const f32x4 t = *reinterpret_cast<const f32x4*>(turn + (lane / LC + s * RS) * PITCH +
                                                        (lane % LC) * 4);
        float z[4] = {t[0], t[1], t[2], t[3]};
        if (P.splits > 1) {
          st4(P.part + (((int64_t)split * P.G + g) * P.m + row) * P.n + col, z, P.n - col);
        } else {
          float r[4] = {};
          if (have) {
            const Raw w = wait[s * 64];
            TO v[4];
            __builtin_memcpy(v, &w, sizeof(Raw));
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = to_f(v[i]);
          }
          epilogue<EPI, TO>(P, g, row, col, P.n - col, z, bias, r);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// ---------------------------------------------------------------------------
// The forward of a few rows (serving: one row), M <= 8.  One pass over the
// weights, which bound it: lanes along k, 16 B of each of NC weight rows per
// step, products and sums in fp32 (no planes), one launch -- the MFMA tiles need
// the reduction split over blocks to fill the chip and a second launch to join
// it.  KW waves share a column's k where there are few columns.
//
// us, this kernel / the MFMA tiles (weights in turn from 3 copies):
//                      M 1          M 2          M 4          M 8
//   4096 x 4096 bf16    7.3 / 13.4   7.6 / 13.3  12.8 / 13.2  15.8 / 13.4
//   4096 x 4096 fp32   12.4 / 21.5  12.5 / 21.5  14.6 / 21.4  28.8 / 22.0
//   8 x 4608 x 4096 b  47.0 / 44.7  46.3 / 44.3  83.6 / 44.3  83.4 / 44.5
//   8 x 4608 x 4096 f   101 / 110    105 / 109    107 / 109    177 / 109
//   2048 x 1000 bf16    5.1 /  8.9   4.5 /  9.1   4.9 /  9.3   6.0 /  9.7
//   8192 x 64 fp32      4.6 / 16.9   5.0 / 15.7   5.1 / 16.6   6.3 / 16.4
//   100 x 8000 bf16     5.5 /  5.2   6.0 /  5.2   7.5 /  5.1  11.1 /  5.3
//   100 x 60000 bf16   15.2 /  7.6  19.9 /  7.7
//   104 x 8000 bf16     4.0 /  4.5   4.4 /  4.5
//   300 x 8000 bf16     5.2 /  5.8   5.9 /  5.9
//   301 x 60000 bf16   18.6 / 13.6  23.9 / 16.1
//   516 x 60000 bf16   20.6 / 19.6  23.8 / 19.6
//   1537 x 40000 bf16  24.6 / 32.5  28.8 / 37.8
//   300 x 60000 fp32   15.2 / 28.3  17.4 / 28.2
// With more rows the products on the vector units weigh more than the second
// launch, the sooner the more weights there are; and a short bf16 row that ends
// inside a vector spends as long on its last elements as on all others, which many
// columns cannot hide: gemv_better.
// ---------------------------------------------------------------------------
constexpr int GEMV_ROWS = 8;

static inline bool gemv_better(int M, int N, int K, int G, int is_bf16) {
  const int64_t bytes = (int64_t)G * N * K * (is_bf16 ? 2 : 4);
  if (M <= 2) return !is_bf16 || K % 8 == 0 || K >= 512 || (int64_t)G * N < 16000;
  if (M <= 4) return K >= 512 && (!is_bf16 || bytes <= (32 << 20));
  return M <= GEMV_ROWS && K >= 512 && bytes <= (8 << 20);
}

template <typename T, int MT, int NC, int KW>
__global__ __launch_bounds__(256) void dense_gemv(const GemmP P) {
  constexpr int V = 16 / sizeof(T), CW = 4 / KW;        // column groups of a block
  __shared__ float sm[KW > 1 ? 4 * NC * MT : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (P.n + CW * NC - 1) / (CW * NC);
  const int g = blockIdx.x / per, blk = blockIdx.x - g * per;
  const int col = (blk * CW + wave / KW) * NC;
  const T* x = reinterpret_cast<const T*>(P.a) + g * P.a_gs;
  const T* w[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)       // columns past the last: the last one's weights
    w[c] = reinterpret_cast<const T*>(P.b) + g * P.b_gs + (int64_t)min(col + c, P.n - 1) * P.ldb;
  float acc[MT][NC];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = 0.f;

  auto step = [&](int k, auto ld) {
    float wv[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c) ld(w[c] + k, wv[c]);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float xv[V];
      ld(x + min(m, P.m - 1) * P.lda + k, xv);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[m][c] = fmaf(xv[e], wv[c][e], acc[m][c]);
    }
  };
  auto whole = [](const T* p, float* v) {
#pragma unroll
    for (int e = 0; e < V; e += 4) ld4(p + e, v + e, 4);
  };
  int k = ((wave % KW) * 64 + lane) * V;
#pragma unroll 2
  for (; k + V <= P.k; k += KW * 64 * V) step(k, whole);
  if (k < P.k)
    step(k, [&](const T* p, float* v) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = k + e < P.k ? ld1(p + e) : 0.f;
    });

#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = warp_sum(acc[m][c]);
  if constexpr (KW > 1) {
    if (lane == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < NC; ++c) sm[(wave * MT + m) * NC + c] = acc[m][c];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) s += sm[(q * MT + m) * NC + c];
        acc[m][c] = s;
      }
  }
  // lane m finishes row m
  if (col >= P.n || lane >= P.m) return;
  float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MT; ++m)
    if (lane == m) {
#pragma unroll
      for (int c = 0; c < NC; ++c) z[c] = acc[m][c];
    }
  epilogue<EPI_FWD, T>(P, g, lane, col, min(NC, P.n - col), z);
}

template <typename T, int MT>
static int launch_gemv(const GemmP& P, hipStream_t st) {
  // columns of a wave: as many as leave 512 waves; where even one leaves fewer
  // than 256 blocks and k is long, the four waves of a block share it
  const int64_t cols = (int64_t)P.G * P.n;
  auto go = [&](auto kern, int per_block) {
    const int64_t blocks = (int64_t)P.G * ((P.n + per_block - 1) / per_block);
    if (blocks > 0x7fffffff) return (int)hipErrorInvalidValue;
    kern<<<(int)blocks, 256, 0, st>>>(P);
    return (int)hipGetLastError();
  };
  constexpr int NM = MT > 4 ? 2 : 4;          // registers: MT * NC sums
  if (cols >= 4 * 512 * NM) return go(dense_gemv<T, MT, NM, 1>, 4 * NM);
  if (cols < 4 * 256 && P.k >= 1024) return go(dense_gemv<T, MT, 1, 4>, 1);
  return go(dense_gemv<T, MT, 1, 1>, 4);
}

// sums the split-K partials in split order (the result does not depend on
// which block finished first) and runs the epilogue
template <int EPI, typename TO>
__global__ __launch_bounds__(256) void dense_join(const GemmP P) {
  const int nq = (P.n + 3) / 4;
  const int64_t total = (int64_t)P.G * P.m * nq;
  const int64_t slab = (int64_t)P.G * P.m * P.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t rr = i / nq;
    const int col = (int)(i - rr * nq) * 4;
    const int g = (int)(rr / P.m), row = (int)(rr - (int64_t)g * P.m);
    const float* q = P.part + rr * P.n + col;
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < P.splits; ++s, q += slab) {
      float v[4];
      ld4(q, v, P.n - col);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] += v[e];
    }
    epilogue<EPI, TO>(P, g, row, col, P.n - col, z);
  }
}

// ---------------------------------------------------------------------------
// dz = dy * act'(z) and the column sums of dz (db).  Blocks own 64 columns x a
// range of rows; the partial sums of several row ranges meet in dense_dbsum in
// a fixed order.
// ---------------------------------------------------------------------------
constexpr int DA_COLS = 64;
// rows of a block: 128, more where that keeps the ranges to 4096
static inline int dact_rows(int M) { return M <= 128 * 4096 ? 128 : (M + 4095) / 4096; }

// D: 0 none (dz is dy, only db is made), 1 u8 mask, 2 fp32 derivative
template <typename T, int D, typename TZ>
__global__ __launch_bounds__(256) void dense_dact(const T* __restrict__ dy, const void* __restrict__ d,
                                                  TZ* __restrict__ dz, float* __restrict__ db,
                                                  int64_t db_gs, float* __restrict__ part, int M,
                                                  int C, int N, int rows) {
  __shared__ float sm[4][DA_COLS];
  const int c = blockIdx.x * DA_COLS + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const int r0 = blockIdx.y * rows, r1 = min(M, r0 + rows);
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int r = r0 + w; r < r1; r += 4) {
      const int64_t i = (int64_t)r * C + c;
      float v = ld1(dy + i);
      if constexpr (D == 1) v = reinterpret_cast<const uint8_t*>(d)[i] ? v : 0.f;
      if constexpr (D == 2) v *= reinterpret_cast<const float*>(d)[i];
      if constexpr (D != 0) st1(dz + i, v);
      s += v;
    }
  }
  if (!db) return;
  sm[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < C) {
    s = (sm[0][threadIdx.x] + sm[1][threadIdx.x]) + (sm[2][threadIdx.x] + sm[3][threadIdx.x]);
    if (gridDim.y > 1) part[(int64_t)blockIdx.y * C + c] = s;
    else db[(c / N) * db_gs + c % N] = s;
  }
}

__global__ __launch_bounds__(256) void dense_dbsum(const float* __restrict__ part, int rows,
                                                   float* __restrict__ db, int64_t db_gs, int C,
                                                   int N) {
  __shared__ float sm[4][DA_COLS];
  const int c = blockIdx.x * DA_COLS + (threadIdx.x & 63), w = threadIdx.x >> 6;
  float s = 0.f;
  if (c < C)
    for (int r = w; r < rows; r += 4) s += part[(int64_t)r * C + c];
  sm[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < C)
    db[(c / N) * db_gs + c % N] =
        (sm[0][threadIdx.x] + sm[1][threadIdx.x]) + (sm[2][threadIdx.x] + sm[3][threadIdx.x]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
enum { T_BIG, T_MID, T_SMALL, T_THIN };

struct Plan {
  int tile, tm, tn, splits, steps;
};

// tile sizes by the planes of both operands together: 2 (bf16), 1 + DZ_PLANES and
// 1 + DX_PLANES (dW and dx of a bf16 layer with a smooth activation), 6 (fp32).
// Two planes leave 2^-16 of dz, which dx's own rounding to bf16 covers: 8192 x 4096
// x 4096 with gelu is 1.66e-3 from 64 bits, as fp32 sums rounded once are (they
// differ by 1.04e-4, with three planes, 160 us more, by 0.77e-4).  One plane is
// 2.35e-3.
constexpr int DZ_PLANES = 3, DX_PLANES = 2;
static constexpr int tile_m(int planes, int t) {
  return t == T_BIG ? (planes == 2 || planes == 6 ? 256 : 128) : t == T_MID ? 128 : t == T_SMALL ? 64 : 32;
}
static constexpr int tile_n(int planes, int t) {
  return t == T_BIG ? (planes == 6 ? 128 : 256) : t == T_MID ? (planes == 6 ? 64 : 128) : 64;
}
static constexpr int tile_k(int planes, int t) {
  return t == T_THIN ? 64 : planes == 2 ? (t == T_MID ? 32 : 64) : 32;
}
static constexpr int tile_threads(int t) { return t == T_BIG ? 512 : 256; }
// blocks of a CU (LDS and registers)
static constexpr int tile_occ(int planes, int t) {
  return t == T_BIG ? 1 : t == T_MID ? 2 : t == T_SMALL ? (planes == 2 ? 4 : 3) : planes == 2 ? 3 : 2;
}

// The tile and the split of the reduction with the least estimated time.  A
// round is as many blocks as the chip holds.  A step of a round costs the
// largest of its MFMA cycles (at the share of the dense peak that the tile
// reaches), its operand bytes (at the rate a CU is fed) and the latency of a
// step; a round also costs its start and its stores, which blocks that share a
// CU hide in each other; partials cost a launch and their traffic.  The
// constants are fitted to 282 products (1 - 16 configurations, 1 - 16384 rows, 2
// - 8192 columns, all three forms, both types), each timed under every tile and
// up to 8 splits: the choice is on average 3 % slower than the best of them,
// against 9 % for the constants that a first guess gave.  splits == 0: no tile
// covers the product in one launch.
static Plan choose_plan(int64_t m, int64_t n, int64_t k, int G, int planes, int out_bytes) {
  const int passes = planes == 6 ? 6 : planes - 1;
  const int esz = planes == 2 ? 2 : 4;
  static const double eff_f32[4] = {0.56, 0.33, 0.34, 0.17}, eff_bf16[4] = {0.40, 0.43, 0.19, 0.09};
  static const double latency[4] = {0.76, 0.69, 0.60, 0.35};       // us of a step
  const double* eff = planes == 2 ? eff_bf16 : eff_f32;
  Plan best = {};
  double best_t = 1e30;
  for (int t = T_BIG; t <= T_THIN; ++t) {
    const int bm = tile_m(planes, t), bn = tile_n(planes, t), bk = tile_k(planes, t);
    const int occ = tile_occ(planes, t);
    const int64_t tm = (m + bm - 1) / bm, tn = (n + bn - 1) / bn;
    const int64_t nt = G * tm * tn, total = (k + bk - 1) / bk;
    const double mfma = 2.0 * bm * bn * bk * passes / 4096.0 / eff[t] / 2400.0;
    const double mem = (double)(bm + bn) * bk * esz / 23.0 / 2400.0;
    for (int64_t s = 1; s <= 16 && s <= (total + 1) / 2; s = s < 4 ? s + 1 : s + s / 3) {
      const int64_t steps = (total + s - 1) / s, sp = (total + steps - 1) / steps;
      const double blocks = (double)nt * sp;
      if (!grid_fits(nt * sp, tile_threads(t))) continue;
      const double rounds = ceil(blocks / (256.0 * occ));
      // a part-filled round runs as fast as its fullest CU
      const double share = rounds > 1 ? occ : ceil(blocks / 256.0);
      double step = share * (mfma > mem ? mfma : mem);
      if (step < latency[t]) step = latency[t];
      const double run = steps * step + 3.9;
      const double store = share * bm * bn * (sp > 1 ? 4 : out_bytes) / 9.4 / 2400.0;
      const double hide = occ > 1 && rounds > 1 ? 0.9 : 0.0;
      double us = rounds * (run + store - hide * (run < store ? run : store));
      if (sp > 1) us += 4.1 + (sp + 1.0) * G * m * n * 4.0 / 7.7e6;
      if (us < best_t) {
        best_t = us;
        best.tile = t;
        best.tm = (int)tm;
        best.tn = (int)tn;
        best.splits = (int)sp;
        best.steps = (int)steps;
      }
    }
  }
  return best;
}

// the last choices of this thread, by sizes (choosing takes a microsecond)
static Plan make_plan(int64_t m, int64_t n, int64_t k, int G, int planes, int out_bytes) {
  struct Entry {
    int64_t key[6];
    Plan plan;
  };
  static thread_local Entry memo[64];
  const int64_t key[6] = {m, n, k, G, planes, out_bytes};
  uint64_t h = 0;
  for (int64_t x : key) h = (h ^ (uint64_t)x) * 0x9e3779b97f4a7c15ull;
  Entry& e = memo[h >> 58];
  bool hit = true;
  for (int i = 0; i < 6; ++i) hit = hit && e.key[i] == key[i];
  if (!hit) {
    e.plan = choose_plan(m, n, k, G, planes, out_bytes);
    for (int i = 0; i < 6; ++i) e.key[i] = key[i];
  }
  return e.plan;
}

template <typename SA, typename SB, int PA, int PB, bool KA, bool KB, int BM, int BN, int BK, int WM,
          int WN, int PF, int EPI, typename TO>
static int launch_gemm(GemmP& P, const Plan& p, hipStream_t st) {
  P.tm = p.tm;
  P.tn = p.tn;
  P.splits = p.splits;
  P.steps = p.steps;
  const int64_t blocks = (int64_t)P.G * p.tm * p.tn * p.splits;
  if (p.splits < 1 || !grid_fits(blocks, WM * WN * 64)) return (int)hipErrorInvalidValue;
  constexpr int stage = 2 * (PA * BM + PB * BN) * BK * 2;
  // the epilogue's: sums, and the residual that waits
  constexpr int turn = WM * WN * (BM / WM < 32 ? 16 : 32) *
                       ((BN / WN + 4) * 4 + (EPI == EPI_FWD ? BN / WN * (int)sizeof(TO) : 0));
  constexpr int lds = stage > turn ? stage : turn;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  auto kern = dense_gemm<SA, SB, PA, PB, KA, KB, BM, BN, BK, WM, WN, PF, EPI, TO>;
  if (lds > 64 * 1024) {
    // once per device
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && !(done.load() >> (dev & 63) & 1)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e == hipSuccess) done.fetch_or((uint64_t)1 << (dev & 63));
    }
    if (e != hipSuccess) return (int)e;
  }
  kern<<<(int)blocks, WM * WN * 64, lds, st>>>(P);
  if (p.splits > 1) {
    const int64_t q = (int64_t)P.G * P.m * ((P.n + 3) / 4);
    int64_t b = (q + 255) / 256;
    if (b > 4096) b = 4096;
    dense_join<EPI, TO><<<(int)b, 256, 0, st>>>(P);
  }
  return (int)hipGetLastError();
}

template <typename SA, typename SB, int PA, int PB, bool KA, bool KB, int EPI, typename TO>
static int run_gemm(GemmP& P, const Plan& p, hipStream_t st) {
  constexpr int PL = PA + PB;
  // Two steps of the small tile in registers where both operands lie along k: fp32
  // forward of 1024^3 28.3 -> 27.1 us.  The transposing loads take more addresses,
  // and two steps of them cost more than they hide (fp32 dgrad of 8 x 32 x 4608 x
  // 4096: 199 -> 203 us), as in the larger tiles.
  constexpr int PF_SMALL = KA || KB ? 1 : 2;
#define CER_TILE(T, WM, WN, PF)                                                                   \
  launch_gemm<SA, SB, PA, PB, KA, KB, tile_m(PL, T), tile_n(PL, T), tile_k(PL, T), WM, WN, PF, EPI, \
              TO>(P, p, st)
  switch (p.tile) {
    case T_BIG: return CER_TILE(T_BIG, (PL == 6 ? 4 : 2), (PL == 6 ? 2 : 4), 1);
    case T_MID: return CER_TILE(T_MID, 2, 2, 1);
    case T_SMALL: return CER_TILE(T_SMALL, 2, 2, PF_SMALL);
    default: return CER_TILE(T_THIN, 1, 4, 3);
  }
#undef CER_TILE
}

static inline int planes_of(int kind, int is_bf16, int act) {
  if (!is_bf16) return 6;
  if (kind == 0 || !act_smooth(act)) return 2;
  return 1 + (kind == 2 ? DZ_PLANES : DX_PLANES);
}

static inline Plan plan_of(int kind, int M, int N, int K, int G, int is_bf16, int act) {
  const int pl = planes_of(kind, is_bf16, act);
  const int out = is_bf16 ? 2 : 4;
  if (kind == 0) return make_plan(M, N, K, G, pl, out);
  if (kind == 1) return make_plan(M, K, N, G, pl, out);
  return make_plan(N, K, M, G, pl, 4);
}

static inline bool sizes_ok(int M, int N, int K, int G, int64_t ldx) {
  // byte offsets inside a tile are 32-bit: 255 rows of the longest pitch and a
  // chunk.  Row numbers are ints, also those of the last tile and of the last of
  // 4096 row ranges, 2^19 rows and more past M
  const int64_t most = ((int64_t)1 << 32) / (256 * 4);
  return M > 0 && M <= 0x7fffffff - (1 << 20) && N > 0 && K > 0 && G > 0 && (int64_t)G * N < most && (int64_t)G * K < most &&
         N < most && K < most && ldx >= (int64_t)G * K && ldx < most;
}

// fp32 workspace (floats) of a call: kind 0 forward, 1 backward; 0 for none,
// -1 for sizes out of range
CER_API int64_t cer_dense_ws(int kind, int M, int N, int K, int G, int is_bf16, int act) {
  if (!sizes_ok(M, N, K, G, (int64_t)G * K) || !act_known(act)) return -1;
  auto need = [&](int kd, int64_t m, int64_t n) {
    const Plan p = plan_of(kd, M, N, K, G, is_bf16, act);
    return p.splits < 1 ? -1 : p.splits > 1 ? (int64_t)p.splits * G * m * n : 0;
  };
  if (kind == 0) return gemv_better(M, N, K, G, is_bf16) ? 0 : need(0, M, N);
  const int64_t a = need(1, M, K), b = need(2, N, K);
  if (a < 0 || b < 0) return -1;
  const int64_t nb = (M + dact_rows(M) - 1) / dact_rows(M);
  const int64_t c = nb > 1 ? nb * G * N : 0;
  return a > b ? (a > c ? a : c) : (b > c ? b : c);
}

// y = r + act(x W^T + b).  x: row pitch ldx, config g at column g K; W, b: per-
// config strides ws, bs (elements); r, y, d: [M][G N], r with row pitch ldr.
// d (or null): act'(z), fp32 for the smooth activations, u8 for relu / relu6.
template <typename T>
static int dense_fwd(const T* x, int64_t ldx, const T* w, int64_t ws, const T* b, int64_t bs,
                     const T* r, int64_t ldr, T* y, void* d, int M, int N, int K, int G, int act,
                     float* part, int64_t part_floats, hipStream_t st) {
  if (!sizes_ok(M, N, K, G, ldx) || !act_known(act) || !x || !w || !y)
    return (int)hipErrorInvalidValue;
  constexpr int is_bf16 = sizeof(T) == 2;
  if (part_floats < cer_dense_ws(0, M, N, K, G, is_bf16, act)) return (int)hipErrorInvalidValue;
  GemmP P = {};
  P.a = x; P.lda = ldx; P.a_gs = K;
  P.b = w; P.ldb = K; P.b_gs = ws;
  P.m = M; P.n = N; P.k = K; P.G = G;
  P.c = y; P.ldc = (int64_t)G * N; P.c_gs = N;
  P.bias = b; P.bias_gs = bs;
  P.res = r; P.ldr = ldr;
  P.d = act == ACT_NONE ? nullptr : d;
  P.act = act;
  P.part = part;
  if (gemv_better(M, N, K, G, is_bf16)) {
    if (M == 1) return launch_gemv<T, 1>(P, st);
    if (M == 2) return launch_gemv<T, 2>(P, st);
    if (M <= 4) return launch_gemv<T, 4>(P, st);
    return launch_gemv<T, GEMV_ROWS>(P, st);
  }
  const Plan p = plan_of(0, M, N, K, G, is_bf16, act);
  constexpr int PL = is_bf16 ? 1 : 3;
  return run_gemm<T, T, PL, PL, false, false, EPI_FWD, T>(P, p, st);
}

// gradients: dx (or null) [M][G K], dW -> gw (fp32, config stride gs),
// db -> gb (or null).  d: act'(z) of the forward; dz: scratch [M][G N] (T for
// relu / relu6, fp32 for the smooth activations, unused for act none).
template <typename T>
static int dense_bwd(const T* dy, const void* d, void* dz, const T* x, int64_t ldx, const T* w,
                     int64_t ws, T* dx, float* gw, int64_t gs, float* gb, int64_t gbs, int M, int N,
                     int K, int G, int act, float* part, int64_t part_floats, hipStream_t st) {
  if (!sizes_ok(M, N, K, G, ldx) || !act_known(act) || !dy || !x || !w || !gw)
    return (int)hipErrorInvalidValue;
  if (act != ACT_NONE && (!d || !dz)) return (int)hipErrorInvalidValue;
  constexpr int is_bf16 = sizeof(T) == 2;
  if (part_floats < cer_dense_ws(1, M, N, K, G, is_bf16, act)) return (int)hipErrorInvalidValue;
  const int C = G * N;
  const bool smooth = act_smooth(act);
  if (act != ACT_NONE || gb) {
    const int rows = dact_rows(M);
    const dim3 grid((C + DA_COLS - 1) / DA_COLS, (M + rows - 1) / rows);
    if (act == ACT_NONE)
      dense_dact<T, 0, T><<<grid, 256, 0, st>>>(dy, nullptr, nullptr, gb, gbs, part, M, C, N, rows);
    else if (smooth)
      dense_dact<T, 2, float><<<grid, 256, 0, st>>>(dy, d, (float*)dz, gb, gbs, part, M, C, N,
                                                      rows);
    else
      dense_dact<T, 1, T><<<grid, 256, 0, st>>>(dy, d, (T*)dz, gb, gbs, part, M, C, N, rows);
    if (gb && grid.y > 1)
      dense_dbsum<<<grid.x, 256, 0, st>>>(part, grid.y, gb, gbs, C, N);
  }
  const void* z = act == ACT_NONE ? (const void*)dy : dz;
  int rc;
  {
    GemmP P = {};
    P.a = z; P.lda = C; P.a_gs = N;
    P.b = x; P.ldb = ldx; P.b_gs = K;
    P.m = N; P.n = K; P.k = M; P.G = G;
    P.c = gw; P.ldc = K; P.c_gs = gs;
    P.part = part;
    const Plan p = plan_of(2, M, N, K, G, is_bf16, act);
    if constexpr (!is_bf16)
      rc = run_gemm<float, float, 3, 3, true, true, EPI_F32, float>(P, p, st);
    else if (smooth)
      rc = run_gemm<float, bf16_t, DZ_PLANES, 1, true, true, EPI_F32, float>(P, p, st);
    else
      rc = run_gemm<bf16_t, bf16_t, 1, 1, true, true, EPI_F32, float>(P, p, st);
    if (rc) return rc;
  }
  if (!dx) return 0;
  GemmP P = {};
  P.a = z; P.lda = C; P.a_gs = N;
  P.b = w; P.ldb = K; P.b_gs = ws;
  P.m = M; P.n = K; P.k = N; P.G = G;
  P.c = dx; P.ldc = (int64_t)G * K; P.c_gs = K;
  P.part = part;
  const Plan p = plan_of(1, M, N, K, G, is_bf16, act);
  if constexpr (is_bf16)
    if (smooth) return run_gemm<float, T, DX_PLANES, 1, false, true, EPI_T, T>(P, p, st);
  constexpr int PL = is_bf16 ? 1 : 3;
  return run_gemm<T, T, PL, PL, false, true, EPI_T, T>(P, p, st);
}

#define CER_DENSE(T, F, B)                                                                         \
  CER_API CER_DENSE_FWD(F) {                                                                       \
    return dense_fwd((const T*)x, ldx, (const T*)w, ws, (const T*)b, bs, (const T*)r, ldr, (T*)y,  \
                     d, M, N, K, G, act, part, part_floats, st);                                   \
  }                                                                                                \
  CER_API CER_DENSE_BWD(B) {                                                                       \
    return dense_bwd((const T*)dy, d, dz, (const T*)x, ldx, (const T*)w, ws, (T*)dx, gw, gs, gb,   \
                     gbs, M, N, K, G, act, part, part_floats, st);                                 \
  }
CER_DENSE(bf16_t, cer_dense_fwd, cer_dense_bwd)
CER_DENSE(float, cer_dense_fwd_f32, cer_dense_bwd_f32)
