// Norm of queries and keys for each head with the position rotation in the same pass, forward and backward.
//
//   r = (mean_c x_c^2 + eps)^(-1/2)     n_c = x_c r     u_c = n_c w_c
//   y = u with every pair (a, b) of the first R channels turned by the angle  position[axis(pair)] * freq[pair]:
//       y_a = u_a cos - u_b sin,  y_b = u_b cos + u_a sin
// pairs: (i, i + R / 2), or (2 i, 2 i + 1) when `interleaved`; pair i < R / 2 belongs to axis i / (R / 2 / axes).
// backward, with g = dy turned back:  dw_c = sum over rows of g_c n_c;  dx = r (g w - n mean_c(g_c w_c n_c)).
//
// Bound: memory (x read, y written; backward reads x and dy and writes dx; r is recomputed, nothing is saved but the inputs).
// A row (one head of one token) belongs to D / (2 V) neighbouring lanes; a lane holds the V channels of one 16-byte chunk and the V
// channels that are turned with them (V = 8 bf16 / 4 fp32; chunks of four when D or R is an odd multiple of 8), so a rotation needs no
// exchange and a norm needs log2(lanes) ones.  The angles depend on the token only: a lane makes its V sines and cosines once and walks
// over `hc` heads with them (they cost some 60 instructions each, as much as eight rows' arithmetic).
//
// Angles: position * freq in 64 bits, reduced to a quarter turn there (positions of 10^6 keep 10 digits of angle), sine and cosine of the
// remainder in 32 bits.
#include "common.h"

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

template <typename T, int V>
struct qkn_vec {
  typedef __attribute__((ext_vector_type(V))) T mem;
  typedef __attribute__((ext_vector_type(V))) float f32;
  static __device__ __forceinline__ f32 load(const T* p) { return __builtin_convertvector(*(const mem*)p, f32); }
  static __device__ __forceinline__ void store(T* p, f32 x) { *(mem*)p = __builtin_convertvector(x, mem); }
};
// the two chunks of a lane: one access of 2 V values when they are neighbours (PAIRS), two of V otherwise
template <typename T, int V, bool PAIRS>
__device__ __forceinline__ void qkn_load(const T* p, int c0, int c1, typename qkn_vec<T, V>::f32& a, typename qkn_vec<T, V>::f32& b) {
  if constexpr (PAIRS) {
    const typename qkn_vec<T, 2 * V>::f32 x = qkn_vec<T, 2 * V>::load(p + c0);
#pragma unroll
    for (int e = 0; e < V; ++e) { a[e] = x[e]; b[e] = x[V + e]; }
  } else {
    a = qkn_vec<T, V>::load(p + c0);
    b = qkn_vec<T, V>::load(p + c1);
  }
}
template <typename T, int V, bool PAIRS>
__device__ __forceinline__ void qkn_store(T* p, int c0, int c1, typename qkn_vec<T, V>::f32 a, typename qkn_vec<T, V>::f32 b) {
  if constexpr (PAIRS) {
    typename qkn_vec<T, 2 * V>::f32 x;
#pragma unroll
    for (int e = 0; e < V; ++e) { x[e] = a[e]; x[V + e] = b[e]; }
    qkn_vec<T, 2 * V>::store(p + c0, x);
  } else {
    qkn_vec<T, V>::store(p + c0, a);
    qkn_vec<T, V>::store(p + c1, b);
  }
}

#define QKN_MAX_BLOCKS 1024           // persistent workgroups of the backward, per side

struct qkn_side {
  const void *x, *pos, *dy;
  int64_t sb, st, sh, p_sb, p_st, p_sa;
  const float* w;
  void *y, *dx;
  int T, H, chunks, blocks;       // chunks of hc heads per token; workgroups of this side
};
struct qkn_args {
  qkn_side s[2];
  const double* freq;
  float* part;                    // backward: (workgroup, D) partial weight gradients
  int B, D, R, axes, interleaved, pos64, hc, lanes;   // lanes per row, a power of two
  float eps;
};

// the lane's two chunks and whether they rotate; pair e of the lane is (chunk 0, e)-(chunk 1, e), or neighbours when interleaved
template <int V, bool PAIRS>
struct qkn_lane {
  int c0, c1, pair;
  bool on, rot;
  __device__ __forceinline__ qkn_lane(const qkn_args& p, int j) {
    on = j < p.D / (2 * V);
    rot = j < p.R / (2 * V);
    pair = V * j;
    if (!rot) { c0 = 2 * V * j; c1 = c0 + V; }
    else if (PAIRS) { c0 = 2 * V * j; c1 = c0 + V; }
    else { c0 = V * j; c1 = p.R / 2 + V * j; }
  }
};

template <int V, bool PAIRS>
__device__ __forceinline__ void qkn_angles(const qkn_args& p, const qkn_side& s, const qkn_lane<V, PAIRS>& ln, int b, int t, float* cs, float* sn) {
#pragma unroll
  for (int e = 0; e < V; ++e) { cs[e] = 1.f; sn[e] = 0.f; }
  if (!ln.rot) return;
  const int per = p.R / 2 / p.axes;
  const int64_t at = b * s.p_sb + t * s.p_st;
  const double p0 = p.pos64 ? (double)((const int64_t*)s.pos)[at] : (double)((const int32_t*)s.pos)[at];
  const int64_t at1 = at + (p.axes - 1) * s.p_sa;
  const double p1 = p.pos64 ? (double)((const int64_t*)s.pos)[at1] : (double)((const int32_t*)s.pos)[at1];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const double turns4 = (ln.pair + e < per ? p0 : p1) * p.freq[ln.pair + e] * 0.63661977236758134308;     // quarter turns: angle * 2 / pi
    const double whole = rint(turns4);
    const int quad = (int)((int64_t)whole & 3);
    float sf, cf;
    sincospif((float)(turns4 - whole) * 0.5f, &sf, &cf);
    const float a = (quad & 1) ? sf : cf, c = (quad & 1) ? cf : sf;
    cs[e] = (quad == 1 || quad == 2) ? -a : a;
    sn[e] = quad >= 2 ? -c : c;
  }
}

template <typename F, int V, bool PAIRS>
__device__ __forceinline__ void qkn_turn(F& a, F& b, const float* cs, const float* sn, float sign) {
  if constexpr (!PAIRS) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x = a[e], y = b[e], s = sign * sn[e];
      a[e] = fmaf(x, cs[e], -y * s);
      b[e] = fmaf(y, cs[e], x * s);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const float x = a[2 * e], y = a[2 * e + 1], s = sign * sn[e];
      a[2 * e] = fmaf(x, cs[e], -y * s);
      a[2 * e + 1] = fmaf(y, cs[e], x * s);
      const float x1 = b[2 * e], y1 = b[2 * e + 1], s1 = sign * sn[V / 2 + e], k1 = cs[V / 2 + e];
      b[2 * e] = fmaf(x1, k1, -y1 * s1);
      b[2 * e + 1] = fmaf(y1, k1, x1 * s1);
    }
  }
}

__device__ __forceinline__ float qkn_row_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename T, int V, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_kernel(qkn_args p) {
  typedef typename qkn_vec<T, V>::f32 F;
  const int side = blockIdx.x >= p.s[0].blocks;
  const qkn_side s = p.s[side];
  const int blk = blockIdx.x - (side ? p.s[0].blocks : 0);
  const int groups = 256 / p.lanes, j = threadIdx.x & (p.lanes - 1);
  const int64_t u = (int64_t)blk * groups + threadIdx.x / p.lanes;
  if (u >= (int64_t)p.B * s.T * s.chunks) return;               // whole groups of lanes leave together
  const uint32_t tk = (uint32_t)u / (uint32_t)s.chunks;         // (the host keeps units below 2^31)
  const int chunk = (int)((uint32_t)u - tk * s.chunks), b = (int)(tk / (uint32_t)s.T), t = (int)(tk - (uint32_t)b * s.T);
  const int64_t tok = tk;
  const qkn_lane<V, PAIRS> ln(p, j);
  F w0 = {}, w1 = {};
  float cs[V], sn[V];
  if (ln.on) {
    qkn_load<float, V, PAIRS>(s.w, ln.c0, ln.c1, w0, w1);
  }
  qkn_angles<V, PAIRS>(p, s, ln, b, t, cs, sn);
  const T* x = (const T*)s.x + b * s.sb + t * s.st;
  T* y = (T*)s.y + tok * s.H * p.D;
  const int h1 = min(s.H, (chunk + 1) * p.hc);
  for (int hd = chunk * p.hc; hd < h1; ++hd) {
    F a = {}, c = {};
    if (ln.on) {
      qkn_load<T, V, PAIRS>(x + hd * s.sh, ln.c0, ln.c1, a, c);
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) q = fmaf(a[e], a[e], fmaf(c[e], c[e], q));
    q = qkn_row_sum(q, p.lanes);
    const float r = rsqrtf(q / (float)p.D + p.eps);
    a = a * r * w0;
    c = c * r * w1;
    if (ln.rot) qkn_turn<F, V, PAIRS>(a, c, cs, sn, 1.f);
    if (ln.on) {
      qkn_store<T, V, PAIRS>(y + (int64_t)hd * p.D, ln.c0, ln.c1, a, c);
    }
  }
}

// persistent workgroups (each walks over units a grid apart), so that the weight gradient is summed in registers and leaves one partial
// row per workgroup
template <typename T, int V, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(qkn_args p) {
  typedef typename qkn_vec<T, V>::f32 F;
  __shared__ float red[256 * 2 * V];
  const int side = blockIdx.x >= p.s[0].blocks;
  const qkn_side s = p.s[side];
  const int blk = blockIdx.x - (side ? p.s[0].blocks : 0);
  const int groups = 256 / p.lanes, j = threadIdx.x & (p.lanes - 1), grp = threadIdx.x / p.lanes;
  const int64_t units = (int64_t)p.B * s.T * s.chunks;
  const qkn_lane<V, PAIRS> ln(p, j);
  F w0 = {}, w1 = {}, d0 = {}, d1 = {};
  if (ln.on) {
    qkn_load<float, V, PAIRS>(s.w, ln.c0, ln.c1, w0, w1);
  }
  for (int64_t u = (int64_t)blk * groups + grp; u < units; u += (int64_t)s.blocks * groups) {
    const uint32_t tk = (uint32_t)u / (uint32_t)s.chunks;
    const int chunk = (int)((uint32_t)u - tk * s.chunks), b = (int)(tk / (uint32_t)s.T), t = (int)(tk - (uint32_t)b * s.T);
    const int64_t tok = tk;
    float cs[V], sn[V];
    qkn_angles<V, PAIRS>(p, s, ln, b, t, cs, sn);
    const T* x = (const T*)s.x + b * s.sb + t * s.st;
    const T* dy = (const T*)s.dy + tok * s.H * p.D;
    T* dx = (T*)s.dx + tok * s.H * p.D;
    const int h1 = min(s.H, (chunk + 1) * p.hc);
    for (int hd = chunk * p.hc; hd < h1; ++hd) {
      F a = {}, c = {}, ga = {}, gc = {};
      if (ln.on) {
        qkn_load<T, V, PAIRS>(x + hd * s.sh, ln.c0, ln.c1, a, c);
        qkn_load<T, V, PAIRS>(dy + (int64_t)hd * p.D, ln.c0, ln.c1, ga, gc);
      }
      if (ln.rot) qkn_turn<F, V, PAIRS>(ga, gc, cs, sn, -1.f);
      float q = 0.f, d = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        q = fmaf(a[e], a[e], fmaf(c[e], c[e], q));
        d = fmaf(a[e], ga[e] * w0[e], fmaf(c[e], gc[e] * w1[e], d));
      }
      q = qkn_row_sum(q, p.lanes);
      d = qkn_row_sum(d, p.lanes);
      const float r = rsqrtf(q / (float)p.D + p.eps);
      const float m = d * r * r / (float)p.D;              // mean(g w n) r
      a *= r;
      c *= r;
      d0 += ga * a;
      d1 += gc * c;
      if (ln.on) {
        qkn_store<T, V, PAIRS>(dx + (int64_t)hd * p.D, ln.c0, ln.c1, (ga * w0) * r - a * m, (gc * w1) * r - c * m);
      }
    }
  }
  // the groups of a wavefront by shuffles, the four wavefronts in LDS, always in the same order
  for (int o = p.lanes; o < 64; o <<= 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      d0[e] += __shfl_xor(d0[e], o, 64);
      d1[e] += __shfl_xor(d1[e], o, 64);
    }
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    red[(wave * 2 * V + e) * 64 + lane] = d0[e];
    red[(wave * 2 * V + V + e) * 64 + lane] = d1[e];
  }
  __syncthreads();
  if (threadIdx.x < p.lanes && ln.on) {
    float* out = p.part + (int64_t)blockIdx.x * p.D;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float* r0 = red + e * 64 + j;
      const float* r1 = r0 + V * 64;
      out[ln.c0 + e] = (r0[0] + r0[2 * V * 64]) + (r0[4 * V * 64] + r0[6 * V * 64]);
      out[ln.c1 + e] = (r1[0] + r1[2 * V * 64]) + (r1[4 * V * 64] + r1[6 * V * 64]);
    }
  }
}

// dw[c] = sum over the workgroups' partial rows, in a fixed order: a workgroup takes four channels, a thread every 256th row of them
__global__ __launch_bounds__(256) void qk_norm_rope_dw_kernel(const float* __restrict__ part, int nq, int nk, int D, float* __restrict__ dwq,
                                                              float* __restrict__ dwk) {
  __shared__ f32x4 red[4];
  const int side = blockIdx.y, c = blockIdx.x * 4;
  if (!(side ? dwk : dwq)) return;                               // (a side without heads may come without a gradient)
  const int n = side ? nk : nq;
  const float* p = part + (side ? (int64_t)nq * D : 0) + c;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < QKN_MAX_BLOCKS; i += 256)
    if (i + threadIdx.x < n) a += *(const f32x4*)(p + (int64_t)(i + threadIdx.x) * D);
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = wave_sum(a[e]);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x < 4) (side ? dwk : dwq)[c + threadIdx.x] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// ---------------------------------------------------------------------------------------------------------------- host
static int qkn_check(const ttdg_qk_norm_rope_t* a) {
  TTDG_REQUIRE(a->dtype == TTDG_F32 || a->dtype == TTDG_BF16, "qk_norm_rope: dtype must be TTDG_F32 or TTDG_BF16");
  TTDG_REQUIRE(a->B >= 0 && a->D >= 8 && a->D <= 256 && a->D % 8 == 0, "qk_norm_rope: the head dimension must be a multiple of 8 up to 256");
  TTDG_REQUIRE(a->R >= 0 && a->R <= a->D && a->R % 8 == 0 && (a->R == 0 || a->freq), "qk_norm_rope: the rotated channels must be a multiple of 8 up to the head dimension, with frequencies");
  TTDG_REQUIRE(a->axes == 1 || (a->axes == 2 && a->R % 4 == 0), "qk_norm_rope: one or two position axes");
  TTDG_REQUIRE(a->eps >= 0.f, "qk_norm_rope: eps must not be negative");
  const int ce = a->dtype == TTDG_F32 ? 4 : 8;
  for (int i = 0; i < 2; ++i) {
    const ttdg_norm_rope_side_t& s = i ? a->k : a->q;
    TTDG_REQUIRE(s.T >= 0 && s.H >= 0, "qk_norm_rope: negative size");
    if (a->B == 0 || s.T == 0 || s.H == 0) continue;
    TTDG_REQUIRE(s.x && s.w && (a->R == 0 || s.pos), "qk_norm_rope: null pointer");
    TTDG_REQUIRE(s.sb >= 0 && s.st >= 0 && s.sh >= 0 && s.sb % ce == 0 && s.st % ce == 0 && s.sh % ce == 0, "qk_norm_rope: strides must be multiples of 16 bytes");
    TTDG_REQUIRE(((uintptr_t)s.x | (uintptr_t)s.w) % 16 == 0, "qk_norm_rope: tensors must be 16-byte aligned");
    TTDG_REQUIRE((int64_t)a->B * s.T < (1ll << 30) && (int64_t)a->B * s.T * s.H < (1ll << 31), "qk_norm_rope: more than 2^31 rows");
  }
  return 0;
}

// V = channels per chunk.  Neighbouring pairs (and no rotation): a lane's two chunks are one access, 16 bytes in all.  Halves: 16 bytes per
// chunk forward; 8 bytes for bf16 when D or R is an odd multiple of 8.
static bool qkn_pairs(const ttdg_qk_norm_rope_t* a) { return a->interleaved || a->R == 0; }
static int qkn_v(const ttdg_qk_norm_rope_t* a) {
  if (qkn_pairs(a)) return a->dtype == TTDG_BF16 ? 4 : 2;
  return a->dtype == TTDG_BF16 && a->D % 16 == 0 && a->R % 16 == 0 ? 8 : 4;
}
#define QKN_LAUNCH(kernel, a, v, grid, stream, p)                                                                                       \
  do {                                                                                                                                  \
    const dim3 g_(grid), b_(256);                                                                                                       \
    if (qkn_pairs(a)) {                                                                                                                 \
      if ((a)->dtype == TTDG_F32) hipLaunchKernelGGL((kernel<float, 2, true>), g_, b_, 0, (hipStream_t)stream, p);                      \
      else hipLaunchKernelGGL((kernel<__bf16, 4, true>), g_, b_, 0, (hipStream_t)stream, p);                                            \
    } else if ((a)->dtype == TTDG_F32) hipLaunchKernelGGL((kernel<float, 4, false>), g_, b_, 0, (hipStream_t)stream, p);                \
    else if ((v) == 8) hipLaunchKernelGGL((kernel<__bf16, 8, false>), g_, b_, 0, (hipStream_t)stream, p);                               \
    else hipLaunchKernelGGL((kernel<__bf16, 4, false>), g_, b_, 0, (hipStream_t)stream, p);                                             \
    if (int e_ = ttdg_launch_status(#kernel)) return e_;                                                                                \
  } while (0)

static qkn_args qkn_make(const ttdg_qk_norm_rope_t* a, int v, bool bwd) {
  qkn_args p = {};
  p.freq = a->freq;
  p.B = a->B; p.D = a->D; p.R = a->R; p.axes = a->axes; p.interleaved = a->interleaved; p.pos64 = a->pos64; p.eps = a->eps;
  p.lanes = 1;
  while (p.lanes < a->D / (2 * v)) p.lanes *= 2;
  // heads per unit: as many as leave a quarter of a million lanes (half of the chip's), one when the call is small
  p.hc = 8;
  while (p.hc > 1) {
    const int64_t units = (int64_t)a->B * ((int64_t)a->q.T * ((a->q.H + p.hc - 1) / p.hc) + (int64_t)a->k.T * ((a->k.H + p.hc - 1) / p.hc));
    if (units * p.lanes >= (bwd ? 524288 : 262144)) break;
    p.hc /= 2;
  }
  for (int i = 0; i < 2; ++i) {
    const ttdg_norm_rope_side_t& s = i ? a->k : a->q;
    qkn_side& d = p.s[i];
    d.x = s.x; d.pos = s.pos; d.dy = s.dy; d.w = s.w; d.y = s.y; d.dx = s.dx;
    d.sb = s.sb; d.st = s.st; d.sh = s.sh; d.p_sb = s.p_sb; d.p_st = s.p_st; d.p_sa = s.p_sa;
    d.T = s.T; d.H = s.H;
    d.chunks = (s.H + p.hc - 1) / p.hc;
    const int64_t units = (int64_t)a->B * s.T * d.chunks, groups = 256 / p.lanes;
    int64_t blocks = (units + groups - 1) / groups;
    if (bwd && blocks > QKN_MAX_BLOCKS) blocks = QKN_MAX_BLOCKS;
    d.blocks = (int)(blocks > 0x7fffffff ? -1 : blocks);
  }
  return p;
}

extern "C" size_t ttdg_qk_norm_rope_bwd_workspace_bytes(const ttdg_qk_norm_rope_t* a) {
  if (!a || qkn_check(a)) return 0;
  const qkn_args p = qkn_make(a, qkn_v(a), true);
  return (size_t)(p.s[0].blocks + p.s[1].blocks) * a->D * 4;
}

extern "C" int ttdg_qk_norm_rope_fwd(const ttdg_qk_norm_rope_t* a, ttdg_stream_t stream) {
  TTDG_REQUIRE(a, "qk_norm_rope_fwd: null pointer");
  if (int e = qkn_check(a)) return e;
  const int v = qkn_v(a);
  const qkn_args p = qkn_make(a, v, false);
  for (int i = 0; i < 2; ++i) {
    TTDG_LIMIT(p.s[i].blocks >= 0 && p.s[i].blocks < (1 << 23), "qk_norm_rope_fwd: too many workgroups");      // (both sides' threads below 2^32)
    TTDG_REQUIRE(p.s[i].blocks == 0 || (p.s[i].y && (uintptr_t)p.s[i].y % 16 == 0), "qk_norm_rope_fwd: outputs must be 16-byte aligned pointers");
  }
  const int grid = p.s[0].blocks + p.s[1].blocks;
  if (grid == 0) return 0;
  QKN_LAUNCH(qk_norm_rope_fwd_kernel, a, v, grid, stream, p);
  return 0;
}

extern "C" int ttdg_qk_norm_rope_bwd(const ttdg_qk_norm_rope_t* a, ttdg_stream_t stream) {
  TTDG_REQUIRE(a, "qk_norm_rope_bwd: null pointer");
  if (int e = qkn_check(a)) return e;
  const int v = qkn_v(a);
  qkn_args p = qkn_make(a, v, true);
  const int grid = p.s[0].blocks + p.s[1].blocks;
  for (int i = 0; i < 2; ++i) {
    const qkn_side& s = p.s[i];
    TTDG_REQUIRE(s.blocks == 0 || (s.dy && s.dx && ((uintptr_t)s.dy | (uintptr_t)s.dx) % 16 == 0), "qk_norm_rope_bwd: gradients must be 16-byte aligned pointers");
  }
  TTDG_REQUIRE((a->q.H == 0 || a->q.dw) && (a->k.H == 0 || a->k.dw), "qk_norm_rope_bwd: null pointer");
  TTDG_REQUIRE(grid == 0 || (a->ws && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= (size_t)grid * a->D * 4), "qk_norm_rope_bwd: workspace too small or misaligned");
  p.part = (float*)a->ws;
  if (grid) QKN_LAUNCH(qk_norm_rope_bwd_kernel, a, v, grid, stream, p);
  const int sides = a->k.dw ? 2 : 1;
  hipLaunchKernelGGL(qk_norm_rope_dw_kernel, dim3(a->D / 4, sides), dim3(256), 0, (hipStream_t)stream, p.part, p.s[0].blocks, p.s[1].blocks, a->D,
                     a->q.dw, a->k.dw);
  return ttdg_launch_status("qk_norm_rope_dw");
}
