// Device building blocks of the attention kernels (attention.hip): operand fragments, LDS tiles, LDS-DMA, row / key bookkeeping.
#pragma once
#include <type_traits>

#include "common.h"

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

struct attn_args {
  const void *q, *k, *v;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;     // elements
  const int32_t* k_lens;
  const uint8_t* key_mask;
  int64_t m_sb, m_st;
  int B, Tq, Tk, H, Hk, D, G, R;                                    // G = H / Hk query heads per key head, R = Tq G rows per problem
  int row_tiles, key_tiles, splits, slots;                          // slots: workgroups of dk / dv that the chip runs at once
  float scale, scale_log2;                                          // scale, scale * log2(e)
  void *out, *out_lo;
  float *lse, *far;                                                 // (problem, row): log2 of the row's sum of exponentials, see attn_ref
  const void* dout;
  void *dq, *dk, *dv;
  float *delta, *part_o, *part_lse;                                 // delta: minus do . o of every row
  int32_t* share;                                                   // (first part or tile, how many) of every sample; null: all alike
};

__device__ __forceinline__ f32x16 f32x16_all(float x) {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = x;
  return z;
}
__device__ __forceinline__ f32x16 f32x16_zero() { return f32x16_all(0.f); }

// register e of a 32 x 32 accumulator holds tile row attn_reg_row(e) + 4 (lane >> 5), tile column lane & 31
__device__ __forceinline__ constexpr int attn_reg_row(int e) { return (e & 3) + 8 * (e >> 2); }

// value of the own lane and of the lane 32 away, joined
__device__ __forceinline__ float attn_half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float attn_half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Waits for every load and LDS-DMA of this wavefront (0xf70: vmcnt 0, the other counters as they are).  The builtin, not assembly text: the
// compiler then knows that nothing is outstanding and adds no waits of its own behind the next tile's LDS-DMA.
__device__ __forceinline__ void attn_wait_dma() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xf70);
  asm volatile("" ::: "memory");
}

// Transposing LDS read: of the 4 x 16 block that 16 neighbouring lanes address (lane i: row i / 4, columns 4 (i % 4) ...) lane i gets column i.
// (restrict: without alias information the compiler would wait here for every LDS-DMA in flight, that is for the next tile.)
__device__ __forceinline__ bf16x4 attn_read_tr(const char* __restrict__ a) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)a);
}

#define ATTN_OOB 0x7ffffff0u          // behind the end of every buffer resource below: reads as zero
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attn_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, 0x7fffff00, 0x00020000);
}
__device__ __forceinline__ void attn_dma16(__amdgpu_buffer_rsrc_t r, char* lds_wave_base, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds_wave_base, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void attn_dma4(__amdgpu_buffer_rsrc_t r, char* lds_wave_base, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds_wave_base, 4, off, 0, 0, 0);
}

__device__ __forceinline__ void attn_store4(float* out, f32x4 x) { *(f32x4*)out = x; }
__device__ __forceinline__ void attn_store4(__bf16* out, f32x4 x) { *(bf16x4*)out = __builtin_convertvector(x, bf16x4); }

// A row's reference point: its terms are 2^((s - far) k - ref), k = scale log2(e).  Up to ATTN_FAR (in powers of two) far is 0 and ref the
// scaled score, so that a term costs one fma and its exponential; the rounding of ref, up to 2^-17, is the same for all terms.  A larger scaled
// score has no 32-bit number near enough (half a step of 10^9 is 2^5), there far is the score itself, which the subtraction cancels
// exactly, and ref 0.  A row's log of the sum is kept as the same two numbers: far, and lse = ref + log2(sum).
// A wavefront asks once whether any of its rows is far and leaves the subtraction out if none is.
#define ATTN_FAR 256.f
struct attn_ref {
  float at;                          // far or ref, whichever is not 0 (one register less than both); -infinity: no key yet
  bool is_far;
  __device__ __forceinline__ float far() const { return is_far ? at : 0.f; }
  __device__ __forceinline__ float ref() const { return is_far ? 0.f : at; }
  __device__ __forceinline__ bool any() const { return is_far || at > -INFINITY; }
  // how far this point lies above the other one, in powers of two
  __device__ __forceinline__ float above(const attn_ref& o, float k) const { return fmaf(far() - o.far(), k, ref() - o.ref()); }
  // the same for a score
  __device__ __forceinline__ float below(float s, float k) const { return fmaf(s - far(), k, -ref()); }
};
// the reference point of score s
__device__ __forceinline__ attn_ref attn_ref_at(float s, float k) {
  const float c = s * k;
  const bool far = !(fabsf(c) <= ATTN_FAR);
  return attn_ref{far ? s : c, far};
}

// sum over the lanes up to the own one
__device__ __forceinline__ uint32_t attn_scan(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);      // from 1, 2, 4, 8 lanes before, inside rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // the last lane of a row, to the next one
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // lane 31, to the upper half
  return x;
}
__device__ __forceinline__ uint32_t attn_ceil(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// keys of sample b
__device__ __forceinline__ int attn_length(const attn_args& p, int b) { return p.k_lens ? max(0, min(p.k_lens[b], p.Tk)) : p.Tk; }

// workgroup -> (sample, its keys, key head, tile, split of how many, first part of the sample)
struct attn_item {
  int b, keys, hk, prob, tile, split, splits, base;
  __device__ __forceinline__ void uniform() {      // (they are; said to the compiler, which otherwise keeps them in vector registers)
    b = __builtin_amdgcn_readfirstlane(b);
    keys = __builtin_amdgcn_readfirstlane(keys);
    hk = __builtin_amdgcn_readfirstlane(hk);
    prob = __builtin_amdgcn_readfirstlane(prob);
    tile = __builtin_amdgcn_readfirstlane(tile);
    split = __builtin_amdgcn_readfirstlane(split);
    splits = __builtin_amdgcn_readfirstlane(splits);
    base = __builtin_amdgcn_readfirstlane(base);
  }
};

// The long axis is in parts: all samples alike, or (RAGGED and p.share, at most 64 samples, one per lane) as many for each as its own length
// gives: the B splits parts there are go round in units of `unit` keys, as few units per part as possible.  False: a part too many.
template <bool RAGGED>
__device__ __forceinline__ bool attn_place(const attn_args& p, int tiles, int unit, attn_item& w) {
  const int L = blockIdx.x;
  if (!RAGGED || !p.share) {
    const int per = tiles * p.splits;
    w.prob = L / per;
    const int rem = L - w.prob * per;
    w.splits = p.splits;
    w.split = rem / tiles;
    w.tile = rem - w.split * tiles;
    w.b = w.prob / p.Hk;
    w.hk = w.prob - w.b * p.Hk;
    w.base = w.b * p.splits;
    w.keys = attn_length(p, w.b);
  } else {
    const int per = p.Hk * tiles, j = L / per, rem = L - j * per;
    w.hk = rem / tiles;
    w.tile = rem - w.hk * tiles;
    const int lane = threadIdx.x & 63;
    const bool on = lane < p.B;
    const int len = on ? attn_length(p, lane) : 0;
    const uint32_t n = attn_ceil(len, unit), room = p.B * p.splits, total = __builtin_amdgcn_readlane(attn_scan(n), 63);
    uint32_t each = max(1u, attn_ceil(total, room)), mine = on ? max(1u, attn_ceil(n, each)) : 0, end = attn_scan(mine);
    if ((uint32_t)__builtin_amdgcn_readlane(end, 63) > room) {
      uint32_t lo = each + 1;
      each = max(lo, attn_ceil(total, room - p.B));            // (with this many they fit: at most total / each + B parts)
      while (lo < each) {
        const uint32_t mid = (lo + each) / 2;
        if ((uint32_t)__builtin_amdgcn_readlane(attn_scan(on ? max(1u, attn_ceil(n, mid)) : 0), 63) <= room) each = mid;
        else lo = mid + 1;
      }
      mine = on ? max(1u, attn_ceil(n, each)) : 0;
      end = attn_scan(mine);
    }
    if (L == 0 && threadIdx.x < p.B) {
      p.share[2 * lane] = end - mine;
      p.share[2 * lane + 1] = mine;
    }
    if (j >= __builtin_amdgcn_readlane(end, 63)) return false;
    w.b = __popcll(__ballot(end <= (uint32_t)j));
    w.splits = __builtin_amdgcn_readlane(mine, w.b);
    w.base = __builtin_amdgcn_readlane(end, w.b) - w.splits;
    w.keys = __builtin_amdgcn_readlane(len, w.b);
    w.split = j - w.base;
    w.prob = w.b * p.Hk + w.hk;
  }
  w.uniform();
  return true;
}

// The same for dk / dv: (sample, key head, key tile, split of the rows).  With p.share the workgroups go to the key tiles that have keys, every
// one of them in as many parts as there is room for; base: number of the key tile among these.
__device__ __forceinline__ bool attn_place_keys(const attn_args& p, int unit, int row_units, attn_item& w) {
  const int L = blockIdx.x;
  if (!p.share) {
    const int per = p.key_tiles * p.splits;
    w.prob = L / per;
    const int rem = L - w.prob * per;
    w.splits = p.splits;
    w.split = rem / p.key_tiles;
    w.tile = rem - w.split * p.key_tiles;
    w.b = w.prob / p.Hk;
    w.hk = w.prob - w.b * p.Hk;
    w.base = w.b * p.key_tiles + w.tile;
    w.keys = attn_length(p, w.b);
    w.uniform();
    return true;
  }
  const int lane = threadIdx.x & 63;
  const int len = lane < p.B ? attn_length(p, lane) : 0;
  const uint32_t mine = attn_ceil(len, unit), end = attn_scan(mine);
  const int tiles = __builtin_amdgcn_readlane(end, 63);
  // (of the host's splits there is always room, of more only what the chip runs at once)
  const int most = min(row_units, max(p.splits, p.slots / (p.Hk * max(tiles, 1))));
  w.splits = attn_ceil(row_units, attn_ceil(row_units, most));
  if (L == 0 && threadIdx.x < p.B) {
    p.share[2 * lane] = end - mine;
    p.share[2 * lane + 1] = mine;
    p.share[2 * 64] = w.splits;
  }
  const int per = tiles * w.splits;
  if (L >= per * p.Hk) return false;
  w.hk = L / per;
  const int rem = L - w.hk * per;
  w.split = rem / tiles;
  w.base = rem - w.split * tiles;
  w.b = __popcll(__ballot(end <= (uint32_t)w.base));
  w.tile = w.base - (__builtin_amdgcn_readlane(end, w.b) - __builtin_amdgcn_readlane(mine, w.b));
  w.keys = __builtin_amdgcn_readlane(len, w.b);
  w.prob = w.b * p.Hk + w.hk;
  w.uniform();
  return true;
}

// the part [t0, t1) of n tiles that falls to one of the splits
__device__ __forceinline__ void attn_part(int n, int split, int splits, int& t0, int& t1) {
  t0 = (int)((int64_t)n * split / splits);
  t1 = (int)((int64_t)n * (split + 1) / splits);
}

// row of a problem -> query position and head (rows behind the last one are clamped to it: they are computed and not stored)
struct attn_row {
  int row, t, head;
  __device__ __forceinline__ attn_row(const attn_args& p, int hk, int r) {
    row = min(r, p.R - 1);
    t = row / p.G;
    head = hk * p.G + row - t * p.G;
  }
};

// the keys of a sample: how many, and which of a tile exist
struct attn_keys {
  int n;
  const uint8_t* mask;
  int64_t m_st;
  __device__ __forceinline__ attn_keys(const attn_args& p, int b, int keys) {
    n = keys;
    mask = p.key_mask ? p.key_mask + b * p.m_sb : nullptr;
    m_st = p.m_st;
  }
  __device__ __forceinline__ bool alive(int key) const { return key < n && (!mask || mask[key * m_st]); }
};

// position of 16-byte chunk c of a tile row.  Eight consecutive rows XOR with eight different numbers (row reads: eight lanes of
// consecutive rows read the same c), and the four rows of a transposing read's 16-lane group land in four different 32-byte windows.
// (The counters still call 25 % of the LDS' busy cycles conflicts with rows of 128 bytes, 40 to 50 % with longer ones; it is busy 25 to 45 % of
// the time in large calls.)
__device__ __forceinline__ int attn_swz(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

// DP channels of tiles whose rows have RD (a wavefront may work on a part of the channels)
template <typename T, int DP, int RD = DP>
struct attn_tile {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int ES = sizeof(T), CE = 16 / ES;      // element size, elements per chunk
  static constexpr int RB = RD * ES;                      // bytes of a tile row
  static constexpr int NC = DP * ES / 16, NP = NC / 2;    // chunks per row; chunk pairs: the wavefront's halves take one chunk each
  static constexpr int bytes(int rows) { return rows * RB; }
  typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T frag;

  // a row of the second operand: half h holds chunks 2 i + h; zeros behind D
  static __device__ __forceinline__ void load_row(frag* f, const T* row, int D, int h) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (2 * i + h) * CE;
      frag z = {};
      f[i] = c < D ? *(const frag*)(row + c) : z;
    }
  }
  // sum over this half's chunks of f * (a + lo)
  static __device__ __forceinline__ float row_dot(const frag* f, const T* a, const T* lo, int D, int h) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (2 * i + h) * CE;
      if (c < D) {
        const frag x = *(const frag*)(a + c);
        frag y = {};
        if (lo) y = *(const frag*)(lo + c);
#pragma unroll
        for (int e = 0; e < CE; ++e) s = fmaf((float)f[i][e], (float)x[e] + (float)y[e], s);
      }
    }
    return s;
  }

  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
      return c;
    } else {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
  }

  // acc[k][n][tile row][lane's row of f[n]] += sum_d tile[row0 + 32 k + .][d] f[n][d]: KK blocks of tile rows times NB blocks of columns,
  // KK NB independent chains of products.  PRE > 0: the chunks of PRE steps are read ahead of their products (the barriers keep the
  // compiler from reading each one just before its use); 0: left to the compiler.
  template <int KK, int NB, int PRE>
  static __device__ __forceinline__ void row_product(f32x16 (*acc)[NB], const char* tile, int row0, const frag (*f)[NP], int l32, int h) {
    const int base = l32 * RB + ((h ^ attn_swz(l32)) << 4);
    if constexpr (PRE == 0) {
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < KK; ++k) {
          const frag a = *(const frag*)(tile + (row0 + 32 * k) * RB + (base ^ (32 * (i & 3))) + 128 * (i >> 2));
#pragma unroll
          for (int n = 0; n < NB; ++n) acc[k][n] = mma(a, f[n][i], acc[k][n]);
        }
    } else {
      frag a[2][PRE][KK];
#pragma unroll
      for (int i = 0; i < NP + PRE; i += PRE) {
        if (i < NP) {
#pragma unroll
          for (int j = 0; j < PRE; ++j)
#pragma unroll
            for (int k = 0; k < KK; ++k)
              a[(i / PRE) & 1][j][k] = *(const frag*)(tile + (row0 + 32 * k) * RB + (base ^ (32 * ((i + j) & 3))) + 128 * ((i + j) >> 2));
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i > 0) {
#pragma unroll
          for (int j = 0; j < PRE; ++j)
#pragma unroll
            for (int k = 0; k < KK; ++k)
#pragma unroll
              for (int n = 0; n < NB; ++n) acc[k][n] = mma(a[(i / PRE + 1) & 1][j][k], f[n][i - PRE + j], acc[k][n]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // 32 tile rows of one column block as the second product's second operand.  For 16-bit types a value is rounded to the inputs' type (round
  // to nearest even, as every operand of the matrix unit is): an error of at most half a step per term, independent from term to term,
  // while the sums stay in 32 bits.  PARTS = 2 adds what that rounding dropped as a second operand (16 bits of significand in all).
  template <int PARTS>
  struct operand {
    typename std::conditional<F32, f32x16, bf16x8>::type x[F32 ? 1 : PARTS][F32 ? 1 : 2];
  };
  template <int PARTS>
  static __device__ __forceinline__ operand<PARTS> pack(const f32x16& p) {
    operand<PARTS> r;
    if constexpr (F32) {
      r.x[0][0] = p;
    } else {
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
        f32x8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = p[8 * kg + e];
        r.x[0][kg] = __builtin_convertvector(y, bf16x8);
        if constexpr (PARTS == 2) {
          // (widened as bits: by conversion the compiler would round every value a second time)
          const u32x4 u = __builtin_bit_cast(u32x4, r.x[0][kg]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] -= __uint_as_float(u[e] << 16);
            y[2 * e + 1] -= __uint_as_float(u[e] & 0xffff0000u);
          }
          r.x[1][kg] = __builtin_convertvector(y, bf16x8);
        }
      }
    }
    return r;
  }
  // l + the lane's terms.  With one part the terms as the product will see them: a row's weights then sum to one whatever their rounding did
  template <int PARTS>
  static __device__ __forceinline__ float sum(const operand<PARTS>& p, float l) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 16; ++e) l += p.x[0][0][e];
    } else {
      const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
      for (int q = 0; q < PARTS; ++q)
#pragma unroll
        for (int kg = 0; kg < 2; ++kg)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const bf16x2 y = {p.x[q][kg][e], p.x[q][kg][e + 1]};
            l = __builtin_amdgcn_fdot2_f32_bf16(y, one, l, false);
          }
    }
    return l;
  }

  // acc[n][d][lane's column] += sum over the 32 tile rows from row0 of tile[.][d] p[n][.]
  template <int NB, int PARTS>
  static __device__ __forceinline__ void col_product(f32x16 (*acc)[DP / 32], const char* tile, int row0, const operand<PARTS>* p, int lane) {
    const int h = lane >> 5;
    if constexpr (F32) {
      const int l32 = lane & 31;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = attn_reg_row(e) + 4 * h;
        const char* a = tile + (row0 + row) * RB + (((l32 >> 2) ^ (((e & 3) << 1) | h)) << 4) + 4 * (l32 & 3);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const float x = *(const float*)(a + 128 * d);
#pragma unroll
          for (int n = 0; n < NB; ++n) acc[n][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[n].x[0][0][e], acc[n][d], 0, 0, 0);
        }
      }
    } else {
      const int i = lane & 15, blk = (lane >> 4) & 1, row = 4 * h + (i >> 2);
      const int base = row * RB + (((2 * blk + ((i & 3) >> 1)) ^ attn_swz(row)) << 4) + 8 * (i & 1);
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const char* a = tile + (row0 + 16 * kg) * RB + (base ^ (64 * (d & 1))) + 128 * (d >> 1);
          const bf16x4 lo = attn_read_tr(a), hi = attn_read_tr(a + 8 * RB);
          const bf16x8 f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int q = 0; q < PARTS; ++q) acc[n][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, p[n].x[q][kg], acc[n][d], 0, 0, 0);
        }
    }
  }

  // the lane's row: channels 32 d + 8 g + 4 h + (0 .. 3) are four consecutive registers.  `lo`: what the rounding of `out` dropped.
  template <typename O>
  static __device__ __forceinline__ void store_row(const f32x16* acc, float factor, O* out, O* lo, int D, int h) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * h;
        if (c < D) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = acc[d][4 * g + e] * factor;
          attn_store4(out + c, x);
          if (lo) {
            if constexpr (sizeof(O) == 2) {
              const bf16x4 hi = __builtin_convertvector(x, bf16x4);
              attn_store4(lo + c, x - __builtin_convertvector(hi, f32x4));
            }
          }
        }
      }
  }
};

// A barrier for what the wavefronts wrote to LDS themselves.  (__syncthreads waits for LDS-DMA in flight as well, that is for the next tile.)
__device__ __forceinline__ void attn_lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Two wavefronts that hold sums over half the channels each add them: `own` and `other` are their 4 KiB of LDS.  Every wavefront of the
// workgroup takes part in the barriers; the one behind the reads is left out (LAST) where another follows before the next exchange.
template <bool LAST>
__device__ __forceinline__ void attn_exchange(f32x16& x, float* own, const float* other, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) ((f32x4*)own)[g * 64 + lane] = f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
  attn_lds_barrier();
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 y = ((const f32x4*)other)[g * 64 + lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * g + e] += y[e];
  }
  if (!LAST) attn_lds_barrier();
}

// LDS-DMA of ROWS tile rows: instruction i of a wavefront fills 1 KiB; its lanes' offsets repeat every PER instructions (the swizzle has a
// period of eight rows), the rest of the distance goes into the scalar offset.  Lanes behind D always point behind the resource's end.
template <typename T, int DP, int ROWS, int WM>
struct attn_loader {
  typedef attn_tile<T, DP> tile_t;
  static constexpr int N = ROWS * tile_t::NC / 64 / WM;              // instructions per wavefront
  static constexpr int STEP = WM * 64 / tile_t::NC;                  // tile rows from one instruction to the next
  static constexpr int PER = STEP >= 8 ? 1 : 8 / STEP;
  uint32_t off[PER];
  int row, cofs[PER];
  __device__ __forceinline__ void init(int D, int wave, int lane) {
    row = (wave * 64 + lane) / tile_t::NC;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = (lane % tile_t::NC) ^ attn_swz(row + j * STEP);
      cofs[j] = c * tile_t::CE < D ? c * 16 : -1;
    }
  }
  // rows stb bytes apart
  __device__ __forceinline__ void strided(uint32_t stb) {
#pragma unroll
    for (int j = 0; j < PER; ++j) off[j] = cofs[j] < 0 ? ATTN_OOB : (row + j * STEP) * stb + cofs[j];
  }
  // rows whose bit in `live` is off become zeros
  __device__ __forceinline__ void issue(char* lds, const void* base, uint32_t stb, uint64_t live, bool all, int wave) const {
    const auto r = attn_rsrc(base);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t o = off[i % PER];
      if (!all) o = (live >> (row + i * STEP)) & 1 ? o : ATTN_OOB;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (i * WM + wave) * 1024), 16, o,
                                               (i / PER) * PER * STEP * stb, 0, 0);
    }
  }
};

// The key / value tiles of a problem, in stages of LDS: k tile, v tile, and for tiles with absent keys the scores' starting values (0, or
// -infinity where no key exists: the scores' sums start from them, so masking costs no vector instruction).
// LEAN: the lanes' offsets are made anew for every tile; kept, they are the registers that the kernel with 64 rows per wavefront lacks, and
// reloading one of them from scratch waits for the LDS-DMA just started (both in one run: 16 x 2048 rows over 4096 keys, 8 heads, with 64
// rows per wavefront 754 -> 712 us; 4 x 4096 rows over 8191 keys, 16 heads, 1188 -> 1131).
template <typename T, int DP, int BN, int WM, bool LEAN = false>
struct attn_stream {
  typedef attn_tile<T, DP> tile_t;
  static constexpr int TB = tile_t::bytes(BN), STAGE = 2 * TB + 256;
  static constexpr uint64_t ALL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
  attn_loader<T, DP, BN, WM> lk, lv;
  attn_keys keys;
  const T *k, *v;
  int64_t k_tile, v_tile;
  uint32_t k_stb, v_stb;
  int next, wave, lane, D;
  uint32_t ahead;                    // the mask byte of this lane's key of the next tile, asked for a tile earlier (kept as it comes: a
                                     // comparison here would wait for it)

  __device__ __forceinline__ attn_stream(const attn_args& p, int b, int hk, int n, int wave_, int lane_) : keys(p, b, n), next(0), wave(wave_), lane(lane_), D(p.D), ahead(0) {
    k = (const T*)p.k + b * p.k_sb + (int64_t)hk * p.k_sh;
    v = (const T*)p.v + b * p.v_sb + (int64_t)hk * p.v_sh;
    k_tile = BN * p.k_st;
    v_tile = BN * p.v_st;
    k_stb = (uint32_t)(p.k_st * tile_t::ES);
    v_stb = (uint32_t)(p.v_st * tile_t::ES);
    lk.init(p.D, wave, lane);
    lv = lk;
    lk.strided(k_stb);
    lv.strided(v_stb);
  }
  __device__ __forceinline__ int tiles() const { return (keys.n + BN - 1) / BN; }
  __device__ __forceinline__ void seek(int t) {
    next = t;
    k += t * k_tile;
    v += t * v_tile;
  }
  __device__ __forceinline__ void peek() {
    const int key = next * BN + lane;
    if (keys.mask) ahead = key < keys.n ? keys.mask[key * keys.m_st] : 0;
  }
  // starts the next tile's way into `stage` and returns which of its keys exist (none: nothing is loaded); asks for the mask of the tile after it
  __device__ __forceinline__ uint64_t issue(char* stage) {
    bool mine = lane < BN && next * BN + lane < keys.n;
    if (keys.mask) {
      asm volatile("" : "+v"(ahead));                   // (awaited in here: without a mask there is nothing to wait for)
      mine = mine && ahead;
    }
    const uint64_t live = __ballot(mine);
    ++next;
    peek();
    if (live) {
      const bool all = live == ALL;
      if (LEAN) {
        int l = lane;
        asm volatile("" : "+v"(l));
        lk.init(D, wave, l);
        lv = lk;
        lk.strided(k_stb);
        lv.strided(v_stb);
      }
      lk.issue(stage, k, k_stb, live, all, wave);
      lv.issue(stage + TB, v, v_stb, live, all, wave);
      if (!all && wave == 0) ((float*)(stage + 2 * TB))[lane] = mine ? 0.f : -INFINITY;
    }
    k += k_tile;
    v += v_tile;
    return live;
  }
  // starting values of the scores
  static __device__ __forceinline__ f32x16 start(const char* stage, int row0, uint64_t live, int h) {
    f32x16 s = f32x16_zero();
    if (live != ALL) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = *(const f32x4*)(stage + 2 * TB + 4 * (row0 + 8 * g + 4 * h));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * g + e] = x[e];
      }
    }
    return s;
  }
};

// The row tiles of the dk / dv kernel, in stages of LDS: q tile, do tile, lse, delta and far of the rows
template <typename T, int DP, int BQ, int WM>
struct attn_rows {
  typedef attn_tile<T, DP> tile_t;
  static constexpr int TB = tile_t::bytes(BQ), STAGE = 2 * TB + 768;
  attn_loader<T, DP, BQ, WM> lq, lg;
  const T *q, *g;
  const float *lse, *delta, *far;
  int next, wave, lane;
  float ahead;                       // far of this lane's row of the next tile
  __device__ __forceinline__ attn_rows(const attn_args& p, int b, int hk, int prob, int first, int wave_, int lane_) : next(first), wave(wave_), lane(lane_), ahead(0.f) {
    lse = p.lse + (int64_t)prob * p.R;
    delta = p.delta + (int64_t)prob * p.R;
    far = p.far + (int64_t)prob * p.R;
    q = (const T*)p.q + b * p.q_sb + (int64_t)hk * p.G * p.q_sh;
    g = (const T*)p.dout + ((int64_t)b * p.Tq * p.H + (int64_t)hk * p.G) * p.D;
    lq.init(p.D, wave, lane);
    lg = lq;
  }
  __device__ __forceinline__ void issue(const attn_args& p, char* stage) {
    const int r0 = next * BQ, tb = r0 / p.G, left = p.R - r0;
    const auto rq = attn_rsrc(q + (int64_t)tb * p.q_st);
    const auto rg = attn_rsrc(g + (int64_t)tb * p.H * p.D);
    const uint32_t qst = (uint32_t)(p.q_st * tile_t::ES), qsh = (uint32_t)(p.q_sh * tile_t::ES);
    const uint32_t gst = (uint32_t)(p.H * p.D * tile_t::ES), gsh = (uint32_t)(p.D * tile_t::ES);
#pragma unroll
    for (int i = 0; i < decltype(lq)::N; ++i) {
      const int row = lq.row + i * decltype(lq)::STEP, c = lq.cofs[i % decltype(lq)::PER];
      const bool ok = c >= 0 && row < left;
      const int r = r0 + row - tb * p.G, tt = p.G == 1 ? r : r / p.G, gg = r - tt * p.G;
      attn_dma16(rq, stage + (i * WM + wave) * 1024, ok ? tt * qst + gg * qsh + c : ATTN_OOB);
      attn_dma16(rg, stage + TB + (i * WM + wave) * 1024, ok ? tt * gst + gg * gsh + c : ATTN_OOB);
    }
    if (wave == WM - 1) {
      const uint32_t off = lane < BQ && lane < left ? lane * 4 : ATTN_OOB;
      attn_dma4(attn_rsrc(lse + r0), stage + 2 * TB, off);
      attn_dma4(attn_rsrc(delta + r0), stage + 2 * TB + 256, off);
      attn_dma4(attn_rsrc(far + r0), stage + 2 * TB + 512, off);
    }
    ahead = lane < BQ && lane < left ? far[r0 + lane] : 0.f;
    ++next;
  }
  // whether a row of the tile that has landed has a far reference point (asked before the next one is started)
  __device__ __forceinline__ bool some_far() const { return __any(ahead != 0.f); }
};
