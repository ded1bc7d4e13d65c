// Multi-head cross attention: queries of one set attend to keys / values of another (an encoder's states), forward and backward.
//
//   s_ij = scale q_i . k_j        p_ij = exp(s_ij) / sum_j exp(s_ij)  over the keys j that exist (j < k_lens[b], key_mask[b, j] != 0)
//   o_i  = sum_j p_ij v_j         (a row without any key: o_i = 0, no gradient)
//   delta_i = o_i . do_i          ds_ij = p_ij (v_j . do_i - delta_i)
//   dv_j = sum_i p_ij do_i        dk_j = scale sum_i ds_ij q_i        dq_i = scale sum_j ds_ij k_j
//
// Shared key heads: the G = H / Hkv query heads of a key head and the Tq queries form ONE list of R = Tq G rows, row r = t G + g, so a
// problem is (batch, key head): R rows against Tk keys, and nothing below knows about heads.
//
// Everything is computed transposed, S^T = K Q^T with v_mfma 32 x 32 tiles: a lane then owns one row (column of the tile) and 16 of the
// 32 keys, so the softmax is in-lane plus one exchange between the wavefront's halves, and the probabilities already lie in the registers
// the way the next product O^T = V^T P^T wants its second operand (which keys sit in which of the operand's slots is free as long as V^T
// uses the same order).  V^T is read from the row-major V tile by the transposing LDS read (16-bit types) or by plain column reads
// (32-bit).  One body serves both types: bfloat16 through v_mfma_f32_32x32x16_bf16, float32 through v_mfma_f32_32x32x2_f32 (exact products).
//
// Tiles go memory -> LDS by LDS-DMA, double-buffered, in 16-byte chunks whose position in the row is XORed with a function of the row
// (attn_swz: neighbouring rows in different places, for row reads and for the transposing reads).  A chunk that must not be read - a row behind the last key, a masked
// key, a channel behind D - gets an offset behind the end of the buffer resource: the hardware then stores zeros, so whatever stands in
// masked places (infinities, NaN) never reaches a product.  The resource starts at the tile, so 32-bit offsets are relative to the tile
// and a cache may be longer than 4 GiB.
#include "attention.h"

// float32 with 256 channels: the operands and sums of 32 rows times 256 channels overflow a wavefront's registers and take 14 us per tile of
// 32 keys, so two wavefronts share 32 rows, each with half the channels: half of every score's sum (exchanged through LDS) and half of
// the output (both sides in one run: dq of 8 x 2048 rows over 4096 keys, 8 heads, 8400 -> 7500 us, dk / dv 9450 -> 9546; 8 x 256 rows over 794
// ragged keys, forward + backward, 184 -> 134 us).  The forward holds one set of sums only: the large call takes 4330 us without the exchange and
// 5180 with it, 2048 rows over 4096 keys 644 and 724, 8 x 256 rows 45 and 36 (with the join); attn_planned compares the two.  bfloat16 fits
// without (with the exchange: 640 -> 560 TFLOP/s).
constexpr int attn_cs(int dp, bool f32) { return dp == 256 && f32 ? 2 : 1; }
constexpr int attn_rows_wg(int dp, bool f32) { return 128 / attn_cs(dp, f32); }      // rows, or keys, of a workgroup of four wavefronts
constexpr int attn_exchange_bytes(int dp, bool f32) { return attn_cs(dp, f32) > 1 ? 4 * 4096 : 0; }

// Wavefronts per SIMD that a kernel's LDS stages and registers allow; told to the compiler as minimum AND maximum, because left free it
// saves registers for an occupancy that the LDS does not allow and then reads every operand just before its use.
template <typename T, int DP, int SMALL>
constexpr int attn_waves() {
  return sizeof(T) == 2 ? (DP == 64 ? SMALL : DP == 128 ? 2 : 1) : (DP == 64 ? 2 : 1);
}
#define ATTN_WAVES(threads, n) __launch_bounds__(threads) __attribute__((amdgpu_waves_per_eu(n, n)))

// How many bfloat16 operands carry a probability or a score gradient into the second product (PARTS of the kernels, attn_tile::pack).  With
// one, the rounding of p (or ds) adds an error of the size of the result's own rounding.  ds takes two everywhere: half of its terms
// cancel in dq and dk, which then had 1.5 times the error of their own rounding (1.04 with two; dq and dk / dv of 4 x 2047 rows over 2500 keys, 16
// heads x 128: 268 + 473 us with one, 324 + 535 with two; of 8 x 1000 over 1500, 12 heads x 64: 79 + 104 and 97 + 122).  p takes two where a
// launch leaves the chip room - few rows, or workgroups for half of the slots at most: few values are averaged there, and the extra products
// hide behind the loads (one token over 53294 keys: 15.2 and 15.6 us) - and one in large calls (the two above: forward 217 and 283 us, dk / dv
// 534 and 608; 69 and 91, 122 and 140), where out and dv have 1.2 to 1.45 times their own rounding's error.
template <typename T>
constexpr int attn_parts(bool two) { return sizeof(T) == 2 && two ? 2 : 1; }

// ---------------------------------------------------------------------------------------------------------------- forward
// A wavefront owns 32 NB rows: every chunk that it reads from LDS serves NB products.  WM wavefronts share the key tiles; KW wavefronts
// (few rows: WM = 1) have key tiles of their own, walk over parts of the keys without a barrier and join their rows at the end.
template <typename T, int DP, int BN, int WM, int NB, int KW, int PARTS, int CS>
__global__ ATTN_WAVES(64 * WM * KW, (WM == 1 ? 1 : DP == 256 && sizeof(T) == 2 ? 2 : attn_waves<T, DP, 4>())) void attn_fwd_kernel(attn_args p) {
  constexpr int DC = DP / CS;
  typedef attn_tile<T, DC, DP> tile_t;
  typedef typename tile_t::frag frag;
  typedef attn_stream<T, DP, BN, WM, (NB > 1)> stream_t;
  // Scores are added up in the same order here and in the backward kernels, bit for bit: s - far must be zero there where it was here.  What
  // two wavefronts add there in halves, one adds here in two sums.
  constexpr int HN = CS == 1 ? attn_cs(DP, sizeof(T) == 4) : 1;
  typedef attn_tile<T, DC / HN, DP> score_t;
  static_assert(HN == 1 || (NB == 1 && BN == 32), "two sums of one block of scores");
  static_assert(WM == 1 || KW == 1, "wavefronts along rows or along keys");
  static_assert(CS == 1 || (NB == 1 && BN == 32), "one sum at a time to exchange");
  extern __shared__ __attribute__((aligned(1024))) char attn_smem[];
  const int lane = threadIdx.x & 63, w_ = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = KW > 1 ? 0 : w_, kw = KW > 1 ? w_ : 0;
  const int h = lane >> 5, l32 = lane & 31;
  const int cs = CS > 1 ? w_ % CS : 0;                        // which part of the channels
  char* const smem = attn_smem + kw * 2 * stream_t::STAGE;
  float* const ex = (float*)(attn_smem + 2 * stream_t::STAGE);
  attn_item at;
  if (!attn_place<(WM > 1)>(p, p.row_tiles, BN, at)) return;
  const int b = at.b, hk = at.hk, prob = at.prob, tile = at.tile, split = at.split;

  const int row0 = (tile * (WM / CS) + wave / CS) * 32 * NB + l32;      // block n of this lane: row0 + 32 n
  frag qf[NB * HN][score_t::NP];
  f32x16 o[NB][DC / 32];
  attn_ref m[NB];
  float l[NB];
  bool far = false;                  // some row of this wavefront has a far reference point
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const attn_row rw(p, hk, row0 + 32 * n);
    const T* row = (const T*)p.q + b * p.q_sb + (int64_t)rw.t * p.q_st + (int64_t)rw.head * p.q_sh + cs * DC;
#pragma unroll
    for (int i = 0; i < HN; ++i) score_t::load_row(qf[n * HN + i], row + i * (DC / HN), p.D - cs * DC - i * (DC / HN), h);
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) o[n][d] = f32x16_zero();
    m[n] = attn_ref{-INFINITY, false};
    l[n] = 0.f;
  }

  stream_t in(p, b, hk, at.keys, wave, lane);
  int t0, t1;
  attn_part(in.tiles(), split * KW + kw, at.splits * KW, t0, t1);
  in.seek(t0);
  uint64_t live_next = 0;
  if (t0 < t1) {
    in.peek();
    live_next = in.issue(smem);
  }
  constexpr int KK = NB == 1 ? BN / 32 : 1;                // blocks of 32 keys at a time: as many sums as the registers hold
  for (int t = t0; t < t1; ++t) {
    char* stage = smem + ((t - t0) & 1) * stream_t::STAGE;
    const uint64_t live = live_next;
    attn_wait_dma();                 // this wavefront's share of tile t has landed
    if (WM > 1) __syncthreads();     // ... everybody's has, and nobody still reads the other stage
    if (t + 1 < t1) live_next = in.issue(smem + ((t + 1 - t0) & 1) * stream_t::STAGE);
    if (live == 0) continue;         // (the same for every wavefront of the workgroup)
#pragma unroll 1
    for (int k0 = 0; k0 < BN; k0 += 32 * KK) {
      f32x16 s[KK][NB];
#pragma unroll
      for (int k = 0; k < KK; ++k)
#pragma unroll
        for (int n = 0; n < NB; ++n) s[k][n] = stream_t::start(stage, k0 + 32 * k, live, h);
      score_t::template row_product<KK, NB, 0>(s, stage + cs * DC * tile_t::ES, k0, qf, l32, h);
      if constexpr (HN > 1) {
        f32x16 s1[1][1] = {{f32x16_zero()}};
        score_t::template row_product<1, 1, 0>(s1, stage + DC / HN * tile_t::ES, k0, qf + 1, l32, h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[0][0][e] += s1[0][0][e];
      }
      if constexpr (CS > 1) attn_exchange<true>(s[0][0], ex + w_ * 1024, ex + (w_ ^ 1) * 1024, lane);
      float mx[NB];
      bool grew = false;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        mx[n] = s[0][n][0];
#pragma unroll
        for (int k = 0; k < KK; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx[n] = fmaxf(mx[n], s[k][n][e]);
        mx[n] = attn_half_max(mx[n]);
        grew |= m[n].below(mx[n], p.scale_log2) > 8.f;
      }
      // A row's reference point m follows its running maximum only when that has grown by more than 2^8: terms up to 2^8 round no worse than
      // terms up to 1 and their sums are far from any limit, and with m at every new maximum most tiles would rescale the sums.  (Row by
      // row: what a row comes to does not depend on the rows beside it.)
      if (__any(grew)) {
        far = false;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const bool up = m[n].below(mx[n], p.scale_log2) > 8.f;
          const attn_ref at_max = attn_ref_at(mx[n], p.scale_log2), mn = {up ? at_max.at : m[n].at, up ? at_max.is_far : m[n].is_far};
          const float a = up ? (m[n].any() ? fast_exp2(m[n].above(mn, p.scale_log2)) : 0.f) : 1.f;
          l[n] *= a;
#pragma unroll
          for (int d = 0; d < DC / 32; ++d) o[n][d] *= a;
          m[n] = mn;
          far |= mn.is_far;
        }
        far = __any(far);
      }
      if (far) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int k = 0; k < KK; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[k][n][e] -= m[n].far();
      }
#pragma unroll
      for (int k = 0; k < KK; ++k) {
        typename tile_t::template operand<PARTS> pr[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const float ref = m[n].any() ? m[n].ref() : 0.f;      // (no key yet in this row: every term is 2^-infinity = 0)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[k][n][e] = fast_exp2(fmaf(s[k][n][e], p.scale_log2, -ref));
          pr[n] = tile_t::template pack<PARTS>(s[k][n]);
          l[n] = tile_t::sum(pr[n], l[n]);
        }
        tile_t::template col_product<NB, PARTS>(o, stage + stream_t::TB + cs * DC * tile_t::ES, k0 + 32 * k, pr, lane);
      }
    }
  }
  if constexpr (KW > 1) {              // the wavefronts' rows meet in LDS, wavefront 0 goes on with them
    static_assert(NB == 1 && KW * 32 * (DP + 3) * 4 <= KW * 2 * stream_t::STAGE, "the rows fit where the tiles were");
    l[0] = attn_half_sum(l[0]);
    __syncthreads();
    constexpr int PART = 32 * (DP + 3);
    float* mine = (float*)attn_smem + kw * PART;
    if (kw > 0) {
#pragma unroll
      for (int d = 0; d < DC / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[(32 * d + attn_reg_row(e) + 4 * h) * 32 + l32] = o[0][d][e];
      if (h == 0) {
        mine[DP * 32 + l32] = m[0].at;
        mine[DP * 32 + 32 + l32] = l[0];
        mine[DP * 32 + 64 + l32] = m[0].is_far ? 1.f : 0.f;
      }
    }
    __syncthreads();
    if (kw > 0) return;
    attn_ref mw[KW], top = m[0];
    float f[KW];
    mw[0] = m[0];
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      mw[w] = attn_ref{mine[w * PART + DP * 32 + l32], mine[w * PART + DP * 32 + 64 + l32] != 0.f};
      const bool up = mw[w].any() && (!top.any() || mw[w].above(top, p.scale_log2) > 0.f);
      top = attn_ref{up ? mw[w].at : top.at, up ? mw[w].is_far : top.is_far};
    }
#pragma unroll
    for (int w = 0; w < KW; ++w) f[w] = mw[w].any() ? fast_exp2(mw[w].above(top, p.scale_log2)) : 0.f;
    l[0] *= f[0];
#pragma unroll
    for (int w = 1; w < KW; ++w) l[0] = fmaf(f[w], mine[w * PART + DP * 32 + 32 + l32], l[0]);
#pragma unroll
    for (int d = 0; d < DC / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = o[0][d][e] * f[0];
#pragma unroll
        for (int w = 1; w < KW; ++w) x = fmaf(f[w], mine[w * PART + (32 * d + attn_reg_row(e) + 4 * h) * 32 + l32], x);
        o[0][d][e] = x;
      }
    m[0] = top;
    l[0] *= 0.5f;                      // (both halves hold the whole sum; they are added below)
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float sum = attn_half_sum(l[n]);
    const bool any = sum > 0.f || sum != sum;
    const float inv = any ? 1.f / sum : 0.f;                // no key at all: zeros
    const float lse = any ? (m[n].any() ? m[n].ref() : 0.f) + fast_log2(sum) : -INFINITY;
    const int row = row0 + 32 * n;
    if (row >= p.R) continue;
    if (p.splits > 1) {
      const int64_t pr = (int64_t)at.base * p.Hk * p.R + ((int64_t)hk * p.R + row) * at.splits + split;
      if (h == 0 && cs == 0) {
        p.part_lse[2 * pr] = lse;
        p.part_lse[2 * pr + 1] = m[n].far();
      }
      tile_t::store_row(o[n], inv, p.part_o + pr * p.D + cs * DC, (float*)nullptr, p.D - cs * DC, h);
    } else {
      const attn_row rw(p, hk, row);
      if (h == 0 && cs == 0 && p.lse) {
        p.lse[(int64_t)prob * p.R + row] = lse;
        p.far[(int64_t)prob * p.R + row] = m[n].far();
      }
      const int64_t off = (((int64_t)b * p.Tq + rw.t) * p.H + rw.head) * p.D + cs * DC;
      tile_t::store_row(o[n], inv, (T*)p.out + off, p.out_lo ? (T*)p.out_lo + off : (T*)nullptr, p.D - cs * DC, h);
    }
  }
}

// Joins the splits of a row: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max), the logs taken from the largest far of the parts on (a part
// with a smaller far is exactly as far below as the difference says, or has no weight at all).  W wavefronts per row: a lane owns four channels and
// every n-th split (n = 64 W / lanes per row), loads several splits ahead, and the lanes' sums meet by shuffles and, for W > 1, in LDS.
// Bound by latency: 32 rows of 105 parts and 128 channels take 9.2 us with one wavefront per row and 5.5 with four.
template <typename T, int W>
__global__ __launch_bounds__(256) void attn_combine_kernel(attn_args p) {
  __shared__ float red[W > 1 ? W * 260 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t id = (int64_t)blockIdx.x * (4 / W) + (W > 1 ? 0 : wave);
  if (id >= (int64_t)p.B * p.Hk * p.R) return;                     // (W > 1: the whole workgroup)
  const int prob = (int)(id / p.R), row = (int)(id - (int64_t)prob * p.R);
  const int b = prob / p.Hk, hk = prob - b * p.Hk;
  const int base = p.share ? p.share[2 * b] : b * p.splits, splits = p.share ? p.share[2 * b + 1] : p.splits;
  const int64_t first_part = (int64_t)base * p.Hk * p.R + ((int64_t)hk * p.R + row) * splits;
  const f32x2* lse = (const f32x2*)p.part_lse + first_part;       // (lse, far)
  const float* part = p.part_o + first_part * p.D;
  float mx = -INFINITY, far = 0.f;
  bool any = false, some_far = false;
  for (int s = lane; s < splits; s += 64) {
    const f32x2 x = lse[s];
    any |= x.x != -INFINITY;
    some_far |= x.y != 0.f;
    mx = fmaxf(mx, x.x);
  }
  any = __any(any);
  const auto log_at = [&](f32x2 x) { return x.x == -INFINITY ? -INFINITY : fmaf(x.y - far, p.scale_log2, x.x); };
  if (__any(some_far)) {
    far = mx = -INFINITY;
    for (int s = lane; s < splits; s += 64) far = fmaxf(far, lse[s].x == -INFINITY ? -INFINITY : lse[s].y);      // (a part without keys has none)
    far = wave_max(far);
    for (int s = lane; s < splits; s += 64) mx = fmaxf(mx, log_at(lse[s]));
  }
  mx = wave_max(mx);
  const float top = mx > -INFINITY ? mx : 0.f;
  const int per = p.D <= 64 ? 16 : p.D <= 128 ? 32 : 64;           // lanes per row
  const int c = 4 * (lane & (per - 1)), first = (W > 1 ? wave * (64 / per) : 0) + lane / per, step = W * (64 / per);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float z = 0.f;
  if (c < p.D) {
#pragma unroll 4
    for (int s = first; s < splits; s += step) {
      const float w = fast_exp2(log_at(lse[s]) - top);
      z += w;
      o += *(const f32x4*)(part + (int64_t)s * p.D + c) * w;
    }
  }
  for (int x = per; x < 64; x *= 2) {
    z += __shfl_xor(z, x, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
  }
  if (W > 1) {
    if (lane < per) {
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave * 260 + 4 * lane + e] = o[e];
      if (lane == 0) red[wave * 260 + 256] = z;
    }
    __syncthreads();
    if (wave > 0 || lane >= per) return;
    z = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < W; ++w) {
      z += red[w * 260 + 256];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += red[w * 260 + 4 * lane + e];
    }
  }
  if (lane >= per || c >= p.D) return;
  const attn_row rw(p, hk, row);
  const int64_t off = (((int64_t)b * p.Tq + rw.t) * p.H + rw.head) * p.D + c;
  o *= any ? 1.f / z : 0.f;
  attn_store4((T*)p.out + off, o);
  if (sizeof(T) == 2 && p.out_lo) attn_store4((T*)p.out_lo + off, o - __builtin_convertvector(__builtin_convertvector(o, bf16x4), f32x4));
  if (lane == 0 && p.lse) {
    p.lse[id] = any ? top + fast_log2(z) : -INFINITY;
    p.far[id] = far;
  }
}

// ---------------------------------------------------------------------------------------------------------------- backward
// dq, and delta_i = do_i . o_i on the way (the dk / dv kernel reads it).  o is taken as out + out_lo: with the output rounded to bfloat16
// alone the error of delta (2^-9 |o| |do|, the same for every key of a row) would reach dq times the mean key.
template <typename T, int DP, int BN, int WM>
__global__ ATTN_WAVES(64 * WM, (WM == 1 ? 1 : attn_waves<T, DP, 3>())) void attn_bwd_dq_kernel(attn_args p) {
  constexpr int CS = WM > 1 ? attn_cs(DP, sizeof(T) == 4) : 1, DC = DP / CS;
  typedef attn_tile<T, DC, DP> tile_t;
  typedef typename tile_t::frag frag;
  typedef attn_stream<T, DP, BN, WM> stream_t;
  extern __shared__ __attribute__((aligned(1024))) char attn_smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  attn_item at;
  if (!attn_place<(WM > 1)>(p, p.row_tiles, BN, at)) return;
  const int b = at.b, hk = at.hk, prob = at.prob, tile = at.tile, split = at.split;

  const int cs = CS > 1 ? wave % CS : 0;                      // which part of the channels
  float* const ex = (float*)(attn_smem + 2 * stream_t::STAGE);
  const int row = (tile * (WM / CS) + wave / CS) * 32 + l32;
  const attn_row rw(p, hk, row);
  frag qf[tile_t::NP], gf[tile_t::NP];
  tile_t::load_row(qf, (const T*)p.q + b * p.q_sb + (int64_t)rw.t * p.q_st + (int64_t)rw.head * p.q_sh + cs * DC, p.D - cs * DC, h);
  const int64_t off = (((int64_t)b * p.Tq + rw.t) * p.H + rw.head) * p.D + cs * DC;
  tile_t::load_row(gf, (const T*)p.dout + off, p.D - cs * DC, h);
  float delta = tile_t::row_dot(gf, (const T*)p.out + off, p.out_lo ? (const T*)p.out_lo + off : (const T*)nullptr, p.D - cs * DC, h);
  delta = attn_half_sum(delta);
  if constexpr (CS > 1) {
    ex[wave * 64 + lane] = delta;
    __syncthreads();
    delta += ex[(wave ^ 1) * 64 + lane];
    __syncthreads();
  }
  float lse = p.lse[(int64_t)prob * p.R + rw.row];
  const float far = p.far[(int64_t)prob * p.R + rw.row];
  const bool some_far = __any(far != 0.f);
  if (split == 0 && h == 0 && cs == 0 && row < p.R) p.delta[(int64_t)prob * p.R + row] = -delta;
  if (lse == -INFINITY) lse = INFINITY;       // a row without any key: p = 0

  const f32x16 start = f32x16_all(cs == 0 ? -delta : 0.f);      // the products v . do start from minus delta: no subtraction per score
  f32x16 acc[DC / 32];
#pragma unroll
  for (int d = 0; d < DC / 32; ++d) acc[d] = f32x16_zero();

  stream_t in(p, b, hk, at.keys, wave, lane);
  int t0, t1;
  attn_part(in.tiles(), split, at.splits, t0, t1);
  in.seek(t0);
  uint64_t live_next = 0;
  if (t0 < t1) {
    in.peek();
    live_next = in.issue(attn_smem);
  }
  for (int t = t0; t < t1; ++t) {
    char* stage = attn_smem + ((t - t0) & 1) * stream_t::STAGE;
    const uint64_t live = live_next;
    attn_wait_dma();
    __syncthreads();
    if (t + 1 < t1) live_next = in.issue(attn_smem + ((t + 1 - t0) & 1) * stream_t::STAGE);
    if (live == 0) continue;
    constexpr int PRE = DP == 256 && sizeof(T) == 2 ? 2 : 0;      // one wavefront per SIMD: nobody else hides the LDS
    constexpr int KK = BN / 32;          // blocks of 32 keys, all at a time: so many independent chains of products
    static_assert(CS == 1 || BN == 32, "one pair of exchanges between two barriers");
    f32x16 s[KK][1], dp[KK][1];
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      s[k][0] = stream_t::start(stage, 32 * k, live, h);
      dp[k][0] = start;
    }
    tile_t::template row_product<KK, 1, PRE>(s, stage + cs * DC * tile_t::ES, 0, &qf, l32, h);
    tile_t::template row_product<KK, 1, PRE>(dp, stage + stream_t::TB + cs * DC * tile_t::ES, 0, &gf, l32, h);
    if constexpr (CS > 1) {
      attn_exchange<false>(s[0][0], ex + wave * 1024, ex + (wave ^ 1) * 1024, lane);
      attn_exchange<true>(dp[0][0], ex + wave * 1024, ex + (wave ^ 1) * 1024, lane);
    }
    if (some_far) {
#pragma unroll
      for (int k = 0; k < KK; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[k][0][e] -= far;
    }
#pragma unroll
    for (int k = 0; k < KK; ++k) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[k][0][e] = fast_exp2(fmaf(s[k][0][e], p.scale_log2, -lse)) * dp[k][0][e];
      const auto ds = tile_t::template pack<attn_parts<T>(true)>(s[k][0]);
      tile_t::template col_product<1, attn_parts<T>(true)>(&acc, stage + cs * DC * tile_t::ES, 32 * k, &ds, lane);
    }
  }
  if (row >= p.R) return;
  const int64_t sample = (int64_t)p.Tq * p.H * p.D;
  if (p.splits > 1) tile_t::store_row(acc, 1.f, p.part_o + (at.base + split - b) * sample + off, (float*)nullptr, p.D - cs * DC, h);
  else tile_t::store_row(acc, p.scale, (T*)p.dq + off, (T*)nullptr, p.D - cs * DC, h);
}

// dk and dv: a wavefront owns 32 keys, their k and v rows in registers, and walks over the rows; q and do tiles in LDS serve both as rows
// (scores) and, transposed, as the second products' first operand.
template <typename T, int DP, int BQ, int WM, int PARTS>
__global__ ATTN_WAVES(64 * WM, (attn_waves<T, DP, 3>())) void attn_bwd_dkv_kernel(attn_args p) {
  constexpr int CS = attn_cs(DP, sizeof(T) == 4), DC = DP / CS;
  typedef attn_tile<T, DC, DP> tile_t;
  typedef typename tile_t::frag frag;
  typedef attn_rows<T, DP, BQ, WM> rows_t;
  extern __shared__ __attribute__((aligned(1024))) char attn_smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, l32 = lane & 31;
  attn_item at;
  if (!attn_place_keys(p, 32 * WM / CS, (p.R + BQ - 1) / BQ, at)) return;
  const int b = at.b, hk = at.hk, prob = at.prob, tile = at.tile, split = at.split;

  const int cs = CS > 1 ? wave % CS : 0;                      // which part of the channels
  float* const ex = (float*)(attn_smem + 2 * rows_t::STAGE);
  const int key = (tile * (WM / CS) + wave / CS) * 32 + l32;
  const attn_keys keys(p, b, at.keys);
  const bool mine = keys.alive(key);
  const int64_t kr = min(key, p.Tk - 1);
  const T* kp = (const T*)p.k + b * p.k_sb + (int64_t)hk * p.k_sh + kr * p.k_st + cs * DC;
  const T* vp = (const T*)p.v + b * p.v_sb + (int64_t)hk * p.v_sh + kr * p.v_st + cs * DC;
  frag kf[tile_t::NP], vf[tile_t::NP];
  tile_t::load_row(kf, kp, p.D - cs * DC, h);
  tile_t::load_row(vf, vp, p.D - cs * DC, h);
  f32x16 dk[DC / 32], dv[DC / 32];
#pragma unroll
  for (int d = 0; d < DC / 32; ++d) { dk[d] = f32x16_zero(); dv[d] = f32x16_zero(); }

  int t0, t1;
  attn_part(__syncthreads_or(mine) ? (p.R + BQ - 1) / BQ : 0, split, at.splits, t0, t1);      // no key of this workgroup exists: zeros
  rows_t in(p, b, hk, prob, t0, wave, lane);
  if (t0 < t1) in.issue(p, attn_smem);
  for (int t = t0; t < t1; ++t) {
    const char* qt = attn_smem + ((t - t0) & 1) * rows_t::STAGE;
    const char* gt = qt + rows_t::TB;
    attn_wait_dma();
    __syncthreads();
    const bool some_far = in.some_far();
    if (t + 1 < t1) in.issue(p, attn_smem + ((t + 1 - t0) & 1) * rows_t::STAGE);
    static_assert(CS == 1 || BQ == 32, "one pair of exchanges between two barriers");
#pragma unroll 1
    for (int qq = 0; qq < BQ / 32; ++qq) {
      constexpr int PRE = DP == 256 && sizeof(T) == 2 ? 4 : 0;
      const float* st = (const float*)(qt + 2 * rows_t::TB) + 32 * qq + 4 * h;
      f32x16 s[1][1] = {{f32x16_zero()}}, dp[1][1] = {{f32x16_zero()}};
      if (cs == 0) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 de = *(const f32x4*)(st + 64 + 8 * g);                // the products v . do start from minus delta
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[0][0][4 * g + e] = de[e];
        }
      }
      tile_t::template row_product<1, 1, PRE>(s, qt + cs * DC * tile_t::ES, 32 * qq, &kf, l32, h);
      tile_t::template row_product<1, 1, PRE>(dp, gt + cs * DC * tile_t::ES, 32 * qq, &vf, l32, h);
      if constexpr (CS > 1) {
        attn_exchange<false>(s[0][0], ex + wave * 1024, ex + (wave ^ 1) * 1024, lane);
        attn_exchange<true>(dp[0][0], ex + wave * 1024, ex + (wave ^ 1) * 1024, lane);
      }
      if (some_far) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 far = *(const f32x4*)(st + 128 + 8 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][0][4 * g + e] -= far[e];
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ls = *(const f32x4*)(st + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pr = fast_exp2(fmaf(s[0][0][4 * g + e], p.scale_log2, -ls[e]));
          s[0][0][4 * g + e] = pr;
          dp[0][0][4 * g + e] *= pr;
        }
      }
      const auto pr = tile_t::template pack<PARTS>(s[0][0]);
      const auto ds = tile_t::template pack<attn_parts<T>(true)>(dp[0][0]);
      tile_t::template col_product<1, PARTS>(&dv, gt + cs * DC * tile_t::ES, 32 * qq, &pr, lane);
      tile_t::template col_product<1, attn_parts<T>(true)>(&dk, qt + cs * DC * tile_t::ES, 32 * qq, &ds, lane);
    }
  }
  if (key >= p.Tk) return;
  const int64_t off = (((int64_t)b * p.Tk + key) * p.Hk + hk) * p.D + cs * DC;
  if (!mine) {                        // (a select, not a factor: the sums of a key that does not exist may be anything)
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) { dk[d] = f32x16_zero(); dv[d] = f32x16_zero(); }
  }
  if (p.splits > 1) {
    constexpr int KEYS = 32 * WM / CS;
    float* part = p.part_o + ((((int64_t)at.base * at.splits + split) * p.Hk + hk) * 2 * KEYS + key - tile * KEYS) * p.D + cs * DC;
    tile_t::store_row(dk, 1.f, part, (float*)nullptr, p.D - cs * DC, h);
    tile_t::store_row(dv, 1.f, part + KEYS * p.D, (float*)nullptr, p.D - cs * DC, h);
  } else {
    tile_t::store_row(dk, p.scale, (T*)p.dk + off, (T*)nullptr, p.D - cs * DC, h);
    tile_t::store_row(dv, 1.f, (T*)p.dv + off, (T*)nullptr, p.D - cs * DC, h);
  }
}

// adds the parts of dq in their order: dq[i] = scale * sum_s part_s[i], four values per thread (D % 4 == 0; with parts dq has less than 2^31 values)
template <typename T>
__global__ __launch_bounds__(256) void attn_reduce_q_kernel(attn_args p) {
  const uint32_t sample = (uint32_t)(p.Tq * p.H * p.D), i = (blockIdx.x * 256 + threadIdx.x) * 4, b = i / sample;
  if (b >= (uint32_t)p.B) return;
  const int base = p.share ? p.share[2 * b] : b * p.splits, splits = p.share ? p.share[2 * b + 1] : p.splits;
  const float* at = p.part_o + (int64_t)base * sample + (i - b * sample);
  f32x4 a = *(const f32x4*)at;
#pragma unroll 4
  for (int s = 1; s < splits; ++s) a += *(const f32x4*)(at + (int64_t)s * sample);
  attn_store4((T*)p.dq + i, a * p.scale);
}

// the same for dk (blockIdx.y = 0) and dv, whose parts lie in tiles of `keys` keys; tiles without keys have no parts
template <typename T>
__global__ __launch_bounds__(256) void attn_reduce_kv_kernel(attn_args p, int keys) {
  const uint32_t head = (blockIdx.x * 256 + threadIdx.x) * 4 / p.D, d = (blockIdx.x * 256 + threadIdx.x) * 4 - head * p.D;
  const uint32_t row = head / p.Hk, hk = head - row * p.Hk, b = row / p.Tk, key = row - b * p.Tk, tile = key / keys;
  if (b >= (uint32_t)p.B) return;
  const int base = p.share ? p.share[2 * b] : b * p.key_tiles, tiles = p.share ? p.share[2 * b + 1] : p.key_tiles;
  const int splits = p.share ? p.share[2 * 64] : p.splits;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  if (tile < (uint32_t)tiles) {
    const int64_t step = (int64_t)p.Hk * 2 * keys * p.D;
    const float* at = p.part_o + (base + tile) * splits * step + ((hk * 2 + blockIdx.y) * keys + key - tile * keys) * p.D + d;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) a += *(const f32x4*)(at + s * step);
  }
  const int64_t i = (int64_t)head * p.D + d;
  if (blockIdx.y) attn_store4((T*)p.dv + i, a);
  else attn_store4((T*)p.dk + i, a * p.scale);
}

// ---------------------------------------------------------------------------------------------------------------- host
// wavefronts along the keys in the forward's form for few rows: two stages of 32 keys each, in 128 KiB of LDS (float32 with 256 channels
// would have room for one only, and takes the form for many rows)
static constexpr int attn_kw(int dp, bool f32) { return dp * (f32 ? 4 : 2) <= 256 ? 4 : 2; }

static int attn_check(const ttdg_attention_t* a, const char* what) {
  static thread_local char msg[160];
#define ATTN_REQUIRE(cond, text)                                        \
  do {                                                                  \
    if (!(cond)) {                                                      \
      snprintf(msg, sizeof(msg), "%s: %s", what, text);                 \
      return ttdg_fail(TTDG_EINVAL, msg);                               \
    }                                                                   \
  } while (0)
  ATTN_REQUIRE(a->dtype == TTDG_F32 || a->dtype == TTDG_BF16, "dtype must be TTDG_F32 or TTDG_BF16");
  ATTN_REQUIRE(a->B >= 0 && a->Tq >= 0 && a->Tk >= 0 && a->H >= 1 && a->Hkv >= 1, "negative size or no head");
  ATTN_REQUIRE(a->H % a->Hkv == 0, "the number of query heads must be a multiple of the number of key heads");
  const int ce = a->dtype == TTDG_F32 ? 4 : 8, es = a->dtype == TTDG_F32 ? 4 : 2;
  ATTN_REQUIRE(a->D >= 8 && a->D <= 256 && a->D % 8 == 0, "the head dimension must be a multiple of 8 up to 256");
  ATTN_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "the scale must be positive and finite");
  if (a->B == 0 || a->Tq == 0) return 0;
  ATTN_REQUIRE(a->q && (a->Tk == 0 || (a->k && a->v)), "null pointer");
  const int64_t st[9] = {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh};
  for (int i = 0; i < 9; ++i) ATTN_REQUIRE(st[i] >= 0 && st[i] % ce == 0, "strides must be multiples of 16 bytes");
  ATTN_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) % 16 == 0, "q, k and v must be 16-byte aligned");
  // offsets inside a tile are 32-bit: 64 rows, of the queries spread over the G heads of a key head
  const int64_t lim = (int64_t)0x7f000000 / es;
  ATTN_REQUIRE(a->k_st <= lim / 64 && a->v_st <= lim / 64, "key / value rows too far apart");
  ATTN_REQUIRE(a->q_st <= lim / 130 && a->q_sh <= lim / 2 / (a->H / a->Hkv), "query rows or heads too far apart");
  const int64_t R = (int64_t)a->Tq * (a->H / a->Hkv);
  ATTN_REQUIRE(R < (1 << 30) && a->Tk < (1 << 30) && (int64_t)a->B * a->Hkv < (1 << 24), "too many rows, keys or heads");
  ATTN_REQUIRE((int64_t)a->H * a->D <= (1 << 20), "more than 2^20 channels in all heads");
  ATTN_REQUIRE(a->m_sb >= 0 && a->m_st >= 0, "negative mask stride");
#undef ATTN_REQUIRE
  return 0;
}

static attn_args attn_make(const ttdg_attention_t* a) {
  attn_args p = {};
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.k_sb = a->k_sb; p.k_st = a->k_st; p.k_sh = a->k_sh;
  p.v_sb = a->v_sb; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.k_lens = a->k_lens; p.key_mask = a->key_mask; p.m_sb = a->m_sb; p.m_st = a->m_st;
  p.B = a->B; p.Tq = a->Tq; p.Tk = a->Tk; p.H = a->H; p.Hk = a->Hkv; p.D = a->D;
  p.G = a->H / a->Hkv; p.R = a->Tq * p.G;
  p.scale = a->scale; p.scale_log2 = a->scale * TTDG_LOG2E;
  p.out = a->out; p.out_lo = a->dtype == TTDG_BF16 ? a->out_lo : nullptr; p.lse = a->lse; p.far = a->lse ? a->lse + (size_t)a->B * a->Hkv * a->Tq * (a->H / a->Hkv) : nullptr;
  p.dout = a->dout; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  p.splits = 1;
  return p;
}

// How many workgroups share one (problem, tile): the long axis (`units` tiles of it) is split into s parts when that shortens the estimated
// time in microseconds: `tile_us` per tile with all of the chip's `slots` taken (where several workgroups fit on a CU, one alone there runs up to
// twice as fast, so the rounds are not counted in full), 6 us per workgroup (first loads, last stores), and for the join a launch and the parts written and read once (`part_bytes` each)
// at 5 TB/s.  Measured both ways: dk / dv of 8 x 256 rows over 794 ragged keys, float32, 256 channels (104 workgroups for 256 slots) 83 us
// unsplit, 43 + 9 for the sums in two parts; of 8 x 1000 x 12 heads x 64 over 1500 keys (1152 for 768) 122 unsplit, 144 + 34 in two; of 4 x 2047
// rows x 16 heads over 4 x 2500 keys (320 for 512) 570 unsplit, 539 + 18 in two, 449 + 24 in three, where the estimate says two.
static int attn_splits(int64_t blocks, int units, int slots, double tile_us, double part_bytes, double* estimate = nullptr) {
  int best = 1;
  double least = 0;
  if (estimate) *estimate = 0;
  if (units < 1 || blocks < 1) return 1;
  for (int s = 1; s <= 256 && (s == 1 || 2 * s <= units) && (s == 1 || blocks * s <= 8 * (int64_t)slots); ++s) {
    const int per = (units + s - 1) / s;
    const double full = (double)blocks * s / slots, rounds = (double)((blocks * s + slots - 1) / slots);
    const double taken = slots <= 256 ? rounds : full < 1 ? 0.5 + 0.5 * full : full + 0.1 * (rounds - full);
    const double us = taken * (per * tile_us + 6) + (s > 1 ? 3 + 2 * s * part_bytes / 5e6 : 0);
    if (s == 1 || us < 0.97 * least) { least = us; best = (units + per - 1) / per; }
  }
  if (estimate) *estimate = least;
  return best;
}

struct attn_plan {
  int dp, slots, few, nb, fwd_cs, fwd_tiles, row_tiles, fwd_splits, dq_splits, key_tiles, dkv_splits, fwd_share, dq_share, dkv_share, fwd_two, dkv_two;
  int64_t dkv_grid;
  size_t fwd_ws, bwd_ws;
};

// keys per tile of the kernels that share tiles between wavefronts; 32 where wavefronts have their own
static int attn_bn(int dp, bool f32) { return dp == 64 || (dp == 128 && !f32) ? 64 : 32; }

#define ATTN_SHARE_BYTES ((2 * 64 + 4) * 4)

static attn_plan attn_planned(const ttdg_attention_t* a) {
  attn_plan q;
  const bool f32 = a->dtype == TTDG_F32;
  const int64_t probs = (int64_t)a->B * a->Hkv;
  const int64_t R = (int64_t)a->Tq * (a->H / a->Hkv);
  q.dp = a->D <= 64 ? 64 : a->D <= 128 ? 128 : 256;
  const int bn = attn_bn(q.dp, f32);
  // 256 CUs; workgroups per CU by the registers and LDS of the kernels
  const int shared = q.dp == 256 || (q.dp == 128 && f32) ? 256 : q.dp == 128 || f32 ? 512 : 768;
  q.slots = shared;
  const int wg = attn_rows_wg(q.dp, f32);
  // One wavefront's 32 rows hold all.  Two such tiles of 33 to 64 rows would read the keys twice: 2 x 48 rows over 53294 keys, one key head x 128,
  // bfloat16, take 19 us in the form for many rows (32 rows: 16), float32 with 64 channels 43 (20), with 128 channels 64 rows 77 (64).
  q.few = R <= 32 && !(f32 && q.dp == 256);
  q.row_tiles = q.few ? 1 : (int)((R + wg - 1) / wg);
  // 64 rows per wavefront where the workgroups still go round twice: 16 x 2048 rows over 4096 keys, 8 heads, 654 -> 618 us; with fewer workgroups
  // the rounds decide (batch 4: 167 -> 173 us and a join of 32, 8: 360 -> 348, 9: 406 -> 443).  With 64 channels 361 -> 378 us.
  q.nb = !f32 && q.dp == 128 && !q.few && probs * ((R + 255) / 256) >= 1024 ? 2 : 1;
  const int kt = (a->Tk + bn - 1) / bn, kt32 = (a->Tk + 31) / 32, kw = attn_kw(q.dp, f32);
  // a tile's time at 800 (bf16) / 110 TFLOP/s (fp32) for the products of a full chip; few rows: its bytes at 20 GB/s per CU
  const double es = f32 ? 4 : 2, prod_us = 2.0 * wg * bn * q.dp * shared / (f32 ? 110e6 : 800e6);
  const double q_bytes = (double)probs * R * a->D * 4, kv_bytes = 2.0 * a->B * a->Tk * a->Hkv * a->D * 4;
  const int fwd_wg = 128 * q.nb;
  const bool pairs = attn_cs(q.dp, f32) > 1;          // (prod_us is the time of 64 rows with the exchange; 128 without take 1.74 times as long)
  q.fwd_cs = 1;
  q.fwd_tiles = q.few ? 1 : (int)((R + fwd_wg - 1) / fwd_wg);
  double us = 0, us2 = 0;
  q.fwd_splits = q.few ? attn_splits(probs, (kt32 + kw - 1) / kw, 1024 / kw, kw * 2 * 32 * a->D * es / 20e3, q_bytes)
                           : attn_splits(probs * q.fwd_tiles, kt, shared, (pairs ? 2 * 1.74 : 2.0 * q.nb) * prod_us, q_bytes, &us);
  if (pairs) {                       // 64 rows per workgroup where that fills the chip better
    const int splits = attn_splits(probs * q.row_tiles, kt, shared, 2 * prod_us, q_bytes, &us2);
    if (us2 < us) { q.fwd_cs = 2; q.fwd_tiles = q.row_tiles; q.fwd_splits = splits; }
  }
  // few rows: workgroups of one wavefront, as many per CU as their two stages of LDS leave room for (one token of 4 x 16 heads x 128 over 20000
  // keys, float32: 16 parts 272 us, 32 parts 148, 64 parts 155; 8 heads x 256 over 30000, bfloat16: 31 parts 88, 62 parts 55, 124 parts 67;
  // + 4, 6 and 9 us for the sums.  Elsewhere the estimate's parts are the best of half, twice and four times as many, or within 2 us)
  const int dq_slots = q.few ? (q.dp == 64 && !f32 ? 1024 : 512) : shared;
  q.dq_splits = attn_splits(probs * q.row_tiles, kt, dq_slots, 3 * prod_us, q_bytes);
  q.key_tiles = (a->Tk + wg - 1) / wg;
  const int qt = (int)((R + bn - 1) / bn);
  q.dkv_splits = attn_splits(probs * q.key_tiles, qt, shared, 4 * prod_us, kv_bytes);
  q.fwd_two = q.few || (q.nb == 1 && 2 * probs * q.fwd_tiles * q.fwd_splits <= shared);        // (see attn_parts)
  q.dkv_two = 2 * probs * q.key_tiles * q.dkv_splits <= shared;
  // Ragged samples: only the device knows their lengths, and the kernels divide by them (attn_place) where the workgroups run all at once.  What
  // the host says is how many parts there may be: as many as the chip has slots for.  Forward and backward of 8 x 256 rows over
  // up to 794 keys, float32, 256 channels: 152 -> 134 us with 447 to 794 keys, 140 -> 88 us with one sample of 794 and seven of 40 to 160; what
  // the division costs when all are alike: 1.6 us of 79 (8 x 64 rows over 128 keys).
  const bool ragged = a->k_lens && a->B > 1 && a->B <= 64;
  const auto share = [&](int& splits, int64_t blocks) {
    if (!ragged || q.few || splits < 2 || blocks * splits > shared) return 0;
    const int64_t most = shared / blocks < kt / 2 ? shared / blocks : kt / 2;
    if (most > splits) splits = (int)most;
    return 1;
  };
  q.fwd_share = share(q.fwd_splits, probs * q.fwd_tiles);
  q.dq_share = share(q.dq_splits, probs * q.row_tiles);
  q.dkv_grid = probs * q.key_tiles * q.dkv_splits;
  q.dkv_share = ragged && q.dkv_splits > 1;
  if (q.dkv_share && q.dkv_grid < shared) q.dkv_grid = shared / a->Hkv * a->Hkv;
  const size_t rows = (size_t)probs * R;
  q.fwd_ws = q.fwd_splits > 1 ? (size_t)q.fwd_splits * rows * (a->D + 2) * 4 + ATTN_SHARE_BYTES : 0;
  const size_t dq = q.dq_splits > 1 ? (size_t)q.dq_splits * rows * a->D * 4 : 0, dkv = q.dkv_splits > 1 ? (size_t)q.dkv_grid * 2 * wg * a->D * 4 : 0;
  q.bwd_ws = rows * 4 + 16 + ATTN_SHARE_BYTES + (dq > dkv ? dq : dkv);
  return q;
}

extern "C" size_t ttdg_attention_fwd_workspace_bytes(const ttdg_attention_t* a) {
  if (!a || attn_check(a, "attention_fwd_workspace_bytes")) return 0;
  return a->B && a->Tq ? attn_planned(a).fwd_ws : 0;
}

extern "C" size_t ttdg_attention_bwd_workspace_bytes(const ttdg_attention_t* a) {
  if (!a || attn_check(a, "attention_bwd_workspace_bytes")) return 0;
  return a->B && a->Tq ? attn_planned(a).bwd_ws : 0;
}

extern "C" int ttdg_attention_forms(const ttdg_attention_t* a, ttdg_attention_forms_t* forms) {
  TTDG_REQUIRE(a && forms, "attention_forms: null pointer");
  if (int e = attn_check(a, "attention_forms")) return e;
  *forms = ttdg_attention_forms_t{};
  if (a->B == 0 || a->Tq == 0) return 0;
  const attn_plan q = attn_planned(a);
  const bool bf16 = a->dtype == TTDG_BF16;
  *forms = {q.few, 32 * q.nb, q.fwd_cs, q.fwd_splits, q.dq_splits, q.dkv_splits, bf16 && q.fwd_two ? 2 : 1, bf16 && q.dkv_two ? 2 : 1};
  return 0;
}

#define ATTN_LAUNCH(kernel, grid, threads, lds, stream, args)                              \
  do {                                                                                     \
    TTDG_ALLOW_LDS((kernel), (lds));                                                       \
    hipLaunchKernelGGL((kernel), dim3((unsigned)(grid)), dim3(threads), (lds), (hipStream_t)(stream), args); \
    if (int e_ = ttdg_launch_status(#kernel)) return e_;                                   \
  } while (0)

template <typename T, int DP, int BN>
static int attn_fwd_launch(const attn_args& p, const attn_plan& q, ttdg_stream_t stream) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int WM = 4, lds = 2 * attn_stream<T, DP, BN, WM>::STAGE + attn_exchange_bytes(DP, F32);
  const int64_t grid = (int64_t)p.B * p.Hk * p.row_tiles * p.splits;         // (of the forward; a launch's threads are counted in 32 bits)
  TTDG_LIMIT(grid < (1ll << 24), "attention_fwd: too many workgroups");
  if constexpr (!(F32 && DP == 256)) {
    constexpr int KW = attn_kw(DP, F32), ldsk = 2 * KW * attn_stream<T, DP, 32, 1>::STAGE;
    if (q.few) ATTN_LAUNCH((attn_fwd_kernel<T, DP, 32, 1, 1, KW, attn_parts<T>(true), 1>), grid, 64 * KW, ldsk, stream, p);
  }
  if constexpr (attn_cs(DP, F32) > 1) {
    if (q.fwd_cs > 1) ATTN_LAUNCH((attn_fwd_kernel<T, DP, BN, WM, 1, 1, 1, attn_cs(DP, F32)>), grid, 64 * WM, lds, stream, p);
  }
  if (q.few || q.fwd_cs > 1) {
  } else if (q.fwd_two) ATTN_LAUNCH((attn_fwd_kernel<T, DP, BN, WM, 1, 1, attn_parts<T>(true), 1>), grid, 64 * WM, lds, stream, p);
  else if (q.nb == 1) ATTN_LAUNCH((attn_fwd_kernel<T, DP, BN, WM, 1, 1, 1, 1>), grid, 64 * WM, lds, stream, p);
  else if constexpr (sizeof(T) == 2 && DP == 128) ATTN_LAUNCH((attn_fwd_kernel<T, DP, BN, WM, 2, 1, 1, 1>), grid, 64 * WM, lds, stream, p);
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.B * p.Hk * p.R;
    // Four wavefronts per row where the rows alone do not fill the chip and the parts are many (one and four wavefronts, us: 32 rows of 105 parts
    // 9.2 / 5.5, 256 of 125 10.8 / 6.5, 512 of 63 6.1 / 5.1, 128 of 21 5.6 / 4.1, 1024 of 48 5.5 / 5.2; up to 16 parts the same within 0.1;
    // 2048 rows 5.4 / 6.0, 4096 5.9 / 9.4, 8192 6.2 / 14.1, whatever the parts, channels and lengths)
    if (rows <= 1024 && p.splits > 16) ATTN_LAUNCH((attn_combine_kernel<T, 4>), rows, 256, 0, stream, p);
    else ATTN_LAUNCH((attn_combine_kernel<T, 1>), (rows + 3) / 4, 256, 0, stream, p);
  }
  return 0;
}

template <typename T, int DP, int BN>
static int attn_bwd_launch(attn_args p, const attn_plan& q, ttdg_stream_t stream) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int WM = 4, lds = 2 * attn_stream<T, DP, BN, WM>::STAGE + attn_exchange_bytes(DP, F32);
  p.splits = q.dq_splits;
  int32_t* const share = p.share;
  if (!q.dq_share) p.share = nullptr;
  int64_t grid = (int64_t)p.B * p.Hk * p.row_tiles * p.splits;
  TTDG_LIMIT(grid < (1ll << 24), "attention_bwd: too many workgroups");
  if constexpr (!(F32 && DP == 256)) {
    if (q.few) ATTN_LAUNCH((attn_bwd_dq_kernel<T, DP, BN, 1>), grid, 64, lds, stream, p);
  }
  if (!q.few) ATTN_LAUNCH((attn_bwd_dq_kernel<T, DP, BN, WM>), grid, 64 * WM, lds, stream, p);
  const int64_t nq = (int64_t)p.B * p.Tq * p.H * p.D, nk = (int64_t)p.B * p.Tk * p.Hk * p.D;
  if (p.splits > 1) {
    hipLaunchKernelGGL(attn_reduce_q_kernel<T>, dim3((unsigned)((nq / 4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream, p);
    if (int e = ttdg_launch_status("attn_reduce")) return e;
  }
  if (p.Tk == 0 || !p.dk) return 0;
  p.splits = q.dkv_splits;
  p.share = q.dkv_share ? share : nullptr;
  grid = q.dkv_grid;
  TTDG_LIMIT(grid < (1ll << 24), "attention_bwd: too many workgroups");
  constexpr int lds2 = 2 * attn_rows<T, DP, BN, WM>::STAGE + attn_exchange_bytes(DP, F32);
  if (q.dkv_two) ATTN_LAUNCH((attn_bwd_dkv_kernel<T, DP, BN, WM, attn_parts<T>(true)>), grid, 64 * WM, lds2, stream, p);
  else ATTN_LAUNCH((attn_bwd_dkv_kernel<T, DP, BN, WM, 1>), grid, 64 * WM, lds2, stream, p);
  if (p.splits > 1) {
    hipLaunchKernelGGL(attn_reduce_kv_kernel<T>, dim3((unsigned)((nk / 4 + 255) / 256), 2), dim3(256), 0, (hipStream_t)stream, p,
                       attn_rows_wg(DP, F32));
    if (int e = ttdg_launch_status("attn_reduce")) return e;
  }
  return 0;
}

#define ATTN_DISPATCH(fn, a, ...)                                                                  \
  do {                                                                                             \
    if ((a)->dtype == TTDG_F32) {                                                                  \
      if (q.dp == 64) return fn<float, 64, 64>(__VA_ARGS__);                                       \
      if (q.dp == 128) return fn<float, 128, 32>(__VA_ARGS__);                                     \
      return fn<float, 256, 32>(__VA_ARGS__);                                                      \
    }                                                                                              \
    if (q.dp == 64) return fn<__bf16, 64, 64>(__VA_ARGS__);                                        \
    if (q.dp == 128) return fn<__bf16, 128, 64>(__VA_ARGS__);                                      \
    return fn<__bf16, 256, 32>(__VA_ARGS__);                                                       \
  } while (0)

extern "C" int ttdg_attention_fwd(const ttdg_attention_t* a, ttdg_stream_t stream) {
  TTDG_REQUIRE(a, "attention_fwd: null pointer");
  if (int e = attn_check(a, "attention_fwd")) return e;
  if (a->B == 0 || a->Tq == 0) return 0;
  TTDG_REQUIRE(a->out && (uintptr_t)a->out % 16 == 0 && (uintptr_t)a->out_lo % 16 == 0, "attention_fwd: out must be a 16-byte aligned pointer");
  const attn_plan q = attn_planned(a);
  TTDG_REQUIRE(q.fwd_ws == 0 || (a->ws && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= q.fwd_ws), "attention_fwd: workspace too small or misaligned");
  attn_args p = attn_make(a);
  p.row_tiles = q.fwd_tiles;
  p.splits = q.fwd_splits;
  p.part_o = (float*)a->ws;
  p.part_lse = p.part_o + (size_t)q.fwd_splits * p.B * p.Hk * p.R * p.D;
  p.share = q.fwd_share ? (int32_t*)(p.part_lse + 2 * (size_t)q.fwd_splits * p.B * p.Hk * p.R) : nullptr;
  ATTN_DISPATCH(attn_fwd_launch, a, p, q, stream);
}

extern "C" int ttdg_attention_bwd(const ttdg_attention_t* a, ttdg_stream_t stream) {
  TTDG_REQUIRE(a, "attention_bwd: null pointer");
  if (int e = attn_check(a, "attention_bwd")) return e;
  if (a->B == 0 || a->Tq == 0) {
    TTDG_REQUIRE(a->B == 0 || a->Tk == 0 || !a->dk, "attention_bwd: without queries dk and dv are zeros; fill them");
    return 0;
  }
  TTDG_REQUIRE(a->out && a->lse && a->dout && a->dq && (!a->dk == !a->dv), "attention_bwd: null pointer (dk and dv: both or none)");
  TTDG_REQUIRE(((uintptr_t)a->out | (uintptr_t)a->out_lo | (uintptr_t)a->dout | (uintptr_t)a->dq | (uintptr_t)a->dk | (uintptr_t)a->dv) % 16 == 0,
               "attention_bwd: out, dout and the gradients must be 16-byte aligned");
  const attn_plan q = attn_planned(a);
  TTDG_REQUIRE(a->ws && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= q.bwd_ws, "attention_bwd: workspace too small or misaligned");
  attn_args p = attn_make(a);
  p.row_tiles = q.row_tiles;
  p.key_tiles = q.key_tiles;
  p.slots = q.slots;
  p.delta = (float*)a->ws;
  p.share = (int32_t*)(p.delta + (((size_t)p.B * p.Hk * p.R + 3) & ~(size_t)3));
  p.part_o = (float*)p.share + ATTN_SHARE_BYTES / 4;
  ATTN_DISPATCH(attn_bwd_launch, a, p, q, stream);
}
