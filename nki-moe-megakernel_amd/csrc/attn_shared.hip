// Decode attention of a batch whose sequences share prefixes, on a paged KV cache
// (mkd_attention_shared_prefix).
//
// The softmax over a sequence's keys splits at any position into partials (max m, sum
// l, weighted values O) that join exactly: O = sum_c 2^(m_c - m) O_c, l alike.  So the
// prefix of a group is attended once by a matrix of ALL its query rows (sequences x new
// tokens x the kv head's query heads), each sequence's own positions by its own rows,
// and a second launch joins a row's partials:
//   1. units of both kinds in one grid, the sequences' own first (short ones, beside which
//      the prefixes' start): (chunk of positions, kv head, tile of a sequence's rows), and
//      (chunk, kv head, tile of a group's rows)
//   2. combine: one wave per row over its live chunks, the sink joined there
//
// Per 32-position step a wave with QT tiles of 16 query rows forms
//   S = K . q^T   v_mfma_f32_16x16x32_bf16, A = 16 K rows, B = 16 query rows;
//                 D lane l holds S[position 4 (l/16) + i][row l % 16]
//   O += P . V    P straight from the S layout, V rows transposed by byte permutes
//   l += P . 1    the sum of the same rounded P, by one more MFMA
// P is rounded to bf16 for the matrix instruction (a relative 2^-9 of each term, the
// rounding of the output itself); scores, maxima, l and O stay fp32.
//
// staged (more than 32 query rows): the block's 4 waves hold 16 QT rows each and share
// the steps' K and V rows through a ring of three LDS stages filled asynchronously
// (global_load_lds), one barrier a step.  direct (few rows, and every sequence's own
// positions): the waves take steps of their own, rows straight to registers a step ahead,
// and merge at the end: nothing to share, and no barrier to wait at.
//
// What bounds it (64 sequences, 32 heads over 4 kv heads of 128, prefix 8192, own 512:
// 52 MB, 8.9 GFLOP): the units take 26.7 us, 2.0 TB/s and 0.33 PFLOP/s, the join 6.1 us (19
// MB of partials written and read).  A prefix unit is 16 steps of 1820 cycles, in which a
// wave issues 34 MFMAs, 16 16-byte LDS reads a lane, 16 exponentials, 32 byte permutes; with
// one wave of each kind per SIMD these follow one another more than they overlap.  Without
// the copies a step takes 8 % less, without the exponentials 13, without Q . K 11, without
// P . V 14; K rows read two steps ahead and scores formed one step ahead gave 2 %, a ring of
// four stages nothing.  FP8 rows (32 sequences, prefix 32768): 42.6 us, 2015 cycles a step,
// the conversions to bf16 in place of half the copies.
//
// whole (short contexts): one direct unit takes a sequence's prefix and own positions as one
// chunk and writes the output itself: one launch, the prefix read again per sequence (2
// sequences of 40 + 17 positions 5.0 us, by chunks and a join 9.7; the rule at shared_plan).
//
// The rows' places in the caches are formed once per chunk in LDS, so blocks of any length
// may end inside a tile; a position past the length or in no valid block is a row of zeros
// (so that what a page holds behind a sequence, NaN among it, never meets a product).
#include <type_traits>

#include "common.h"
#include "mkd_internal.h"
#include "coherent.h"

namespace mkd {

namespace {

constexpr int kShWaves = 4;
constexpr int kShStep = 32;                     // positions per wave step
constexpr int kShMaxChunk = 1024;               // positions per block
constexpr float kLog2e = 1.4426950408889634f;

__device__ u32x4_t g_zero_row[16];              // 256 bytes of zeros

typedef const __attribute__((address_space(1))) char* gptr;
MKD_DEV u32x4_t g_ld16(gptr p) { return *reinterpret_cast<const __attribute__((address_space(1))) u32x4_t*>(p); }
MKD_DEV uint2 g_ld8(gptr p) {
  const uint64_t v = *reinterpret_cast<const __attribute__((address_space(1))) uint64_t*>(p);
  return uint2{(uint32_t)v, (uint32_t)(v >> 32)};
}
MKD_DEV uint32_t g_ld4(gptr p) { return *reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(p); }
MKD_DEV f32x2_t cvt2_lo(uint32_t v) { return __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false); }
MKD_DEV f32x2_t cvt2_hi(uint32_t v) { return __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true); }
// eight e4m3 codes -> eight bf16 (exact)
MKD_DEV u32x4_t codes_to_bf16(uint32_t a, uint32_t b) {
  const f32x2_t x = cvt2_lo(a), y = cvt2_hi(a), z = cvt2_lo(b), w = cvt2_hi(b);
  return u32x4_t{pack2bf(x[0], x[1]), pack2bf(y[0], y[1]), pack2bf(z[0], z[1]), pack2bf(w[0], w[1])};
}
// 1 / l; a row that sees nothing (l = 0) becomes zeros, a NaN stays one
MKD_DEV float inverse(float l) { return l > 0.f ? 1.f / l : l; }
MKD_DEV float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The tile-th tile of `per` rows among the groups' rows (r1 rows a sequence), by one
// wave's scan over 64 groups at a time; false where there is none.
MKD_DEV bool find_tile(const SharedArgs& a, int tile, int per, int r1, int lane, int& g, int& first) {
  for (int g0 = 0; g0 < a.p.G; g0 += 64) {
    const int i = min(g0 + lane, a.p.G - 1);
    const int lo = min(max(a.p.prefix_starts[i], 0), a.p.B), hi = min(max(a.p.prefix_starts[i + 1], lo), a.p.B);
    int n = g0 + lane < a.p.G ? ((hi - lo) * r1 + per - 1) / per : 0, sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o, 64);
      if (lane >= o) sum += up;
    }
    const unsigned long long past = __ballot(sum > tile);
    if (past) {
      const int at = __ffsll((long long)past) - 1;
      g = g0 + at;
      first = tile - (__shfl(sum, at, 64) - __shfl(n, at, 64));
      return true;
    }
    tile -= __shfl(sum, 63, 64);
  }
  return false;
}

// The group of sequence b: the last one that starts at b or before it, -1 where that one
// has ended (by every wave for itself).
MKD_DEV int group_of(const SharedArgs& a, int b, int lane) {
  int started = 0;
  for (int g0 = 0; g0 <= a.p.G; g0 += 64) {
    const int i = g0 + lane;
    started += __popcll(__ballot(a.p.G > 0 && i <= a.p.G && a.p.prefix_starts[min(i, a.p.G)] <= b));
  }
  return started <= a.p.G ? started - 1 : -1;
}

}  // namespace

namespace {

constexpr int kShStages = 3;                    // LDS ring of the staged form

// One unit: `nrow` query rows (from row0 of the sequences from b0 on) against the
// positions [chunk0, min(chunk0 + CP, len)) of one table, as partial `slot`.
struct Unit {
  int b0, row0, nrow, len, chunk0, CP, kvh, slot, width;
  bool own;                                     // new token i sees len - (S - 1 - i) positions ..
  int first_own;                                // .. but the prefix in front of these always (whole units)
};

// Query rows of the unit as B operands: lane's row 16 t + col, head element 32 kk + 8 q4
// (FP8: q4 D/4 + 8 kk, as a lane's K bytes lie).  A negative scale goes to the queries'
// signs, so that the largest product is the largest score.
template <int D, int QT, bool FP8>
MKD_DEV void load_q(const SharedArgs& a, const Unit& u, int first, u32x4_t (&qf)[QT][D / 32], int (&lim)[QT]) {
  const int lane = threadIdx.x & 63, q4 = lane >> 4, col = lane & 15;
  const int gqa = a.p.nq / a.p.nkv, S = a.p.s_tkg, r1 = S * gqa;
  const uint16_t* qp = static_cast<const uint16_t*>(a.p.q);
  const uint32_t flip = a.p.softmax_scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = first + 16 * t + col, rr = u.row0 + min(r, u.nrow - 1);
    const int b = u.b0 + rr / r1, s = (rr / gqa) % S, h = u.kvh * gqa + rr % gqa;
    const uint16_t* src = qp + b * a.p.q_stride[0] + s * a.p.q_stride[1] + h * a.p.q_stride[2];
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const u32x4_t v = ld16(src + (FP8 ? q4 * (D / 4) + 8 * kk : 32 * kk + 8 * q4));
      qf[t][kk] = r < u.nrow ? v ^ u32x4_t{flip, flip, flip, flip} : u32x4_t{0u, 0u, 0u, 0u};
    }
    lim[t] = u.own ? max(u.len - (S - 1 - s), u.first_own) : u.len;
  }
}
// Addresses of the chunk's rows in the caches; a row of zeros for a position past the
// length or in no valid block.  The table is read before the length is known.
struct Places {
  int blk[kShMaxChunk / (64 * kShWaves)];
  int front;                                    // whole units: positions of the prefix table in front
  MKD_DEV void load(const SharedArgs& a, const int* table, int width, int chunk0, int CP) {
    front = 0;
#pragma unroll
    for (int k = 0; k < kShMaxChunk / (64 * kShWaves); ++k) {
      const int i = threadIdx.x + 64 * kShWaves * k;
      blk[k] = i < CP ? table[min((chunk0 + i) / a.p.block_len, width - 1)] : -1;
    }
  }
  MKD_DEV void load(const SharedArgs& a, const int* prefix, int plen, const int* own, int olen) {
    front = plen;
#pragma unroll
    for (int k = 0; k < kShMaxChunk / (64 * kShWaves); ++k) {
      const int i = threadIdx.x + 64 * kShWaves * k;
      blk[k] = i < plen ? prefix[i / a.p.block_len] : (i < plen + olen ? own[(i - plen) / a.p.block_len] : -1);
    }
  }
  MKD_DEV void store(const SharedArgs& a, const Unit& u, int eb, int n, uint64_t* kat, uint64_t* vat) const {
    const char* const kc = static_cast<const char*>(a.p.k_cache) + u.kvh * a.p.k_cache_stride[2] * eb;
    const char* const vc = static_cast<const char*>(a.p.v_cache) + u.kvh * a.p.v_cache_stride[2] * eb;
#pragma unroll
    for (int k = 0; k < kShMaxChunk / (64 * kShWaves); ++k) {
      const int i = threadIdx.x + 64 * kShWaves * k, t = u.chunk0 + i;
      if (i >= n) break;
      const char *ka = reinterpret_cast<const char*>(g_zero_row), *va = ka;
      if (t < u.len && (unsigned)blk[k] < (unsigned)a.p.num_blocks) {
        const int r = (t < front ? t : t - front) % a.p.block_len;
        ka = kc + (blk[k] * a.p.k_cache_stride[0] + r * a.p.k_cache_stride[1]) * eb;
        va = vc + (blk[k] * a.p.v_cache_stride[0] + r * a.p.v_cache_stride[1]) * eb;
      }
      kat[i] = reinterpret_cast<uint64_t>(ka);
      vat[i] = reinterpret_cast<uint64_t>(va);
    }
  }
};

// (a NaN wins; without the canonicalisation that fmaxf's operands get)
MKD_DEV float most(float x, float y) { return __builtin_elementwise_maximum(x, y); }
// the largest over the four lanes sharing lane % 16
MKD_DEV float quad_rows_max(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = most(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return most(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The running softmax of one wave's rows: scores of a step to probabilities, and what
// they leave of the sums so far.
template <int QT, int NDT>
struct Rows {
  f32x4_t o[QT][NDT], l[QT];                    // rows 4 q4 + i of tile t
  float m[QT];                                  // row col of tile t, in units of log2
  MKD_DEV Rows() {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = -INFINITY;
      l[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  // (kept in registers: else formed anew in front of every product)
  static MKD_DEV u32x4_t ones() {
    u32x4_t v = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    asm("" : "+v"(v));
    return v;
  }
  // After the last step: the accumulators in their registers (else the compiler brings them
  // into the order of the stores in every step, behind each product).
  MKD_DEV void settle() {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      asm("" : "+v"(l[t]));
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) asm("" : "+v"(o[t][dt]));
    }
  }
  // Raw products sc (times scale2: scores) to the tiles' P operands.  The maximum that the
  // exponentials refer to follows the largest score only where that is more than 2^8 above
  // it: the sums keep their relative precision, and the accumulators are seldom rescaled.
  // (One branch for all tiles, so that their chains of operations interleave.)
  MKD_DEV void weigh(const f32x4_t (&sc)[QT][2], float scale2, u32x4_t ones, u32x4_t (&ph)[QT]) {
    const int q4 = (threadIdx.x & 63) >> 4;
    float mx[QT];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const f32x4_t x = sc[t][0], y = sc[t][1];
      mx[t] = quad_rows_max(most(most(most(most(x[0], x[1]), x[2]), most(x[3], y[0])), most(most(y[1], y[2]), y[3]))) * scale2;
      moved = moved || mx[t] > m[t] + 8.f;
    }
    if (__any(moved)) {                         // uniform
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float mn = most(m[t], mx[t]), alpha = m[t] == -INFINITY ? 0.f : exp2_hw(m[t] - mn);
        m[t] = mn;
        float al[4];                            // (o and l rows are 4 q4 + i)
#pragma unroll
        for (int i = 0; i < 4; ++i) al[i] = __shfl(alpha, 4 * q4 + i, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) l[t][i] *= al[i];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][dt][i] *= al[i];
      }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float ms = m[t] == -INFINITY ? 0.f : -m[t];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = exp2_hw(fmaf(sc[t][u][i], scale2, ms));
        ph[t][2 * u] = pack2bf(p[0], p[1]);
        ph[t][2 * u + 1] = pack2bf(p[2], p[3]);
      }
      l[t] = mfma16x16x32(ph[t], ones, l[t]);
    }
  }
};
// positions that row `lim` does not see
MKD_DEV void hide(f32x4_t (&sc)[2], int p0, int lim) {
  const int q4 = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + 16 * u + 4 * q4 + i >= lim) sc[u][i] = -INFINITY;
}
MKD_DEV float scale_log2(const SharedArgs& a) {   // (0: small enough, and -inf stays -inf)
  return fmaxf(fabsf(a.p.softmax_scale) * kLog2e, 1e-37f);
}
MKD_DEV long long part_at(const SharedArgs& a, const Unit& u, int r) {   // the unit's row r
  const int gqa = a.p.nq / a.p.nkv, S = a.p.s_tkg, r1 = S * gqa, rr = u.row0 + r;
  return (((long long)(u.b0 + rr / r1) * S + (rr / gqa) % S) * a.p.nq + u.kvh * gqa + rr % gqa) * a.slots + u.slot;
}

// The B operand of P . V for d-tile dt, element dt of the D / 16 contiguous ones that lane
// column l % 16 holds of its 8 V rows (u, j: position 16 u + 4 (l / 16) + j).  bf16: the
// operand's halves from two rows by one byte permute per dword (selector 0x05040100: bytes
// 0-1 of each row; 0x07060302: bytes 2-3).
template <bool FP8, int VD>
MKD_DEV u32x4_t v_operand(const uint32_t (&vr)[2][4][VD], int dt) {
  u32x4_t bop;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if constexpr (FP8) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2_t v = (dt & 2) ? cvt2_hi(vr[u][j][dt >> 2]) : cvt2_lo(vr[u][j][dt >> 2]);
        x[j] = v[dt & 1];
      }
      bop[2 * u] = pack2bf(x[0], x[1]);
      bop[2 * u + 1] = pack2bf(x[2], x[3]);
    } else {
      const int e = dt >> 1;
      const uint32_t sel = (dt & 1) ? 0x07060302u : 0x05040100u;
      bop[2 * u] = __builtin_amdgcn_perm(vr[u][1][e], vr[u][0][e], sel);
      bop[2 * u + 1] = __builtin_amdgcn_perm(vr[u][3][e], vr[u][2][e], sel);
    }
  }
  return bop;
}

// ---- direct: position steps w, w + 4, .. to wave w, the waves merged at the end ----
template <int D, int QT, bool FP8, bool WHOLE>
MKD_DEV void direct_unit(const SharedArgs& a, const Unit& un, const Places& places, char* mem, float (*m_s)[32],
                         float (*l_s)[32]) {
  constexpr int EB = FP8 ? 1 : 2;               // bytes per cached element
  constexpr int NK = D / 32, NDT = D / 16, ROWS = 16 * QT;
  constexpr int KL = D * EB / 64;               // 16-byte loads of a lane's K row share
  constexpr int VD = D * EB / 64;               // dwords of a lane's V row share
  uint64_t* const kat = reinterpret_cast<uint64_t*>(mem);
  uint64_t* const vat = kat + kShMaxChunk;
  float* const o_s = reinterpret_cast<float*>(mem);
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, col = lane & 15;
  const int nst = (min(un.CP, un.len - un.chunk0) + kShStep - 1) / kShStep;
  u32x4_t qf[QT][NK];
  int lim[QT];
  load_q<D, QT, FP8>(a, un, 0, qf, lim);
  places.store(a, un, EB, nst * kShStep, kat, vat);
  const int lim_min = un.own ? un.len - (a.p.s_tkg - 1) : un.len;
  const float scale2 = scale_log2(a);
  __syncthreads();

  u32x4_t kr[2][KL];
  uint32_t vr[2][4][VD];
  auto load_k = [&](int st) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const gptr p = (gptr)kat[st * kShStep + 16 * u + col];
#pragma unroll
      for (int j = 0; j < KL; ++j) kr[u][j] = g_ld16(p + (FP8 ? q4 * (D / 4) + 16 * j : q4 * 16 + 64 * j));
    }
  };
  auto load_v = [&](int st) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const gptr p = (gptr)vat[st * kShStep + 16 * u + 4 * q4 + j] + col * (4 * VD);
        if constexpr (VD == 4) {
          const u32x4_t v = g_ld16(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[u][j][e] = v[e];
        } else if constexpr (VD == 2) {
          const uint2 v = g_ld8(p);
          vr[u][j][0] = v.x;
          vr[u][j][1] = v.y;
        } else {
          vr[u][j][0] = g_ld4(p);
        }
      }
  };
  Rows<QT, NDT> rows;
  const u32x4_t ones = rows.ones();
  int st = w;
  if (st < nst) {
    load_k(st);
    load_v(st);
  }
  for (; st < nst; st += kShWaves) {
    const int p0 = un.chunk0 + st * kShStep, sn = st + kShWaves;
    f32x4_t sc[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4_t kf[NK];
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        if constexpr (FP8) kf[kk] = codes_to_bf16(kr[u][kk / 2][(kk & 1) * 2], kr[u][kk / 2][(kk & 1) * 2 + 1]);
        else kf[kk] = kr[u][kk];
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        sc[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) sc[t][u] = mfma16x16x32(kf[kk], qf[t][kk], sc[t][u]);
      }
    }
    if (sn < nst) load_k(sn);
    u32x4_t ph[QT];
    if (p0 + kShStep > lim_min)
#pragma unroll
      for (int t = 0; t < QT; ++t) hide(sc[t], p0, lim[t]);
    rows.weigh(sc, scale2, ones, ph);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const u32x4_t bop = v_operand<FP8>(vr, dt);
#pragma unroll
      for (int t = 0; t < QT; ++t) rows.o[t][dt] = mfma16x16x32(ph[t], bop, rows.o[t][dt]);
    }
    if (sn < nst) load_v(sn);
  }
  // ---- merge the waves into this chunk's partial ----
  rows.settle();
  __syncthreads();                              // the addresses are read; o_s takes their place
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (lane < 16) m_s[w][16 * t + lane] = rows.m[t];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + 4 * q4 + i;
      if (col == 0) l_s[w][r] = rows.l[t][i];
#pragma unroll
      for (int q = 0; q < NDT / 4; ++q)
        *reinterpret_cast<f32x4_t*>(o_s + ((w * ROWS + r) * D + col * NDT + 4 * q)) =
            f32x4_t{rows.o[t][4 * q][i], rows.o[t][4 * q + 1][i], rows.o[t][4 * q + 2][i], rows.o[t][4 * q + 3][i]};
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x * 4; idx < un.nrow * D; idx += 64 * kShWaves * 4) {
    const int r = idx / D, e0 = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int q = 0; q < kShWaves; ++q) M = fmaxf(M, m_s[q][r]);
    float L = 0.f;
    f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < kShWaves; ++q) {
      const float f = m_s[q][r] == -INFINITY ? 0.f : exp2_hw(m_s[q][r] - M);
      L += l_s[q][r] * f;
      O += *reinterpret_cast<const f32x4_t*>(o_s + ((q * ROWS + r) * D + e0)) * f;
    }
    if constexpr (WHOLE) {
      const int gqa = a.p.nq / a.p.nkv, rr = un.row0 + r, h = un.kvh * gqa + rr % gqa;
      if (a.p.sink) {
        const float sk = a.p.sink[h] * kLog2e, top = most(M, sk), f = M == -INFINITY ? 0.f : exp2_hw(M - top);
        L = L * f + (sk == -INFINITY ? 0.f : exp2_hw(sk - top));
        O *= f;
      }
      const float inv = inverse(L);
      uint16_t* dst = static_cast<uint16_t*>(a.p.out) + un.b0 * a.p.out_stride[0] + rr / gqa % a.p.s_tkg * a.p.out_stride[1] +
                      h * a.p.out_stride[2] + e0;
      reinterpret_cast<uint32_t*>(dst)[0] = pack2bf(O[0] * inv, O[1] * inv);
      reinterpret_cast<uint32_t*>(dst)[1] = pack2bf(O[2] * inv, O[3] * inv);
      continue;
    }
    const long long at = part_at(a, un, r);
    *reinterpret_cast<f32x4_t*>(a.part_o + at * D + e0) = O;
    if (e0 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{M, L};
  }
}

// Wrappers outside the templates.
MKD_DEV void g_to_lds16(gptr src, char* dst) {   // lane l's 16 bytes to dst + 16 l (dst uniform)
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
template <int N>
MKD_DEV void wait_loads() {                     // all but the last N vector memory accesses
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// ---- staged: wave w holds rows 16 QT w .., every step's K and V rows through LDS ----
// A stage holds 32 K rows, then 32 V rows, in pieces of 16 bytes; the piece p of row r lies
// at p ^ turn(r): the 8 rows that a K read takes at a time lie on different banks (256
// bytes of them).
template <int CPR>
constexpr MKD_DEV int turn(int r) {
  return CPR == 16 ? r & 15 : (CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3);
}
template <int D, int QT, bool FP8>
MKD_DEV void staged_unit(const SharedArgs& a, const Unit& un, const Places& places, char* mem) {
  constexpr int EB = FP8 ? 1 : 2, NK = D / 32, NDT = D / 16;
  constexpr int RB = D * EB, CPR = RB / 16;     // bytes, pieces of a row
  constexpr int VD = RB / 64;                   // dwords of a lane's V row share
  constexpr int kStage = 2 * kShStep * RB, CPW = CPR / kShWaves;   // 1 KiB copies per wave and stage
  static_assert(CPW >= 1, "a copy per wave");
  char* const ring = mem;
  uint64_t* const kat = reinterpret_cast<uint64_t*>(mem + kShStages * kStage);
  uint64_t* const vat = kat + kShMaxChunk;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, col = lane & 15;
  const int nst = (min(un.CP, un.len - un.chunk0) + kShStep - 1) / kShStep;
  const int first = 16 * QT * w;                // this wave's rows
  u32x4_t qf[QT][NK];
  int lim[QT];
  load_q<D, QT, FP8>(a, un, first, qf, lim);
  places.store(a, un, EB, nst * kShStep, kat, vat);
  const float scale2 = scale_log2(a);
  __syncthreads();
  // (the stage read, the stage filled and the addresses never overlap: without that promise the
  // compiler waits for the copies in flight in front of every read)
  auto copy = [&](char* __restrict dst, const uint64_t* __restrict ka, const uint64_t* __restrict va) {
    uint64_t at[CPW];
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      const int n = w * CPW + i;                // (uniform) the stage's n-th KiB: K in the first half
      at[i] = n >= CPR / 2 ? va[((n - CPR / 2) * 64 + lane) / CPR] : ka[(n * 64 + lane) / CPR];
    }
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      const int n = w * CPW + i;
      const int piece = (n >= CPR / 2 ? n - CPR / 2 : n) * 64 + lane, row = piece / CPR, p = piece % CPR;
      g_to_lds16((gptr)at[i] + ((p ^ turn<CPR>(row)) << 4), dst + n * 1024);
    }
  };
#pragma unroll 1
  for (int st = 0; st < min(nst, 2); ++st) copy(ring + st * kStage, kat + st * kShStep, vat + st * kShStep);
  Rows<QT, NDT> rows;
  const bool live = first < un.nrow;            // (uniform)
  const int kx = turn<CPR>(col) << 4;
  const u32x4_t ones = rows.ones();
  auto step = [&](const char* __restrict ks, char* __restrict dst, const uint64_t* __restrict ka,
                  const uint64_t* __restrict va, int p0, bool more) {
    if (more) copy(dst, ka, va);
    if (!live) return;
    const char* const vs = ks + kShStep * RB;
    f32x4_t sc[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4_t kf[NK];
      if constexpr (FP8) {
#pragma unroll
        for (int j = 0; j < RB / 64; ++j) {
          const u32x4_t v = ld16(ks + (16 * u + col) * RB + ((((RB / 64) * q4 + j) << 4) ^ kx));
          kf[2 * j] = codes_to_bf16(v[0], v[1]);
          kf[2 * j + 1] = codes_to_bf16(v[2], v[3]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = ld16(ks + (16 * u + col) * RB + (((4 * kk + q4) << 4) ^ kx));
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        sc[t][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) sc[t][u] = mfma16x16x32(kf[kk], qf[t][kk], sc[t][u]);
      }
    }
    // the V rows, on their way through the softmax
    uint32_t vr[2][4][VD];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * u + 4 * q4 + j, byte = col * (4 * VD);
        const char* p = vs + row * RB + ((byte & ~15) ^ (turn<CPR>(row & 15) << 4)) + (byte & 15);
        typedef uint32_t __attribute__((ext_vector_type(VD == 1 ? 2 : VD))) dwords;
        if constexpr (VD == 1) {
          vr[u][j][0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
          const dwords v = *reinterpret_cast<const dwords*>(p);
#pragma unroll
          for (int e = 0; e < VD; ++e) vr[u][j][e] = v[e];
        }
      }
    u32x4_t ph[QT];
    if (p0 + kShStep > un.len)
#pragma unroll
      for (int t = 0; t < QT; ++t) hide(sc[t], p0, un.len);
    rows.weigh(sc, scale2, ones, ph);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const u32x4_t bop = v_operand<FP8>(vr, dt);
#pragma unroll
      for (int t = 0; t < QT; ++t) rows.o[t][dt] = mfma16x16x32(ph[t], bop, rows.o[t][dt]);
    }
  };
  // (three stages a turn: their places in LDS are constants)
  auto turn_of = [&](int st, auto slot) {
    constexpr int S = decltype(slot)::value;
    if (st >= nst) return;
    if (st + 1 < nst) wait_loads<CPW>();        // stage st landed: this wave's part ..
    else wait_loads<0>();
    lds_barrier();                              // .. and everyone's; stage st - 1 is read
    step(ring + S * kStage, ring + (S + 2) % kShStages * kStage, kat + (st + 2) * kShStep, vat + (st + 2) * kShStep,
         un.chunk0 + st * kShStep, st + 2 < nst);
  };
  for (int st = 0; st < nst; st += kShStages) {
    turn_of(st, std::integral_constant<int, 0>{});
    turn_of(st + 1, std::integral_constant<int, 1>{});
    turn_of(st + 2, std::integral_constant<int, 2>{});
  }
  if (!live) return;
  rows.settle();
  // ---- the wave's rows out: row 4 q4 + i of tile t, its sum from every lane column, its
  // maximum from lane column 4 q4 + i (a lane forms one row's place, the others ask it) ----
  const int n = min(un.nrow - first, 16 * QT);
  const long long place = part_at(a, un, first + min(lane % (16 * QT), n - 1));
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + 4 * q4 + i;
      const long long at = __shfl(place, r, 64);
      const float mx = __shfl(rows.m[t], 4 * q4 + i, 64);
      if (r >= n) continue;
#pragma unroll
      for (int q = 0; q < NDT / 4; ++q)
        *reinterpret_cast<f32x4_t*>(a.part_o + at * D + col * NDT + 4 * q) =
            f32x4_t{rows.o[t][4 * q][i], rows.o[t][4 * q + 1][i], rows.o[t][4 * q + 2][i], rows.o[t][4 * q + 3][i]};
      if (col == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{mx, rows.l[t][i]};
    }
}

}  // namespace

// PQ: 16-row tiles per wave of the staged prefixes, 0: prefixes direct; OQ: tiles of the
// direct units.
template <int D, bool FP8, int PQ, int OQ>
__global__ void __launch_bounds__(64 * kShWaves, 2) attn_shared_kernel(SharedArgs a) {
  constexpr int EB = FP8 ? 1 : 2, kTab = 2 * kShMaxChunk * 8;
  constexpr int kDirect = kShWaves * 16 * OQ * D * 4 > kTab ? kShWaves * 16 * OQ * D * 4 : kTab;
  constexpr int kStaged = PQ > 0 ? kShStages * 2 * kShStep * D * EB + kTab : 0;
  constexpr int kMem = kDirect > kStaged ? kDirect : kStaged;
  __shared__ __attribute__((aligned(1024))) char mem[kMem];
  __shared__ float m_s[kShWaves][32], l_s[kShWaves][32];
  const int r1 = a.p.s_tkg * (a.p.nq / a.p.nkv);
  int L = blockIdx.x;
  Unit u;
  u.first_own = 0;
  Places places;
  if (L >= a.own_units) {
    L -= a.own_units;
    // the tiles of one (chunk, kv head) on one XCD (workgroups go round-robin by index)
    constexpr int per = PQ > 0 ? kShWaves * 16 * PQ : 16 * OQ;
    const int cell = L / (8 * a.prefix_tiles) * 8 + L % 8, tile = L / 8 % a.prefix_tiles;
    const int c = cell / a.p.nkv;
    if (c >= a.prefix_chunks) return;
    int g, first;
    u.width = a.p.prefix_blocks;
    u.CP = a.prefix_chunk;
    u.chunk0 = c * u.CP;
    if (a.p.G == 1) {                           // (its table at once)
      g = 0;
      first = tile;
      places.load(a, a.p.prefix_tables, u.width, u.chunk0, u.CP);
    } else {
      if (!find_tile(a, tile, per, r1, threadIdx.x & 63, g, first)) return;
      places.load(a, a.p.prefix_tables + (long long)g * u.width, u.width, u.chunk0, u.CP);
    }
    const int lo = min(max(a.p.prefix_starts[g], 0), a.p.B), hi = min(max(a.p.prefix_starts[g + 1], lo), a.p.B);
    u.own = false;
    u.b0 = lo;
    u.row0 = first * per;
    u.nrow = min((hi - lo) * r1 - u.row0, per);
    u.len = a.p.prefix_lens[g];
    u.kvh = cell % a.p.nkv;
    u.slot = c;
  } else {
    if (L >= a.p.B * a.own_tiles * a.p.nkv * a.own_chunks) return;   // (their number is rounded up to 8)
    const int c = L % a.own_chunks, rest = L / a.own_chunks, tile = rest / a.p.nkv % a.own_tiles;
    u.own = true;
    u.kvh = rest % a.p.nkv;
    u.b0 = rest / a.p.nkv / a.own_tiles;
    u.row0 = tile * 16 * OQ;
    u.nrow = min(r1 - u.row0, 16 * OQ);
    u.width = a.p.own_blocks;
    u.CP = a.own_chunk;
    u.chunk0 = c * u.CP;
    places.load(a, a.p.tables + (long long)u.b0 * u.width, u.width, u.chunk0, u.CP);
    u.len = a.p.lens[u.b0];
    u.slot = a.prefix_chunks + c;
  }
  u.len = __builtin_amdgcn_readfirstlane(min(max(u.len, 0), u.width * a.p.block_len));
  u.b0 = __builtin_amdgcn_readfirstlane(u.b0);
  u.row0 = __builtin_amdgcn_readfirstlane(u.row0);
  u.nrow = __builtin_amdgcn_readfirstlane(u.nrow);
  if (u.chunk0 >= u.len || u.nrow <= 0) return; // whole block
  if constexpr (PQ > 0) {
    if (!u.own) {
      staged_unit<D, PQ, FP8>(a, u, places, mem);
      return;
    }
  }
  direct_unit<D, OQ, FP8, false>(a, u, places, mem, m_s, l_s);
}

// Short contexts: block (kv head, tile of a sequence's rows, sequence).
template <int D, bool FP8, int OQ>
__global__ void __launch_bounds__(64 * kShWaves, OQ == 1 ? 3 : 2) attn_shared_whole_kernel(SharedArgs a) {
  constexpr int kTab = 2 * kShMaxChunk * 8, kOut = kShWaves * 16 * OQ * D * 4;
  __shared__ __attribute__((aligned(1024))) char mem[kOut > kTab ? kOut : kTab];
  __shared__ float m_s[kShWaves][32], l_s[kShWaves][32];
  const int r1 = a.p.s_tkg * (a.p.nq / a.p.nkv);
  Unit u;
  u.own = true;
  u.kvh = blockIdx.x;
  u.row0 = blockIdx.y * 16 * OQ;
  u.b0 = blockIdx.z;
  u.nrow = min(r1 - u.row0, 16 * OQ);
  u.chunk0 = u.slot = 0;
  const int olen = min(max(a.p.lens[u.b0], 0), a.p.own_blocks * a.p.block_len);
  const int g = __builtin_amdgcn_readfirstlane(group_of(a, u.b0, threadIdx.x & 63));
  const int plen = g >= 0 ? min(max(a.p.prefix_lens[g], 0), a.p.prefix_blocks * a.p.block_len) : 0;
  Places places;
  places.load(a, a.p.prefix_tables + (long long)max(g, 0) * a.p.prefix_blocks, plen,
              a.p.tables + (long long)u.b0 * a.p.own_blocks, olen);
  u.len = __builtin_amdgcn_readfirstlane(plen + olen);
  u.CP = kShMaxChunk;
  u.first_own = plen;
  direct_unit<D, OQ, FP8, true>(a, u, places, mem, m_s, l_s);
}

// One wave per query row: its group's live prefix chunks, its own live chunks, the sink.  Bound
// by the partials' bytes (2048 rows x 17 of 520 bytes: 6.1 us, 1920 x 9: 5.1); loads that do not
// wait for the lengths made it no faster.
template <int D>
__global__ void __launch_bounds__(256) attn_shared_combine_kernel(SharedArgs a) {
  const int lane = threadIdx.x & 63;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (row >= (long long)a.p.B * a.p.s_tkg * a.p.nq) return;
  const int h = (int)(row % a.p.nq), b = (int)(row / a.p.nq / a.p.s_tkg), s = (int)(row / a.p.nq % a.p.s_tkg);
  const int g = group_of(a, b, lane);
  int np = 0;
  if (g >= 0) np = (min(max(a.p.prefix_lens[g], 0), a.p.prefix_blocks * a.p.block_len) + a.prefix_chunk - 1) / a.prefix_chunk;
  const int no = (min(max(a.p.lens[b], 0), a.p.own_blocks * a.p.block_len) + a.own_chunk - 1) / a.own_chunk;
  const int n = np + no;
  const float* ml = a.part_ml + row * a.slots * 2;
  const float* po = a.part_o + row * a.slots * D;
  auto slot_of = [&](int i) { return i < np ? i : a.prefix_chunks + i - np; };
  float M = a.p.sink ? a.p.sink[h] * kLog2e : -INFINITY;
  for (int i = lane; i < n; i += 64) M = fmaxf(M, ml[2 * slot_of(i)]);
  M = wave_max(M);
  const float ms = M == -INFINITY ? 0.f : M;
  // 16 bytes of a partial per lane: the wave takes 64 / (D / 4) partials at a time
  constexpr int LP = D / 4, PW = 64 / LP;
  const int sub = lane / LP, d = lane % LP * 4;
  float L = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = sub; i < n; i += PW) {
    const int c = slot_of(i);
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * c);
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(po + (long long)c * D + d);
    const float f = exp2_hw(x.x - ms);           // (a chunk that the row does not see: 0)
    L += x.y * f;
    o += v * f;
  }
#pragma unroll
  for (int k = LP; k < 64; k <<= 1) {
    L += __shfl_xor(L, k, 64);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], k, 64);
  }
  if (a.p.sink) L += exp2_hw(a.p.sink[h] * kLog2e - ms);
  const float inv = inverse(L);
  uint16_t* dst = static_cast<uint16_t*>(a.p.out) + b * a.p.out_stride[0] + s * a.p.out_stride[1] + h * a.p.out_stride[2];
  if (sub == 0) {
    reinterpret_cast<uint32_t*>(dst + d)[0] = pack2bf(o[0] * inv, o[1] * inv);
    reinterpret_cast<uint32_t*>(dst + d)[1] = pack2bf(o[2] * inv, o[3] * inv);
  }
}

// Shapes alone decide the split (lengths stay on the device).  Staged prefixes take 32 rows
// per wave where that leaves every CU a unit of 512 positions (64 sequences x 8 heads x 8192
// positions x 4 kv heads: 27.5 us, 16 rows per wave 30.7), else 16 (15 sequences x 4 tokens x
// 4100 positions: 22.5 and 20.0 us; 6 groups of 42 x 2000: 18.1 and 14.4), two units a CU.
// Direct to 32 rows: 8 rows x 32768 positions 21.7 us, staged 25.2; 32 rows 24.0 and 26.3
// (at 2000 positions 11.6 and 10.9).
// One launch for short contexts (us with it, and with chunks and a join; 4 kv heads of 128, 8
// heads each): a block per sequence and kv head goes through its positions alone, so long
// contexts want many blocks, and each reads the prefix anew, so many want short ones.
//   positions   4 blocks    64 blocks   128 blocks  512 blocks   1024 blocks
//   128         4.9   7.8   5.1   8.8   5.1   9.2    6.7  14.9   12.4  22.3
//   512         8.5   9.0   8.6  11.1   8.7  11.8   13.4  20.3   23.2  27.8
//   768        10.8   9.5  10.9  11.7  11.0  13.0   17.9  23.4   32.0  29.2
//   1024       13.1   8.8  13.4  11.3  13.4  12.8   22.5  24.9   40.8  30.5
SharedPlan shared_plan(const mkd_shared_prefix_args& p) {
  SharedPlan s{};
  const long long r1 = (long long)p.s_tkg * (p.nq / p.nkv), rows = r1 * p.B;
  const long long plen = p.G > 0 ? (long long)p.prefix_blocks * p.block_len : 0, olen = (long long)p.own_blocks * p.block_len;
  const bool wide = (rows + 127) / 128 * p.nkv * ((plen + 511) / 512) >= 256;
  s.prefix_qt = rows <= 32 ? 0 : (wide ? 2 : 1);
  const long long whole = (r1 + 31) / 32 * p.nkv * p.B, len = plen + olen;
  s.whole = len <= 512 ? whole <= 1024 : len <= kShMaxChunk && whole <= 512 && (len <= 768 || whole >= 128);
  s.own_qt = (rows <= 32 && !s.whole ? rows : r1) <= 16 ? 1 : 2;
  s.own_tiles = (int)((r1 + 16 * s.own_qt - 1) / (16 * s.own_qt));
  const int per = s.prefix_qt ? 16 * kShWaves * s.prefix_qt : 16 * s.own_qt;
  s.prefix_tiles = p.G > 0 ? (rows + per - 1) / per + p.G - 1 : 0;
  // positions per unit, in whole steps of all waves, for about `want` units
  auto chunk_for = [](long long len, long long units, long long want) {
    const long long n = units > 0 ? (want + units - 1) / units : 1;
    const long long c = ((len + n - 1) / n + 127) / 128 * 128;
    return (int)(c < 128 ? 128 : (c > kShMaxChunk ? kShMaxChunk : c));
  };
  s.prefix_chunk = chunk_for(plen, s.prefix_tiles * p.nkv, wide ? 256 : 512);
  s.own_chunk = chunk_for(olen, (long long)p.B * s.own_tiles * p.nkv, 256);
  s.prefix_chunks = (plen + s.prefix_chunk - 1) / s.prefix_chunk;
  s.own_chunks = (olen + s.own_chunk - 1) / s.own_chunk;
  s.prefix_units = (s.prefix_chunks * p.nkv + 7) / 8 * 8 * s.prefix_tiles;
  s.own_units = (s.own_chunks * p.nkv * s.own_tiles * p.B + 7) / 8 * 8;
  return s;
}

namespace {

template <int D, bool FP8>
void shared_run(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  if (p.whole) {
    const int gqa = a.p.nq / a.p.nkv, per = 16 * p.own_qt;
    const dim3 whole(a.p.nkv, (a.p.s_tkg * gqa + per - 1) / per, a.p.B);
    if (p.own_qt == 1) hipLaunchKernelGGL((attn_shared_whole_kernel<D, FP8, 1>), whole, dim3(64 * kShWaves), 0, s, a);
    else hipLaunchKernelGGL((attn_shared_whole_kernel<D, FP8, 2>), whole, dim3(64 * kShWaves), 0, s, a);
    return;
  }
  const dim3 grid((unsigned)(p.prefix_units + p.own_units)), block(64 * kShWaves);
  if (grid.x > 0) {
    switch (p.prefix_qt * 2 + p.own_qt) {
      case 1: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 0, 1>), grid, block, 0, s, a); break;
      case 2: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 0, 2>), grid, block, 0, s, a); break;
      case 3: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 1, 1>), grid, block, 0, s, a); break;
      case 4: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 1, 2>), grid, block, 0, s, a); break;
      case 5: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 2, 1>), grid, block, 0, s, a); break;
      default: hipLaunchKernelGGL((attn_shared_kernel<D, FP8, 2, 2>), grid, block, 0, s, a);
    }
  }
  const long long rows = (long long)a.p.B * a.p.s_tkg * a.p.nq;
  hipLaunchKernelGGL(attn_shared_combine_kernel<D>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
}

}  // namespace

hipError_t attn_shared_launch(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  const bool fp8 = a.p.kv_format & MKD_KV_FP8;
  if (a.p.d == 128) fp8 ? shared_run<128, true>(a, p, s) : shared_run<128, false>(a, p, s);
  else fp8 ? shared_run<64, true>(a, p, s) : shared_run<64, false>(a, p, s);
  return hipGetLastError();
}

}  // namespace mkd
