// Decode attention of a batch whose sequences share prefixes, on a paged KV cache
// (mkd_attention_shared_prefix).
//
// The softmax over a sequence's keys splits at any position into partials (max m, sum
// l, weighted values O) that join exactly: O = sum_c 2^(m_c - m) O_c, l alike.  So the
// prefix of a group is attended once by a matrix of ALL its query rows (sequences x new
// tokens x the kv head's query heads), each sequence's own positions by its own rows,
// and one launch joins a row's partials:
//   1. prefix: block (chunk of positions, kv head, tile of 16 QT rows of a group)
//   2. own:    block (chunk, kv head, tile of 16 QT rows of a sequence)
//   3. combine: one wave per row over its live chunks, the sink joined there
//
// In 1 and 2 wave w of 4 takes the chunk's 32-position steps w, w + 4, ..; per step
// (two 16-row tiles of the cache)
//   S = K . q^T   v_mfma_f32_16x16x32_bf16, A = 16 K rows, B = 16 query rows;
//                 D lane l holds S[position 4 (l/16) + i][row l % 16]
//   O += P . V    P straight from the S layout, V rows as they come (lane column
//                 l % 16 owns D / 16 contiguous elements; d-tile dt is element dt)
//   l += P . 1    the sum of the same rounded P, by one more MFMA
// A K or V operand is loaded and formed once for the QT row tiles.  P is rounded to
// bf16 for the matrix instruction (a relative 2^-9 of each term, the rounding of the
// output itself); scores, maxima, l and O stay fp32.
//
// The rows' addresses are formed once per chunk in LDS, so blocks of any length may end
// inside a tile; a position past the length or in no valid block reads a row of zeros
// (so that what a page holds behind a sequence, NaN among it, never meets a product).
#include "common.h"
#include "mkd_internal.h"

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

}  // namespace

template <int D, int QT, bool FP8, bool PREFIX>
__global__ void __launch_bounds__(64 * kShWaves, QT == 4 ? 1 : (QT == 2 ? 2 : 3))
attn_shared_kernel(SharedArgs a) {
  constexpr int EB = FP8 ? 1 : 2;               // bytes per cached element
  constexpr int NK = D / 32, NDT = D / 16, ROWS = 16 * QT;
  constexpr int KL = D * EB / 64;               // 16-byte loads of a lane's K row share
  constexpr int VD = D * EB / 64;               // dwords of a lane's V row share
  constexpr int kTab = 2 * kShMaxChunk * 8, kOut = kShWaves * ROWS * D * 4;
  __shared__ __attribute__((aligned(16))) char mem[kTab > kOut ? kTab : kOut];
  __shared__ float m_s[kShWaves][ROWS], l_s[kShWaves][ROWS];
  long long* const koff = reinterpret_cast<long long*>(mem);   // (until the merge)
  long long* const voff = koff + kShMaxChunk;
  float* const o_s = reinterpret_cast<float*>(mem);
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q4 = lane >> 4, col = lane & 15;
  const int gqa = a.p.nq / a.p.nkv, S = a.p.s_tkg, r1 = S * gqa;
  const int c = blockIdx.x / a.p.nkv, kvh = blockIdx.x % a.p.nkv;

  // ---- this block's rows, table and length ----
  int b0, row0, nrow, len, width;
  const int* table;
  if constexpr (PREFIX) {
    if (c >= a.prefix_chunks) return;
    int g, first;
    if (!find_tile(a, blockIdx.y, ROWS, r1, lane, g, first)) return;
    b0 = min(max(a.p.prefix_starts[g], 0), a.p.B);
    row0 = first * ROWS;
    nrow = (min(max(a.p.prefix_starts[g + 1], b0), a.p.B) - b0) * r1 - row0;
    width = a.p.prefix_blocks;
    table = a.p.prefix_tables + (long long)g * width;
    len = a.p.prefix_lens[g];
  } else {
    b0 = blockIdx.z;
    row0 = blockIdx.y * ROWS;
    nrow = r1 - row0;
    width = a.p.own_blocks;
    table = a.p.tables + (long long)b0 * width;
    len = a.p.lens[b0];
  }
  len = __builtin_amdgcn_readfirstlane(min(max(len, 0), width * a.p.block_len));
  b0 = __builtin_amdgcn_readfirstlane(b0);
  row0 = __builtin_amdgcn_readfirstlane(row0);
  nrow = __builtin_amdgcn_readfirstlane(min(nrow, ROWS));
  const int CP = PREFIX ? a.prefix_chunk : a.own_chunk, chunk0 = c * CP;
  if (chunk0 >= len) return;                    // whole block
  const int nst = (min(CP, len - chunk0) + kShStep - 1) / kShStep;

  // ---- byte offsets of the chunk's rows, -1: a row of zeros ----
  for (int i = threadIdx.x; i < nst * kShStep; i += 64 * kShWaves) {
    const int t = chunk0 + i;
    long long k = -1, v = -1;
    if (t < len) {
      const int blk = table[t / a.p.block_len], r = t % a.p.block_len;
      if ((unsigned)blk < (unsigned)a.p.num_blocks) {
        k = (blk * a.p.k_cache_stride[0] + r * a.p.k_cache_stride[1] + kvh * a.p.k_cache_stride[2]) * EB;
        v = (blk * a.p.v_cache_stride[0] + r * a.p.v_cache_stride[1] + kvh * a.p.v_cache_stride[2]) * EB;
      }
    }
    koff[i] = k;
    voff[i] = v;
  }

  // ---- the tile's queries: B operands, head element 32 kk + 8 q4 (FP8: q4 D/4 + 8 kk) ----
  u32x4_t qf[QT][NK];
  int lim[QT];                                  // positions that row 16 t + col sees
  const uint16_t* qp = static_cast<const uint16_t*>(a.p.q);
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = 16 * t + col, rr = row0 + min(r, nrow - 1);
    const int b = b0 + rr / r1, s = (rr / gqa) % S, h = kvh * gqa + rr % gqa;
    const uint16_t* src = qp + b * a.p.q_stride[0] + s * a.p.q_stride[1] + h * a.p.q_stride[2];
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const u32x4_t v = ld16(src + (FP8 ? q4 * (D / 4) + 8 * kk : 32 * kk + 8 * q4));
      qf[t][kk] = r < nrow ? v : u32x4_t{0u, 0u, 0u, 0u};
    }
    lim[t] = PREFIX ? len : len - (S - 1 - s);
  }
  const int lim_min = PREFIX ? len : len - (S - 1);
  const float scale2 = a.p.softmax_scale * kLog2e;
  __syncthreads();

  const char* const kc = static_cast<const char*>(a.p.k_cache);
  const char* const vc = static_cast<const char*>(a.p.v_cache);
  u32x4_t kr[2][KL];
  uint32_t vr[2][4][VD];
  auto load_k = [&](int st) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const long long off = koff[st * kShStep + 16 * u + col];
      const gptr p = (gptr)(off < 0 ? reinterpret_cast<const char*>(g_zero_row) : kc + off);
#pragma unroll
      for (int j = 0; j < KL; ++j) kr[u][j] = g_ld16(p + (FP8 ? q4 * (D / 4) + 16 * j : q4 * 16 + 64 * j));
    }
  };
  auto load_v = [&](int st) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long off = voff[st * kShStep + 16 * u + 4 * q4 + j];
        const gptr p = (gptr)(off < 0 ? reinterpret_cast<const char*>(g_zero_row) : vc + off) + col * (4 * VD);
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

  f32x4_t o[QT][NDT], l[QT];
  float m[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -INFINITY;
    l[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[t][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const u32x4_t ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};

  int st = w;
  if (st < nst) {
    load_k(st);
    load_v(st);
  }
  for (; st < nst; st += kShWaves) {
    const int p0 = chunk0 + st * kShStep, sn = st + kShWaves;
    // ---- scores, in units of log2 ----
    float sc[QT][2][4];
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
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) acc = mfma16x16x32(kf[kk], qf[t][kk], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][u][i] = acc[i] * scale2;
      }
    }
    if (sn < nst) load_k(sn);
    if (p0 + kShStep > lim_min) {               // (uniform) positions some row does not see
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (p0 + 16 * u + 4 * q4 + i >= lim[t]) sc[t][u][i] = -INFINITY;
    }
    // ---- online softmax per row (the four lanes sharing col) ----
    u32x4_t ph[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float mx = sc[t][0][0];
#pragma unroll
      for (int k = 1; k < 8; ++k) mx = fmaxf(mx, sc[t][k >> 2][k & 3]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m[t], mx);
      if (__any(mn > m[t])) {                   // uniform: a maximum moved
        const float alpha = m[t] == -INFINITY ? 0.f : exp2_hw(m[t] - mn);
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
      const float ms = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = exp2_hw(sc[t][u][i] - ms);
        ph[t][2 * u] = pack2bf(p[0], p[1]);
        ph[t][2 * u + 1] = pack2bf(p[2], p[3]);
      }
      l[t] = mfma16x16x32(ph[t], ones, l[t]);
    }
    // ---- P . V: the operand's 16-bit halves from two V rows by one byte permute per
    // dword (selector 0x05040100: bytes 0-1 of each row; 0x07060302: bytes 2-3) ----
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
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
#pragma unroll
      for (int t = 0; t < QT; ++t) o[t][dt] = mfma16x16x32(ph[t], bop, o[t][dt]);
    }
    if (sn < nst) load_v(sn);
  }

  // ---- merge the waves into this chunk's partial ----
  __syncthreads();                              // the offsets are read; o_s takes their place
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (lane < 16) m_s[w][16 * t + lane] = m[t];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + 4 * q4 + i;
      if (col == 0) l_s[w][r] = l[t][i];
#pragma unroll
      for (int q = 0; q < NDT / 4; ++q)
        *reinterpret_cast<f32x4_t*>(o_s + ((w * ROWS + r) * D + col * NDT + 4 * q)) =
            f32x4_t{o[t][4 * q][i], o[t][4 * q + 1][i], o[t][4 * q + 2][i], o[t][4 * q + 3][i]};
    }
  }
  __syncthreads();
  const int slot = PREFIX ? c : a.prefix_chunks + c;
  for (int idx = threadIdx.x * 4; idx < nrow * D; idx += 64 * kShWaves * 4) {
    const int r = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int q = 0; q < kShWaves; ++q) M = fmaxf(M, m_s[q][r]);
    float L = 0.f;
    f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < kShWaves; ++q) {
      const float f = m_s[q][r] == -INFINITY ? 0.f : exp2_hw(m_s[q][r] - M);
      L += l_s[q][r] * f;
      O += *reinterpret_cast<const f32x4_t*>(o_s + ((q * ROWS + r) * D + d)) * f;
    }
    const int rr = row0 + r;
    const long long row = ((long long)(b0 + rr / r1) * S + (rr / gqa) % S) * a.p.nq + kvh * gqa + rr % gqa;
    const long long at = row * a.slots + slot;
    *reinterpret_cast<f32x4_t*>(a.part_o + at * D + d) = O;
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = float2{M, L};
  }
}

// One wave per query row: its group's live prefix chunks, its own live chunks, the sink.
template <int D>
__global__ void __launch_bounds__(256) attn_shared_combine_kernel(SharedArgs a) {
  const int lane = threadIdx.x & 63;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 6);
  if (row >= (long long)a.p.B * a.p.s_tkg * a.p.nq) return;
  const int h = (int)(row % a.p.nq), b = (int)(row / a.p.nq / a.p.s_tkg), s = (int)(row / a.p.nq % a.p.s_tkg);
  // the group: the last one that starts at b or before
  int started = 0;
  for (int g0 = 0; g0 <= a.p.G; g0 += 64) {
    const int i = g0 + lane;
    started += __popcll(__ballot(a.p.G > 0 && i <= a.p.G && a.p.prefix_starts[min(i, a.p.G)] <= b));
  }
  int np = 0;
  if (started > 0 && started <= a.p.G)
    np = (min(max(a.p.prefix_lens[started - 1], 0), a.p.prefix_blocks * a.p.block_len) + a.prefix_chunk - 1) / a.prefix_chunk;
  const int no = (min(max(a.p.lens[b], 0), a.p.own_blocks * a.p.block_len) + a.own_chunk - 1) / a.own_chunk;
  const int n = np + no;
  const float* ml = a.part_ml + row * a.slots * 2;
  const float* po = a.part_o + row * a.slots * D;
  auto slot_of = [&](int i) { return i < np ? i : a.prefix_chunks + i - np; };
  float M = a.p.sink ? a.p.sink[h] * kLog2e : -INFINITY;
  for (int i = lane; i < n; i += 64) M = fmaxf(M, ml[2 * slot_of(i)]);
  M = wave_max(M);
  const float ms = M == -INFINITY ? 0.f : M;
  float L = a.p.sink ? exp2_hw(a.p.sink[h] * kLog2e - ms) : 0.f;
  float o[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const int c = slot_of(i);
    const float f = exp2_hw(ml[2 * c] - ms);     // (a chunk that the row does not see: 0)
    L += ml[2 * c + 1] * f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] += po[(long long)c * D + lane * (D / 64) + e] * f;
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  uint16_t* dst = static_cast<uint16_t*>(a.p.out) + b * a.p.out_stride[0] + s * a.p.out_stride[1] + h * a.p.out_stride[2];
  if constexpr (D == 128) *reinterpret_cast<uint32_t*>(dst + 2 * lane) = pack2bf(o[0] * inv, o[1] * inv);
  else dst[lane] = (uint16_t)f2bf(o[0] * inv);
}

// Shapes alone decide the split (lengths stay on the device): see SharedPlan.
SharedPlan shared_plan(const mkd_shared_prefix_args& p) {
  SharedPlan s{};
  const long long r1 = (long long)p.s_tkg * (p.nq / p.nkv), rows = r1 * p.B;
  const long long plen = p.G > 0 ? (long long)p.prefix_blocks * p.block_len : 0, olen = (long long)p.own_blocks * p.block_len;
  s.prefix_qt = rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
  s.own_qt = r1 <= 16 ? 1 : (r1 <= 32 ? 2 : 4);
  s.own_tiles = (int)((r1 + 16 * s.own_qt - 1) / (16 * s.own_qt));
  const int per = 16 * s.prefix_qt;
  s.prefix_tiles = p.G > 0 ? (rows + per - 1) / per + p.G - 1 : 0;
  auto chunk_for = [](long long len, long long units, long long want) {   // positions per block
    long long n = units > 0 ? (want + units - 1) / units : 1;              // chunks wanted
    long long c = (len + n - 1) / n;
    c = (c + 127) / 128 * 128;
    return (int)(c < 128 ? 128 : (c > kShMaxChunk ? kShMaxChunk : c));
  };
  s.prefix_chunk = chunk_for(plen, s.prefix_tiles * p.nkv, s.prefix_qt == 4 ? 256 : 768);
  s.own_chunk = chunk_for(olen, (long long)p.B * s.own_tiles * p.nkv, 1024);
  s.prefix_chunks = (plen + s.prefix_chunk - 1) / s.prefix_chunk;
  s.own_chunks = (olen + s.own_chunk - 1) / s.own_chunk;
  return s;
}

namespace {

template <int D, bool FP8, bool PREFIX>
void shared_rows(const SharedArgs& a, int qt, dim3 grid, hipStream_t s) {
  switch (qt) {
    case 1: hipLaunchKernelGGL((attn_shared_kernel<D, 1, FP8, PREFIX>), grid, dim3(64 * kShWaves), 0, s, a); break;
    case 2: hipLaunchKernelGGL((attn_shared_kernel<D, 2, FP8, PREFIX>), grid, dim3(64 * kShWaves), 0, s, a); break;
    default: hipLaunchKernelGGL((attn_shared_kernel<D, 4, FP8, PREFIX>), grid, dim3(64 * kShWaves), 0, s, a);
  }
}
template <int D, bool FP8>
void shared_run(const SharedArgs& a, const SharedPlan& p, hipStream_t s) {
  // (units of one chunk and kv head on one XCD: x, a multiple of 8, runs fastest)
  if (p.prefix_tiles > 0 && p.prefix_chunks > 0)
    shared_rows<D, FP8, true>(a, p.prefix_qt, dim3((unsigned)((p.prefix_chunks * a.p.nkv + 7) / 8 * 8), (unsigned)p.prefix_tiles), s);
  if (p.own_chunks > 0)
    shared_rows<D, FP8, false>(a, p.own_qt, dim3((unsigned)(p.own_chunks * a.p.nkv), p.own_tiles, a.p.B), s);
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
