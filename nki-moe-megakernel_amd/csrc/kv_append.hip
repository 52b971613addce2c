// New tokens' heads into a paged KV cache, normed and rotated on the way, and the
// rotated queries beside them (mkd_kv_append_rope).
//
// Per head of D elements, in fp32: x * rsqrt(mean(x^2) + eps) * w, then for i < r / 2
//   y_i = x_i c_i - x_{i + r/2} s_i,   y_{i + r/2} = x_{i + r/2} c_i + x_i s_i
// with row positions[t] of the tables, then one rounding to bf16 or e4m3.
//
// D / 8 lanes per head.  Lane j < r / 8 holds the elements 4j .. 4j + 3 and their
// partners 4j + r/2 ..: the rotation stays inside the lane; the lanes behind hold the 8
// contiguous elements of the part that is not rotated.  The norm's sum is a DPP sum over
// the head's lanes.  Bound by its bytes for prompts (figures at append_size), by the launch at
// decode batches: one token of 32 + 2 x 4 heads of 128 3.5 us, 61 of 64 + 2 x 8 of 64 into an
// FP8 cache 3.8; a call takes 6 us with its host side.
#include "common.h"
#include "fp8.h"
#include "mkd_internal.h"

namespace mkd {

namespace {

struct Quad { float v[4]; };

template <bool F32>
MKD_DEV u32x4_t quad_ld(const void* p, long long off) {   // 4 elements: 16 bytes, or 8
  if constexpr (F32) return ld16(static_cast<const float*>(p) + off);
  const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + off);
  return u32x4_t{r.x, r.y, 0u, 0u};
}
template <bool F32>
MKD_DEV Quad quad_f(u32x4_t r) {
  if constexpr (F32)
    return Quad{{__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]), __uint_as_float(r[3])}};
  return Quad{{bf_lo(r[0]), bf_hi(r[0]), bf_lo(r[1]), bf_hi(r[1])}};
}
MKD_DEV void quad_st_bf16(uint16_t* p, const Quad& q) {
  *reinterpret_cast<uint2*>(p) = uint2{pack2bf(q.v[0], q.v[1]), pack2bf(q.v[2], q.v[3])};
}
// e4m3(clip(x * scale, +-240)), round to nearest even; a NaN stays one
MKD_DEV float kv_clip(float x, float scale) {
  const float y = x * scale;
  return y != y ? y : fminf(fmaxf(y, -kFp8Max), kFp8Max);
}
MKD_DEV void quad_st_fp8(uint8_t* p, const Quad& q, float scale) {
  int o = __builtin_amdgcn_cvt_pk_fp8_f32(kv_clip(q.v[0], scale), kv_clip(q.v[1], scale), 0, false);
  o = __builtin_amdgcn_cvt_pk_fp8_f32(kv_clip(q.v[2], scale), kv_clip(q.v[3], scale), o, true);
  *reinterpret_cast<int*>(p) = o;
}
MKD_DEV long long index_at(const void* p, int i64, int t) {
  return i64 ? static_cast<const long long*>(p)[t] : static_cast<const int*>(p)[t];
}

}  // namespace

// HPT heads of one token per lane group: they share the token's table row.
template <int D, bool F32, bool FP8, int HPT>
__global__ void __launch_bounds__(256) kv_append_kernel(mkd_kv_append_args a) {
  constexpr int LH = D / 8;                            // lanes per head
  const int j = threadIdx.x % LH;
  const int nh = a.nq + 2 * a.nkv, per = (nh + HPT - 1) / HPT;
  const unsigned item = blockIdx.x * (256u / LH) + threadIdx.x / LH;
  const bool have = item < (unsigned)a.T * (unsigned)per;
  // (every lane stays active for the DPP sums: groups without an item repeat the last)
  const unsigned it = have ? item : (unsigned)a.T * (unsigned)per - 1u;
  const int t = (int)(it / (unsigned)per), h0 = (int)(it % (unsigned)per) * HPT;
  const int rl = a.rot / 8;                            // lanes that rotate
  const int e0 = j < rl ? 4 * j : 8 * j, e1 = j < rl ? 4 * j + a.rot / 2 : 8 * j + 4;

  const long long slot = index_at(a.slots, a.slots_i64, t);
  const long long pos = a.cos ? index_at(a.positions, a.positions_i64, t) : 0;
  u32x4_t x0[HPT], x1[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = min(h0 + i, nh - 1);
    const void* src;
    long long off;
    if (h < a.nq) {
      src = a.q;
      off = t * a.q_stride[0] + h * a.q_stride[1];
    } else if (h < a.nq + a.nkv) {
      src = a.k;
      off = t * a.k_stride[0] + (h - a.nq) * a.k_stride[1];
    } else {
      src = a.v;
      off = t * a.v_stride[0] + (h - a.nq - a.nkv) * a.v_stride[1];
    }
    x0[i] = quad_ld<F32>(src, off + e0);
    x1[i] = quad_ld<F32>(src, off + e1);
  }
  const bool known = !a.cos || (pos >= 0 && pos < a.table_rows);
  Quad c{{1.f, 1.f, 1.f, 1.f}}, s{{0.f, 0.f, 0.f, 0.f}};
  if (a.cos && known && j < rl) {
    c = quad_f<true>(ld16(a.cos + pos * (a.rot / 2) + 4 * j));
    s = quad_f<true>(ld16(a.sin + pos * (a.rot / 2) + 4 * j));
  }
  const bool cached = have && known && slot >= 0 && slot < (long long)a.num_blocks * a.block_len;
  const int blk = cached ? (int)slot / a.block_len : 0, row = cached ? (int)slot % a.block_len : 0;

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = min(h0 + i, nh - 1);
    const bool mine = h0 + i < nh;
    const int kind = h < a.nq ? 0 : (h < a.nq + a.nkv ? 1 : 2);
    Quad p = quad_f<F32>(x0[i]), q = quad_f<F32>(x1[i]);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += p.v[e] * p.v[e] + q.v[e] * q.v[e];
    ss += dpp_f<0xB1>(ss);                             // the head's 8 lanes, or 16
    ss += dpp_f<0x4E>(ss);
    ss += dpp_f<0x141>(ss);
    if constexpr (D == 128) ss += dpp_f<0x140>(ss);
    const void* nw = kind == 0 ? a.q_norm : (kind == 1 ? a.k_norm : nullptr);
    if (nw) {
      const float rinv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      const Quad w0 = quad_f<false>(quad_ld<false>(nw, e0)), w1 = quad_f<false>(quad_ld<false>(nw, e1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p.v[e] = p.v[e] * rinv * w0.v[e];
        q.v[e] = q.v[e] * rinv * w1.v[e];
      }
    }
    if (kind < 2 && j < rl) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = p.v[e] * c.v[e] - q.v[e] * s.v[e];
        q.v[e] = q.v[e] * c.v[e] + p.v[e] * s.v[e];
        p.v[e] = u;
      }
    }
    if (kind == 0) {
      if (!have || !mine) continue;
      if (!known) p = q = Quad{{0.f, 0.f, 0.f, 0.f}};
      uint16_t* dst = static_cast<uint16_t*>(a.q_out) + t * a.q_out_stride[0] + h * a.q_out_stride[1];
      quad_st_bf16(dst + e0, p);
      quad_st_bf16(dst + e1, q);
    } else if (cached && mine) {
      const int g = h - a.nq - (kind == 2 ? a.nkv : 0);
      const long long* st = kind == 1 ? a.k_cache_stride : a.v_cache_stride;
      void* cache = kind == 1 ? a.k_cache : a.v_cache;
      const long long off = blk * st[0] + row * st[1] + g * st[2];
      if constexpr (FP8) {
        const float scale = kind == 1 ? a.k_scale[0] : a.v_scale[0];
        quad_st_fp8(static_cast<uint8_t*>(cache) + off + e0, p, scale);
        quad_st_fp8(static_cast<uint8_t*>(cache) + off + e1, q, scale);
      } else {
        quad_st_bf16(static_cast<uint16_t*>(cache) + off + e0, p);
        quad_st_bf16(static_cast<uint16_t*>(cache) + off + e1, q);
      }
    }
  }
}

namespace {

template <int D, bool F32, bool FP8, int HPT>
void append_run(const mkd_kv_append_args& a, hipStream_t s) {
  const long long items = (long long)a.T * ((a.nq + 2 * a.nkv + HPT - 1) / HPT);
  const unsigned blocks = (unsigned)((items + 2048 / D - 1) / (2048 / D));
  hipLaunchKernelGGL((kv_append_kernel<D, F32, FP8, HPT>), dim3(blocks), dim3(256), 0, s, a);
}
// Four heads per lane group (more loads in flight, the table row read once) for bf16 grids
// that fill the chip: 4096 tokens of 32 + 2 x 4 heads of 128 in 20.7 us instead of 23.4 (86 MB,
// 4.2 TB/s; a copy reaches 4.85), 2047 fp32 tokens of 16 + 2 x 16 heads 17.2 instead of 15.8.
template <int D, bool F32, bool FP8>
void append_size(const mkd_kv_append_args& a, hipStream_t s) {
  const long long lanes = (long long)a.T * (a.nq + 2 * a.nkv) * (D / 8);
  if constexpr (!F32) {
    if (lanes >= 1 << 20) return append_run<D, F32, FP8, 4>(a, s);
  }
  append_run<D, F32, FP8, 1>(a, s);
}
template <int D>
void append_pick(const mkd_kv_append_args& a, hipStream_t s) {
  const bool f32 = a.x_dtype == MKD_DT_F32, fp8 = a.kv_format & MKD_KV_FP8;
  if (f32) fp8 ? append_size<D, true, true>(a, s) : append_size<D, true, false>(a, s);
  else fp8 ? append_size<D, false, true>(a, s) : append_size<D, false, false>(a, s);
}

}  // namespace

hipError_t kv_append_launch(const mkd_kv_append_args& a, hipStream_t s) {
  if (a.T <= 0) return hipSuccess;
  if (a.d == 128) append_pick<128>(a, s);
  else append_pick<64>(a, s);
  return hipGetLastError();
}

}  // namespace mkd
