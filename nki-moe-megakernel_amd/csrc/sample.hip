// One token per row of logits from a given random number, under temperature, top-k,
// top-p and min-p (mkd_sample_tokens), without sorting the vocabulary.
//
// With the tokens in falling order of logit, every filter keeps a front part and the
// random number asks for the first token whose cumulative mass passes a target: each is
// a weighted selection, "the first token at which a count or a mass reaches T".
//   1. chunks: block (8192 logits, row): the tokens counted and weighed in 512 bins of
//      1/16 of logit / temperature, at fixed places of that scale (so the chunks' bins
//      line up whatever their maxima), and listed by bin.
//   2. rows: one block adds the chunks' bins, scans them, and finds each filter's end and
//      then the token.  Where the tokens that can stay are few (512 at most: the usual
//      top-k, a peaked top-p), they are sorted once and every question is a lookup.
//      Otherwise the bin is found by its cumulative count or mass, and the token in the
//      bin by histograms over its members' bit patterns until a wave can sort the rest.
// Tokens 512 bins (32, e^-32) below the maximum get no mass: together at most 2^-26 of
// the row's for 2^20 of them.
//
// The answer is a whole number, and a sum off in its last places would change it where a
// border lies near.  A token's weight is therefore exp(z - middle of its bin), z = logit /
// temperature in fp64, as an integer of 36 bits (the bin's unit, exp(middle - z_max), joins
// in fp64 per bin): sums of a bin are exact, whatever the order of atomic additions, and
// its relative precision does not depend on how far below the maximum it lies.
//
// What it takes: chunks 6.1 us for one fp32 row of 151,936 logits, 19.7 for 64 (39 MB), 36.4
// for 128 bf16 rows of 201,088 (51 MB read, 64 written: 3.2 TB/s).  A block is a chain of
// loads, maximum, atomics, scan and stores, four of them on a CU; without the series 6 us
// less of the 36, without the lists 4, without the atomics 3; blocks of 16384 logits 40 us.
// rows 10.6 us for one row and 16 for 64, a chain of memory latencies and barriers; 38 for
// the 128 rows, whose two searches gather the logits of some 3000 members of a bin each (a
// memory line a logit: as much as all logits).  Both bins gathered together 37 to 42, the row
// read again in place of the lists 66.
#include "common.h"
#include "mkd_internal.h"

namespace mkd {

namespace {

typedef unsigned long long u64;
constexpr int kSmChunk = 8192, kSmThreads = 512, kSmPer = kSmChunk / kSmThreads;
constexpr int kSmBins = 512;
constexpr double kSmRes = 16.0;                 // bins per unit of z
constexpr int kSmMaxChunks = (1 << 20) / kSmChunk;
constexpr int kSmRow = 512;                     // threads of a row's block: a bin each
constexpr int kSmStage = 8192;                  // members of a bin held in LDS
constexpr int kSmRankBit = 18;                  // of the upper word
constexpr int kSmMassBits = 32 + kSmRankBit;    // a chunk's bin: count above, mass (8192 weights) below
constexpr double kSmOne = 0x1p36;               // weight of the middle of a bin; at its edges 3 % off

// What stage 1 leaves per (row, chunk).
struct SmRecord {
  u64 bins[kSmBins];                            // count << kSmMassBits | mass
  uint16_t list[kSmChunk];                      // positions in the chunk, by bin
  uint16_t start[kSmBins + 8];                  // of bin j in `list`; [kSmBins]: their number
  float top;                                    // the chunk's largest logit
  int pad[3];
};

struct SmSetting {
  double t, inv_t, top_p, min_p, u;
  int top_k;
};
MKD_DEV SmSetting setting_of(const mkd_sample_args& a, int b) {
  SmSetting s;
  const float t = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const bool greedy = !(t > 0.f);               // as top_k = 1
  s.t = greedy ? 1.0 : fmin((double)t, 0x1p127);   // (an infinite t: all the same, but never 0 * -inf)
  s.inv_t = 1.0 / s.t;
  s.top_k = greedy ? 1 : (a.top_k_rows ? a.top_k_rows[b] : a.top_k);
  s.top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  s.min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  s.u = a.uniforms[b];
  if (!(s.u > 0.0)) s.u = 0.0;
  if (s.u >= 1.0) s.u = 1.0 - 0x1p-24;
  return s;
}
// exp((l - top) * inv_t), 1 for l = top whatever it is, 0 below an infinite top
MKD_DEV double mass_of(float l, float top, double inv_t) {
  if (l == top) return 1.0;
  if (top == INFINITY) return 0.0;
  return exp(((double)l - (double)top) * inv_t);
}
// z in bins: the nearest whole number is the bin's place (monotone in l), the rest the
// token's fraction f of a bin, -1/2 to 1/2.  Adding kSmWhole rounds the exact product.
constexpr double kSmWhole = 0x1.8p52;
struct SmPlace { double place, f; };
MKD_DEV SmPlace place_of(float l, double inv_t) {
  const double c = inv_t * kSmRes, x = l, z = x * c;
  if (fabs(z) < 0x1p51) {
    const double place = fma(x, c, kSmWhole) - kSmWhole;
    return {place, fma(x, c, -place)};
  }
  return {rint(z), z - rint(z)};                // (-inf: a NaN fraction, used by none)
}
// A token's weight from its fraction: exp(f / 16), whose series to the fifth power leaves
// 2^-39; + 2^52 rounds to a whole number.
constexpr double sm_term(int k) {
  double term = kSmOne;
  for (int m = 1; m <= k; ++m) term /= kSmRes * m;
  return term;
}
struct SmSeries {                               // the coefficients, in scalar registers
  double c[6];
  MKD_DEV SmSeries() {
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      c[k] = sm_term(k) + (k == 0 ? 0x1p52 : 0.0);
      asm("" : "+s"(c[k]));                     // (else every use moves two literals first)
    }
  }
  MKD_DEV u64 bits(double f) const {            // of 2^52 + the weight
    double p = c[5];
#pragma unroll
    for (int k = 4; k >= 0; --k) p = fma(p, f, c[k]);
    return __double_as_longlong(p);
  }
  MKD_DEV u64 weight(double f) const { return bits(f) & ((1ull << 52) - 1); }
  MKD_DEV u64 counted(double f) const {         // count << kSmMassBits | weight, by one 32-bit addition
    const u64 b = bits(f);
    return (u64)((uint32_t)(b >> 32) + ((1u << (kSmMassBits - 32)) - 0x43300000u)) << 32 | (uint32_t)b;
  }
};
// bit patterns in the order of the logits (a bf16 one's upper half); -0 and +0 are one value
template <bool BF>
MKD_DEV uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return (u & 0x80000000u ? ~u : u | 0x80000000u) >> (BF ? 16 : 0);
}
template <bool BF>
MKD_DEV float logit_of(uint32_t k) {
  if constexpr (BF) return __uint_as_float((k & 0x8000u ? k & 0x7fffu : ~k) << 16);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// a token in the falling order, as one number that rises: ~key above, index below
MKD_DEV u64 token_of(uint32_t key, uint32_t index) { return (u64)~key << 32 | index; }
MKD_DEV uint32_t key_in(u64 token) { return ~(uint32_t)(token >> 32); }

template <bool BF>
MKD_DEV float logit_at(const mkd_sample_args& a, long long row, int i) {
  const long long off = row * a.row_stride + i;
  const float l = BF ? bf2f(static_cast<const uint16_t*>(a.logits)[off]) : static_cast<const float*>(a.logits)[off];
  return l == l ? l : -INFINITY;
}

}  // namespace

// VEC: rows on 16-byte boundaries.  Element i of thread x is 4 x + 2048 (i / 4) + i % 4
// (bf16: 8 x + 4096 (i / 8) + i % 8).
template <bool BF, bool VEC>
__global__ void __launch_bounds__(kSmThreads) sample_chunk_kernel(mkd_sample_args a, SmRecord* rec) {
  __shared__ u64 bins[kSmBins + 32];            // (32 behind, for what lies outside: no branches)
  __shared__ unsigned first[kSmBins];
  __shared__ __attribute__((aligned(16))) uint16_t list[kSmChunk];
  __shared__ float wtop[kSmThreads / 64];
  __shared__ unsigned wsum[kSmThreads / 64];
  const int x = threadIdx.x, lane = x & 63, w = x >> 6;
  const int b = blockIdx.y, base = blockIdx.x * kSmChunk, n = min(kSmChunk, a.V - base);
  SmRecord& r = rec[(long long)b * gridDim.x + blockIdx.x];
  for (int i = x; i < kSmBins; i += kSmThreads) bins[i] = 0;
  const SmSetting s = setting_of(a, b);
  constexpr int G = BF ? 8 : 4;                 // elements of a 16-byte piece
  float l[kSmPer];
#pragma unroll
  for (int q = 0; q < kSmPer / G; ++q) {
    const int e0 = G * x + G * kSmThreads * q;
    if (VEC && e0 + G <= n) {
      const u32x4_t v = ld16(static_cast<const char*>(a.logits) + (b * a.row_stride + base + e0) * (BF ? 2 : 4));
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float f = BF ? ((e & 1) ? bf_hi(v[e / 2]) : bf_lo(v[e / 2])) : __uint_as_float(v[e & 3]);
        l[G * q + e] = fmaxf(f, -INFINITY);     // (a NaN: -inf)
      }
    } else {
#pragma unroll
      for (int e = 0; e < G; ++e) l[G * q + e] = e0 + e < n ? logit_at<BF>(a, b, base + e0 + e) : -INFINITY;
    }
  }
  float top = l[0];
#pragma unroll
  for (int i = 1; i < kSmPer; ++i) top = fmaxf(top, l[i]);
  top = wave_max(top);
  if (lane == 0) wtop[w] = top;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kSmThreads / 64; ++q) top = fmaxf(top, wtop[q]);
  if (x == 0) r.top = top;
  if (top == -INFINITY) return;                 // nothing to choose here (the rest is not read)
  const double top_place = place_of(top, s.inv_t).place;
  uint32_t at[kSmPer];                          // rank among the bin's members << kSmRankBit | bin
  const uint32_t outside = kSmBins + (x & 31);
  // Places of 30 bits, and what lies over 900 bins below the maximum raised to there: the
  // distance is then a difference of the low words.
  const float floor_l = (float)((top_place - 1024.0) * (s.t / kSmRes));
  const SmSeries series;
  auto put = [&](uint32_t bin, u64 one) {
    return ((uint32_t)(atomicAdd(&bins[bin], one) >> 32) & ~((1u << kSmRankBit) - 1)) | bin;
  };
  if (top < INFINITY && fabs(top_place) < 0x1p30 && floor_l > -3.402823466e38f) {
    const double c = s.inv_t * kSmRes;
    const uint32_t top_low = (uint32_t)__double_as_longlong(top_place + kSmWhole);
#pragma unroll
    for (int i = 0; i < kSmPer; ++i) {
      const double v = fmaxf(l[i], floor_l), t = fma(v, c, kSmWhole);
      at[i] = put(min(top_low - (uint32_t)__double_as_longlong(t), outside), series.counted(fma(v, c, -(t - kSmWhole))));
    }
  } else if (top < INFINITY) {
    for (int i = 0; i < kSmPer; ++i) {
      const SmPlace z = place_of(l[i], s.inv_t);
      const double below = top_place - z.place; // (-inf: infinitely far)
      at[i] = below < kSmBins ? put((uint32_t)below, series.counted(z.f)) : outside;
    }
  } else {                                      // infinite logits share the mass
    for (int i = 0; i < kSmPer; ++i) at[i] = l[i] == top ? put(0u, (1ull << kSmMassBits) | (u64)kSmOne) : outside;
  }
  __syncthreads();
  // exclusive scan of the counts, a bin a thread
  static_assert(kSmBins == kSmThreads, "one bin a thread");
  const u64 mine = bins[x];
  const unsigned cnt = (unsigned)(mine >> kSmMassBits);
  unsigned sum = cnt;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(sum, o, 64);
    if (lane >= o) sum += up;
  }
  if (lane == 63) wsum[w] = sum;
  __syncthreads();
  unsigned before = sum - cnt, total = 0;
#pragma unroll
  for (int q = 0; q < kSmThreads / 64; ++q) {
    if (q < w) before += wsum[q];
    total += wsum[q];
  }
  first[x] = before;
  r.start[x] = (uint16_t)before;
  if (x == 0) r.start[kSmBins] = (uint16_t)total;
  r.bins[x] = mine;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSmPer; ++i) {
    const uint32_t j = at[i] & ((1u << kSmRankBit) - 1);
    if (j < kSmBins) list[first[j] + (at[i] >> kSmRankBit)] = (uint16_t)(G * x + G * kSmThreads * (i / G) + i % G);
  }
  __syncthreads();
  for (unsigned i = x * 8; i < total; i += kSmThreads * 8) st16(r.list + i, ld16(list + i));
}

namespace {

struct SmShared {
  double cum[kSmBins];                          // mass up to bin j, itself included, of the maximum's
  double unit[kSmBins];                         // mass of weight 1 in bin j
  u64 bins[kSmBins];                            // weight in bin j
  u64 sub[kSmRow];                              // sub-bins' weights; the sort's exchange; sorted tokens' masses
  u64 token[64], found_t;                       // a few tokens, and one
  u64 wave_m[kSmRow / 64];
  double wave_d[kSmRow / 64];
  u64 found_m;
  unsigned cum_n[kSmBins];
  unsigned sub_n[kSmRow], wave_n[kSmRow / 64];
  int shift[kSmMaxChunks];                      // chunk's first bin in the row's
  unsigned first[kSmMaxChunks + 1];             // the staged members before chunk c
  unsigned at[kSmMaxChunks];                    // where they start in the chunk's list
  uint32_t key[kSmStage], index[kSmStage];
  unsigned hits[kSmMaxChunks], bits[kSmChunk / 32];
  unsigned found_n;
  int found;
  uint32_t wave_lo[kSmRow / 64], wave_hi[kSmRow / 64];
};

static_assert(kSmRow == kSmBins && kSmChunk / 32 <= kSmRow && kSmMaxChunks <= kSmRow, "one of each per thread");

// Inclusive scans over the block's threads.
MKD_DEV void scan_n(SmShared& s, unsigned& v) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  if (lane == 63) s.wave_n[w] = v;
  __syncthreads();
  for (int q = 0; q < w; ++q) v += s.wave_n[q];
  __syncthreads();
}
template <typename T>
MKD_DEV void scan_nm(SmShared& s, T* wave, unsigned& n, T& m) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned un = __shfl_up(n, o, 64);
    const T um = __shfl_up(m, o, 64);
    if (lane >= o) {
      n += un;
      m += um;
    }
  }
  if (lane == 63) {
    s.wave_n[w] = n;
    wave[w] = m;
  }
  __syncthreads();
  T front = 0;
  for (int q = 0; q < w; ++q) {
    n += s.wave_n[q];
    front += wave[q];
  }
  m += front;
  __syncthreads();
}
// How many threads say so.
MKD_DEV unsigned count_of(SmShared& s, bool yes) {
  const unsigned c = (unsigned)__popcll(__ballot(yes));
  if ((threadIdx.x & 63) == 0) s.wave_n[threadIdx.x >> 6] = c;
  __syncthreads();
  unsigned v = 0;
#pragma unroll
  for (int q = 0; q < kSmRow / 64; ++q) v += s.wave_n[q];
  __syncthreads();
  return v;
}
// Up to 64 distinct numbers in rising order, one a lane (the others hold ~0), by one wave:
// each lane's rank is the count of smaller ones.
MKD_DEV u64 sort_wave(u64* buf, u64 v, unsigned n) {
  const int lane = threadIdx.x & 63;
  unsigned rank = 0;
  for (unsigned i = 0; i < n; ++i) {
    const u64 o = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
                  (uint32_t)__builtin_amdgcn_readlane((int)v, i);
    rank += o < v;
  }
  if (lane < (int)n) buf[rank] = v;
  wave_lds_sync();
  return lane < (int)n ? buf[lane] : ~0ull;
}
// Rising bitonic sort of one number per thread among the first `n` threads (the others
// hold ~0): strides inside a wave by shuffles, longer ones through LDS.
MKD_DEV u64 sort_up(SmShared& s, u64 v, unsigned n) {
  const unsigned x = threadIdx.x;
  if (n <= 64) return x < 64 ? sort_wave(s.token, v, n) : v;
  for (unsigned size = 2; size / 2 < n; size <<= 1)
    for (unsigned stride = size >> 1; stride > 0; stride >>= 1) {
      u64 o;
      if (stride < 64) {
        o = __shfl_xor(v, (int)stride, 64);
      } else {
        s.sub[x] = v;
        __syncthreads();
        o = s.sub[x ^ stride];
        __syncthreads();
      }
      const bool keep_low = ((x & stride) == 0) == ((x & size) == 0);
      v = (v < o) == keep_low ? v : o;
    }
  return v;
}

struct SmEnd {
  u64 token;                                    // the last one kept (or a number behind it)
  double mass;                                  // of everything up to it
};

template <bool BF>
struct SmRow {
  const mkd_sample_args& a;
  SmShared& s;
  const SmRecord* rec;                          // the row's records
  int b, nc;
  float top;
  double inv_t;
  SmSeries series{};
  int staged = -1;
  unsigned n = 0;                               // members of the staged bin
  uint32_t kmin = 0, kmax = 0;                  // their least and largest bit patterns

  MKD_DEV u64 weight(uint32_t key) const {
    if (top == INFINITY) return (u64)kSmOne;
    return series.weight(place_of(logit_of<BF>(key), inv_t).f);
  }
  // member m of the staged bin: its index, and its logit's bit pattern
  MKD_DEV void member(unsigned m, uint32_t& key, uint32_t& index) const {
    if (n <= kSmStage) {
      key = s.key[m];
      index = s.index[m];
    } else {
      uint32_t k[1], i[1];
      fetch<1>(m, k, i);
      key = k[0];
      index = i[0];
    }
  }
  // members m, m + kSmRow, .. (N of them; those behind the last repeat it): their chunks by
  // bisection (first[lo] <= m), the loads of all in flight together
  template <int N>
  MKD_DEV void fetch(unsigned m, uint32_t (&key)[N], uint32_t (&index)[N]) const {
    unsigned at[N];
    int lo[N];
    const unsigned end = s.first[nc] - 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      at[i] = min(m + i * kSmRow, end);
      lo[i] = 0;
    }
#pragma unroll
    for (int step = kSmMaxChunks / 2; step > 0; step >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int to = lo[i] + step;
        if (to < nc && s.first[to] <= at[i]) lo[i] = to;
      }
#pragma unroll
    for (int i = 0; i < N; ++i) index[i] = rec[lo[i]].list[s.at[lo[i]] + at[i] - s.first[lo[i]]];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      index[i] += lo[i] * kSmChunk;
      key[i] = key_of<BF>(logit_at<BF>(a, b, index[i]));
    }
  }
  // the members of bins [from, bin]: their number in each chunk, and where they are listed
  MKD_DEV unsigned locate(int from, int bin) {
    __syncthreads();
    const int c = threadIdx.x;
    unsigned cnt = 0, at = 0;
    if (c < nc && s.shift[c] <= bin) {          // (a chunk without tokens lies behind every bin)
      at = rec[c].start[max(from - s.shift[c], 0)];
      cnt = rec[c].start[bin - s.shift[c] + 1] - at;
    }
    unsigned v = cnt;
    scan_n(s, v);
    if (c < nc) {
      s.first[c] = v - cnt;
      s.at[c] = at;
      if (c == nc - 1) s.first[nc] = v;
    }
    __syncthreads();
    return s.first[nc];
  }
  // this thread's members, N in flight, into LDS where they fit; their range in kmin, kmax
  template <int N>
  MKD_DEV void load() {
    for (unsigned m = threadIdx.x; m < n; m += N * kSmRow) {
      uint32_t key[N], index[N];
      fetch<N>(m, key, index);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (n <= kSmStage && m + i * kSmRow < n) {
          s.key[m + i * kSmRow] = key[i];
          s.index[m + i * kSmRow] = index[i];
        }
        kmin = min(kmin, key[i]);
        kmax = max(kmax, key[i]);
      }
    }
  }
  MKD_DEV void stage(int bin) {
    if (staged == bin) return;
    staged = bin;
    n = locate(bin, bin);
    kmin = 0xffffffffu;
    kmax = 0u;
    if (n <= kSmRow) load<1>();
    else load<8>();
    uint32_t lo = kmin, hi = kmax;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
    }
    if ((threadIdx.x & 63) == 0) {
      s.wave_lo[threadIdx.x >> 6] = lo;
      s.wave_hi[threadIdx.x >> 6] = hi;
    }
    __syncthreads();
    kmin = 0xffffffffu;
    kmax = 0u;
#pragma unroll
    for (int q = 0; q < kSmRow / 64; ++q) {
      kmin = min(kmin, s.wave_lo[q]);
      kmax = max(kmax, s.wave_hi[q]);
    }
  }
  // The first member (in falling order) of `bin` at which the count (by_count) or the
  // weight reaches want >= 1, the last one if none does.
  MKD_DEV SmEnd select(int bin, bool by_count, u64 want) {
    stage(bin);
    uint32_t base = 0, range = kmax - kmin;   // the members' distances kmax - key: [base, base + range]
    unsigned left = n;                          // members there
    u64 front = 0;                              // weight before them
    const int x = threadIdx.x;
    while (left > 64 && range > 0) {
      const int bits = 32 - __clz(range), shift = bits > 9 ? bits - 9 : 0;
      s.sub_n[x] = 0;
      s.sub[x] = 0;
      if (x == 0) s.found = -1;
      __syncthreads();
      if (shift == 0) {
        // one key a sub-bin: counted, and weighed once
        for (unsigned m = x; m < n; m += kSmRow) {
          uint32_t key, index;
          member(m, key, index);
          const uint32_t d = kmax - key - base;
          if (d <= range) atomicAdd(&s.sub_n[d], 1u);
        }
      } else {
        for (unsigned m = x; m < n; m += kSmRow) {
          uint32_t key, index;
          member(m, key, index);
          const uint32_t d = kmax - key;
          if (d < base || d - base > range) continue;
          atomicAdd(&s.sub_n[(d - base) >> shift], 1u);
          atomicAdd(&s.sub[(d - base) >> shift], weight(key));
        }
      }
      __syncthreads();
      const unsigned cn = s.sub_n[x];
      const u64 cm = shift == 0 ? (cn ? cn * weight(kmax - (base + x)) : 0ull) : s.sub[x];
      unsigned sn = cn;
      u64 sm = cm;
      scan_nm(s, s.wave_m, sn, sm);
      // the sub-bin that reaches it, or the last one with members
      if (cn && (by_count ? sn : sm) >= want && (by_count ? sn - cn : sm - cm) < want) s.found = x;
      __syncthreads();
      const bool none = s.found < 0;
      __syncthreads();
      if (none) {
        if (cn) atomicMax(&s.found, x);
        __syncthreads();
      }
      const int hit = s.found;
      if (x == hit) {
        s.found_n = sn - cn;
        s.found_m = sm - cm;
      }
      __syncthreads();
      const u64 passed = by_count ? s.found_n : s.found_m;
      want = want > passed ? want - passed : 1;
      front += s.found_m;
      base += (uint32_t)hit << shift;
      left = s.sub_n[hit];
      range = (1u << shift) - 1u;
      __syncthreads();
    }
    if (left > 64) return equal_ones(bin, kmax - base, by_count, want, front, left);
    // ---- what is left, sorted by one wave ----
    if (x == 0) s.found_n = 0;
    __syncthreads();
    for (unsigned m = x; m < n; m += kSmRow) {
      uint32_t key, index;
      member(m, key, index);
      const uint32_t d = kmax - key;
      if (d >= base && d - base <= range) s.token[atomicAdd(&s.found_n, 1u)] = token_of(key, index);
    }
    __syncthreads();
    if (x < 64) {
      const u64 t = sort_wave(s.token, x < (int)left ? s.token[x] : ~0ull, left);
      const u64 own = x < (int)left ? weight(key_in(t)) : 0ull;
      u64 m = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const u64 up = __shfl_up(m, o, 64);
        if (x >= o) m += up;
      }
      const int pos = __popcll(__ballot(x + 1 < (int)left && (by_count ? (u64)x + 1 : m) < want));
      if (x == pos) {
        s.found_t = t;
        s.found_m = m;
      }
    }
    __syncthreads();
    const SmEnd e{s.found_t, before(bin) + (double)(front + s.found_m) * s.unit[bin]};
    __syncthreads();
    return e;
  }
  // more equal members than are sorted: the one at which it reaches `want`, by index
  MKD_DEV SmEnd equal_ones(int bin, uint32_t key, bool by_count, u64 want, u64 front, unsigned left) {
    const u64 each = weight(key);
    const unsigned rank = (unsigned)min(by_count ? want : (want + each - 1) / each, (u64)left);   // from 1
    const int x = threadIdx.x;
    if (x < nc) s.hits[x] = 0;
    if (x < kSmChunk / 32) s.bits[x] = 0;
    __syncthreads();
    for (unsigned m = x; m < n; m += kSmRow) {
      uint32_t k, index;
      member(m, k, index);
      if (k == key) atomicAdd(&s.hits[index / kSmChunk], 1u);
    }
    __syncthreads();
    unsigned v = x < nc ? s.hits[x] : 0, own = v;
    scan_n(s, v);
    if (x < nc && v >= rank && v - own < rank) {
      s.found = x;
      s.found_n = rank - (v - own);             // its rank in that chunk, from 1
    }
    __syncthreads();
    const int chunk = s.found;
    const unsigned in_chunk = s.found_n;
    for (unsigned m = x; m < n; m += kSmRow) {
      uint32_t k, index;
      member(m, k, index);
      if (k == key && (int)(index / kSmChunk) == chunk) atomicOr(&s.bits[index % kSmChunk / 32], 1u << (index % 32));
    }
    __syncthreads();
    uint32_t word = x < kSmChunk / 32 ? s.bits[x] : 0;
    v = own = __popc(word);
    scan_n(s, v);
    if (v >= in_chunk && v - own < in_chunk) {
      for (unsigned k = in_chunk - (v - own); k > 1; --k) word &= word - 1;
      s.found_t = token_of(key, chunk * kSmChunk + 32 * x + __ffs((int)word) - 1);
    }
    __syncthreads();
    const SmEnd e{s.found_t, before(bin) + (double)(front + rank * each) * s.unit[bin]};
    __syncthreads();
    return e;
  }
  MKD_DEV double before(int bin) const { return bin > 0 ? s.cum[bin - 1] : 0.0; }
};

}  // namespace

template <bool BF>
__global__ void __launch_bounds__(kSmRow) sample_row_kernel(mkd_sample_args a, const SmRecord* rec, int nc) {
  __shared__ SmShared s;
  const int b = blockIdx.x, x = threadIdx.x;
  rec += (long long)b * nc;
  const SmSetting set = setting_of(a, b);
  // ---- the row's largest logit, and each chunk's place below it ----
  const float mine = x < nc ? rec[x].top : -INFINITY;
  float top = wave_max(mine);                   // (chunks are 128 at most: the first 2 waves)
  if ((x & 63) == 0) s.wave_d[x >> 6] = top;
  __syncthreads();
  top = (float)fmax(s.wave_d[0], s.wave_d[1]);
  if (top == -INFINITY) {                       // nothing to choose
    if (x == 0) {
      a.tokens[b] = -1;
      if (a.logprobs) a.logprobs[b] = -INFINITY;
    }
    return;
  }
  const SmPlace top_at = place_of(top, set.inv_t);
  const double top_place = top_at.place;
  if (x < nc) {
    const double d = mine == top ? 0.0 : top_place - place_of(mine, set.inv_t).place;
    s.shift[x] = d < kSmBins ? (int)d : kSmBins;
  }
  __syncthreads();
  // ---- the row's bins, one a thread, the loads of 16 chunks in flight together ----
  {
    unsigned sn = 0;
    u64 m = 0;
    for (int c0 = 0; c0 < nc; c0 += 16) {
      u64 v[16];
      int k[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = min(c0 + i, nc - 1);
        k[i] = c0 + i < nc ? x - s.shift[c] : -1;
        v[i] = rec[c].bins[max(k[i], 0)];       // (what a chunk without tokens holds is not used)
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k[i] >= 0) {
          sn += (unsigned)(v[i] >> kSmMassBits);
          m += v[i] & ((1ull << kSmMassBits) - 1);
        }
    }
    // exp(middle - z_max)
    const double unit = top == INFINITY ? 1.0 / kSmOne
        : exp((-top_at.f - x) / kSmRes) / kSmOne;
    double sm = (double)m * unit;
    scan_nm(s, s.wave_d, sn, sm);
    s.cum_n[x] = sn;
    s.cum[x] = sm;
    s.unit[x] = unit;
  }
  __syncthreads();
  SmRow<BF> row{a, s, rec, b, nc, top, set.inv_t};
  // the first bin that reaches a target (all behind it do too); `last` if none does
  int last = kSmBins - 1;
  auto find_bin = [&](auto reached) { return min((int)count_of(s, !reached(x)), last); };
  const unsigned tokens = s.cum_n[kSmBins - 1];
  const double all = s.cum[kSmBins - 1];
  last = find_bin([&](int i) { return s.cum_n[i] >= tokens; });   // the last with members
  const bool by_k = set.top_k > 0 && (unsigned)set.top_k < tokens, by_p = set.top_p < 1.0;
  const int jk = by_k ? find_bin([&](int i) { return s.cum_n[i] >= (unsigned)set.top_k; }) : last;
  // ---- few tokens can stay: sort them ----
  // (all of the first top_k, whose mass top_p refers to; else those that top_p or min_p,
  // or without a filter the random number, can reach at most)
  int far = jk;
  if (!by_k) {
    far = last;
    if (set.min_p > 0.0 && top != INFINITY)     // one bin to spare
      far = (int)fmin(floor(-log(set.min_p) * kSmRes - top_at.f) + 2.0, (double)last);
    if (by_p || !(set.min_p > 0.0)) {
      const double most = (by_p ? set.top_p : set.u) * all;
      const int j = find_bin([&](int i) { return by_p ? s.cum[i] >= most : s.cum[i] > most; });
      far = min(far, j);
    }
  }
  far = max(far, 0);
  if (s.cum_n[far] <= kSmRow) {
    const unsigned n = row.locate(0, far);
    u64 t = ~0ull;
    if (x < (int)n) {
      uint32_t key[1], index[1];
      row.template fetch<1>(x, key, index);
      t = token_of(key[0], index[0]);
    }
    t = sort_up(s, t, n);
    const float l = logit_of<BF>(key_in(t));
    const double own = x < (int)n ? mass_of(l, top, set.inv_t) : 0.0;
    unsigned c = 0;
    double cum = own;
    scan_nm(s, s.wave_d, c, cum);
    double* at = reinterpret_cast<double*>(s.sub);
    at[x] = cum;
    __syncthreads();
    unsigned kept = by_k ? min((unsigned)set.top_k, n) : n;
    const double whole = n == tokens ? at[n - 1] : all;   // (sorted: without the bins' rounding)
    const double m1 = by_k ? at[kept - 1] : whole;
    if (by_p) kept = max(min(kept, count_of(s, x < (int)kept && cum - own < set.top_p * m1)), 1u);
    if (set.min_p > 0.0) kept = max(count_of(s, x < (int)kept && own >= set.min_p), 1u);
    // (without a filter the whole row's mass counts; the tokens sorted reach past u of it)
    const double m3 = by_k || by_p || set.min_p > 0.0 ? at[kept - 1] : whole;
    const unsigned pick = min(count_of(s, x < (int)kept && cum <= set.u * m3), kept - 1);
    if (x == (int)pick) {
      a.tokens[b] = (int)(uint32_t)t;
      if (a.logprobs) a.logprobs[b] = (float)log(own / m3);
    }
    return;
  }
  // ---- many: in steps ----
  // integer weight of a bin's front part that holds t of the row's mass
  auto in_bin = [&](int j, double t, bool past) -> u64 {
    const double v = (t - row.before(j)) / s.unit[j];
    if (!(v > 0.0)) return 1;
    return v < 0x1p62 ? (past ? (u64)v + 1 : (u64)ceil(v)) : 1ull << 62;
  };
  SmEnd end{~0ull, all};                        // behind everything
  if (by_k) end = row.select(jk, true, set.top_k - (jk > 0 ? s.cum_n[jk - 1] : 0u));
  if (by_p) {
    const double t = set.top_p * end.mass;
    const int j = find_bin([&](int i) { return s.cum[i] >= t; });
    end = row.select(j, false, in_bin(j, t, false));
  }
  if (set.min_p > 0.0) {
    // the smallest logit whose mass is min_p at least, from its estimate by steps of one
    float cut = top;
    if (set.min_p < 1.0 && top != INFINITY) {
      cut = fminf((float)((double)top + log(set.min_p) / set.inv_t), top);
      if (cut == -INFINITY) cut = -3.402823466e38f;
      uint32_t k = key_of<BF>(cut);
      for (int i = 0; i < 64 && logit_of<BF>(k) < top && mass_of(logit_of<BF>(k), top, set.inv_t) < set.min_p; ++i) ++k;
      for (int i = 0; i < 64 && mass_of(logit_of<BF>(k - 1), top, set.inv_t) >= set.min_p; ++i) --k;
      cut = logit_of<BF>(k);
    }
    const uint32_t key = key_of<BF>(cut);
    const double below = cut == top ? 0.0 : top_place - place_of(cut, set.inv_t).place;
    if (token_of(key, 0xffffffffu) < end.token && below < kSmBins) {
      const int j = (int)below;
      row.stage(j);                             // the weight of the bin's members at least as large
      u64 m = 0;
      for (unsigned i = x; i < row.n; i += kSmRow) {
        uint32_t k, index;
        row.member(i, k, index);
        if (k >= key) m += row.weight(k);
      }
      unsigned c = 0;
      scan_nm(s, s.wave_m, c, m);
      if (x == kSmRow - 1) s.found_m = m;
      __syncthreads();
      end = SmEnd{token_of(key, 0xffffffffu), row.before(j) + (double)s.found_m * s.unit[j]};
      __syncthreads();
    }
  }
  // ---- the token: the first whose cumulative mass passes u times the kept ----
  const double t = set.u * end.mass;
  const int j = find_bin([&](int i) { return s.cum[i] > t; });
  const SmEnd pick = row.select(j, false, in_bin(j, t, true));
  if (x == 0) {
    a.tokens[b] = (int)(uint32_t)pick.token;
    if (a.logprobs) a.logprobs[b] = (float)log(mass_of(logit_of<BF>(key_in(pick.token)), top, set.inv_t) / end.mass);
  }
}

size_t sample_workspace(int B, int V) {
  return (size_t)B * ((V + kSmChunk - 1) / kSmChunk) * sizeof(SmRecord);
}

namespace {

template <bool BF>
void sample_run(const mkd_sample_args& a, SmRecord* rec, bool vec, hipStream_t s) {
  const int nc = (a.V + kSmChunk - 1) / kSmChunk;
  const dim3 grid(nc, a.B);
  if (vec) hipLaunchKernelGGL((sample_chunk_kernel<BF, true>), grid, dim3(kSmThreads), 0, s, a, rec);
  else hipLaunchKernelGGL((sample_chunk_kernel<BF, false>), grid, dim3(kSmThreads), 0, s, a, rec);
  hipLaunchKernelGGL(sample_row_kernel<BF>, dim3(a.B), dim3(kSmRow), 0, s, a, rec, nc);
}

}  // namespace

hipError_t sample_launch(const mkd_sample_args& a, void* ws, hipStream_t s) {
  SmRecord* rec = static_cast<SmRecord*>(ws);
  const bool bf = a.logits_dtype == MKD_DT_BF16;
  const bool vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.row_stride * (bf ? 2 : 4) % 16 == 0;
  if (bf) sample_run<true>(a, rec, vec, s);
  else sample_run<false>(a, rec, vec, s);
  return hipGetLastError();
}

}  // namespace mkd
