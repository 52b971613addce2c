// One token per row of logits from a given random number, under temperature, top-k,
// top-p and min-p (mkd_sample_tokens), without sorting the vocabulary.
//
// With the tokens in falling order of logit, every filter keeps a front part and the
// random number asks for the first token whose cumulative mass passes a target: each is
// a weighted selection, "the first token at which a count or a mass reaches T".
//   1. chunks: block (4096 logits, row): masses exp((l - chunk max) / temperature) into
//      512 bins of 1/16 of scaled logit, at fixed places of that scale (so the chunks'
//      bins line up whatever their maxima), the members of each bin listed.
//   2. rows: one block joins the chunks' bins, scans them, and finds each filter's end
//      and then the token: the bin by its cumulative count or mass, then the exact logit
//      inside the bin by histograms over its members' bit patterns (ordered like the
//      logits, 10 bits a time), then among equal logits the index by rank.
// Tokens 512 bins (32, e^-32) below the maximum get no mass: together at most 2^-26 of
// the row's for 2^20 of them.
//
// The answer is a whole number, and a sum off in its last places would change it where a
// border lies near: masses are formed in fp64 and summed as 64-bit integers (of 2^-50 of
// the chunk's largest, 2^-42 of the bin's), which no order of atomic additions changes;
// only the joining of chunks is in fp64, in a fixed order.  Bound by reading the logits
// for large batches and by the two dependent launches for small ones.
#include "common.h"
#include "mkd_internal.h"

namespace mkd {

namespace {

constexpr int kSmChunk = 4096, kSmThreads = 256, kSmPer = kSmChunk / kSmThreads;
constexpr int kSmBins = 512;
constexpr double kSmRes = 16.0;                 // bins per unit of logit / temperature
constexpr int kSmMaxChunks = (1 << 20) / kSmChunk;
constexpr int kSmRow = 1024;                    // threads of a row's block, sub-bins of a level
constexpr int kSmStage = 8192;                  // members of a bin held in LDS

// What stage 1 leaves per (row, chunk).
struct SmRecord {
  unsigned long long mass[kSmBins];             // of 2^-50
  uint16_t list[kSmChunk];                      // positions in the chunk, by bin
  uint16_t start[kSmBins + 8];                  // of bin j in `list`; [kSmBins]: their number
  float top;                                    // the chunk's largest logit
  int pad[3];
};

struct SmSetting {
  double inv_t, top_p, min_p, u;
  int top_k;
};
MKD_DEV SmSetting setting_of(const mkd_sample_args& a, int b) {
  SmSetting s;
  const float t = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const bool greedy = !(t > 0.f);               // as top_k = 1
  s.inv_t = greedy ? 1.0 : 1.0 / (double)t;
  s.top_k = greedy ? 1 : (a.top_k_rows ? a.top_k_rows[b] : a.top_k);
  s.top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  s.min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  s.u = a.uniforms[b];
  if (!(s.u > 0.0)) s.u = 0.0;
  return s;
}
// exp((l - top) * inv_t), 1 for l = top whatever it is, 0 below an infinite top
MKD_DEV double mass_of(float l, float top, double inv_t) {
  if (l == top) return 1.0;
  if (top == INFINITY) return 0.0;
  return exp(((double)l - (double)top) * inv_t);
}
// the bin's place on the scale of logit / temperature (monotone in l)
MKD_DEV double place_of(float l, double inv_t) { return floor((double)l * inv_t * kSmRes); }
// bins between a logit and a larger one (kSmBins: outside)
MKD_DEV int bins_below(float l, float top, double inv_t) {
  if (l == top) return 0;
  const double d = place_of(top, inv_t) - place_of(l, inv_t);
  return d < kSmBins ? (int)d : kSmBins;        // (an infinite difference: outside)
}
// bit patterns in the order of the logits; -0 and +0 are one value
MKD_DEV uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
MKD_DEV float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <bool BF>
MKD_DEV float logit_at(const mkd_sample_args& a, long long row, int i) {
  const long long off = row * a.row_stride + i;
  const float l = BF ? bf2f(static_cast<const uint16_t*>(a.logits)[off]) : static_cast<const float*>(a.logits)[off];
  return l == l ? l : -INFINITY;
}

}  // namespace

// VEC: rows on 16-byte boundaries.  Element i of thread x is 4 x + 1024 (i / 4) + i % 4
// (bf16: 8 x + 2048 (i / 8) + i % 8).
template <bool BF, bool VEC>
__global__ void __launch_bounds__(kSmThreads) sample_chunk_kernel(mkd_sample_args a, SmRecord* rec) {
  __shared__ unsigned long long mass[kSmBins];
  __shared__ unsigned count[kSmBins];
  __shared__ __attribute__((aligned(16))) uint16_t list[kSmChunk];
  __shared__ float wtop[kSmThreads / 64];
  __shared__ unsigned wsum[kSmThreads / 64];
  const int x = threadIdx.x, lane = x & 63, w = x >> 6;
  const int b = blockIdx.y, base = blockIdx.x * kSmChunk, n = min(kSmChunk, a.V - base);
  SmRecord& r = rec[(long long)b * gridDim.x + blockIdx.x];
  for (int i = x; i < kSmBins; i += kSmThreads) { mass[i] = 0; count[i] = 0; }
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
        l[G * q + e] = f == f ? f : -INFINITY;
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
  top = fmaxf(fmaxf(wtop[0], wtop[1]), fmaxf(wtop[2], wtop[3]));
  if (x == 0) r.top = top;
  if (top == -INFINITY) return;                 // nothing to choose here (the rest is not read)
  uint16_t bin[kSmPer], rank[kSmPer];
#pragma unroll
  for (int i = 0; i < kSmPer; ++i) {
    bin[i] = kSmBins;
    if (l[i] == -INFINITY) continue;
    const int j = bins_below(l[i], top, s.inv_t);
    if (j >= kSmBins) continue;
    bin[i] = (uint16_t)j;
    rank[i] = (uint16_t)atomicAdd(&count[j], 1u);
    atomicAdd(&mass[j], (unsigned long long)rint(mass_of(l[i], top, s.inv_t) * 0x1p50));
  }
  __syncthreads();
  // exclusive scan of the counts, two bins a thread
  const unsigned c0 = count[2 * x], c1 = count[2 * x + 1];
  unsigned sum = c0 + c1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(sum, o, 64);
    if (lane >= o) sum += up;
  }
  if (lane == 63) wsum[w] = sum;
  __syncthreads();
  unsigned before = sum - c0 - c1, total = 0;
#pragma unroll
  for (int q = 0; q < kSmThreads / 64; ++q) {
    if (q < w) before += wsum[q];
    total += wsum[q];
  }
  count[2 * x] = before;
  count[2 * x + 1] = before + c0;
  reinterpret_cast<uint32_t*>(r.start)[x] = before | ((before + c0) << 16);
  if (x == 0) r.start[kSmBins] = (uint16_t)total;
  r.mass[2 * x] = mass[2 * x];
  r.mass[2 * x + 1] = mass[2 * x + 1];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSmPer; ++i)
    if (bin[i] < kSmBins) list[count[bin[i]] + rank[i]] = (uint16_t)(G * x + G * kSmThreads * (i / G) + i % G);
  __syncthreads();
  for (unsigned i = x * 8; i < total; i += kSmThreads * 8) st16(r.list + i, ld16(list + i));
}

namespace {

// A place in the falling order: the `ties`-th lowest index (from 1) among the members of
// `bin` with bit pattern `key`; `mass`: of everything up to it.
struct SmCut {
  int bin;
  uint32_t key, ties;
  double mass;
};
MKD_DEV bool later(const SmCut& a, const SmCut& b) {
  if (a.bin != b.bin) return a.bin > b.bin;
  return a.key != b.key ? a.key < b.key : a.ties > b.ties;
}

struct SmShared {
  double factor[kSmMaxChunks];                  // chunk's mass unit in the row's
  double cum[kSmBins];                          // mass up to bin j, itself included
  unsigned long long sub_mass[kSmRow], wave_m[kSmRow / 64];
  unsigned cum_n[kSmBins];
  unsigned sub_n[kSmRow], wave_n[kSmRow / 64];
  double wave_d[kSmRow / 64];
  int shift[kSmMaxChunks];                      // chunk's first bin in the row's
  unsigned first[kSmMaxChunks + 1];             // the staged bin's members before chunk c
  unsigned at[kSmMaxChunks];                    // where they start in the chunk's list
  uint32_t key[kSmStage], index[kSmStage];
  unsigned hits[kSmMaxChunks], bits[kSmChunk / 32];
  unsigned long long found_m;
  unsigned found_n;
  int found, token;
  uint32_t kmin, kmax;
};

// Inclusive scan over the block's 1024 threads (a thread's own total last).
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
MKD_DEV void scan_m(SmShared& s, unsigned long long& v) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  if (lane == 63) s.wave_m[w] = v;
  __syncthreads();
  for (int q = 0; q < w; ++q) v += s.wave_m[q];
  __syncthreads();
}
MKD_DEV void scan_d(SmShared& s, double& v) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  if (lane == 63) s.wave_d[w] = v;
  __syncthreads();
  double before = 0.0;
  for (int q = 0; q < w; ++q) before += s.wave_d[q];
  v += before;
  __syncthreads();
}

template <bool BF>
struct SmRow {
  const mkd_sample_args& a;
  SmShared& s;
  const SmRecord* rec;                          // the row's records
  int b, nc;
  float top;
  double inv_t;
  int staged = -1;
  unsigned n = 0;                               // members of the staged bin

  // member m of the staged bin: its index, and its logit's bit pattern
  MKD_DEV void member(unsigned m, uint32_t& key, uint32_t& index) const {
    if (n <= kSmStage) {
      key = s.key[m];
      index = s.index[m];
    } else {
      fetch(m, key, index);
    }
  }
  MKD_DEV void fetch(unsigned m, uint32_t& key, uint32_t& index) const {
    int lo = 0, hi = nc;                        // the chunk: first[lo] <= m < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s.first[mid] <= m) lo = mid;
      else hi = mid;
    }
    index = lo * kSmChunk + rec[lo].list[s.at[lo] + m - s.first[lo]];
    key = key_of(logit_at<BF>(a, b, index));
  }
  MKD_DEV void stage(int bin) {
    if (staged == bin) return;
    staged = bin;
    __syncthreads();
    const int c = threadIdx.x;
    unsigned cnt = 0, at = 0;
    if (c < nc && rec[c].top != -INFINITY && s.shift[c] <= bin && bin - s.shift[c] < kSmBins) {
      const int j = bin - s.shift[c];
      at = rec[c].start[j];
      cnt = rec[c].start[j + 1] - at;
    }
    unsigned v = cnt;
    scan_n(s, v);
    if (c < nc) {
      s.first[c] = v - cnt;
      s.at[c] = at;
      if (c == nc - 1) s.first[nc] = v;
    }
    if (c == 0) { s.kmin = 0xffffffffu; s.kmax = 0u; }
    __syncthreads();
    n = s.first[nc];
    uint32_t lo = 0xffffffffu, hi = 0u;
    for (unsigned m = threadIdx.x; m < n; m += kSmRow) {
      uint32_t key, index;
      fetch(m, key, index);
      if (n <= kSmStage) {
        s.key[m] = key;
        s.index[m] = index;
      }
      lo = min(lo, key);
      hi = max(hi, key);
    }
    if (hi >= lo) {
      atomicMin(&s.kmin, lo);
      atomicMax(&s.kmax, hi);
    }
    __syncthreads();
  }
  // a member's mass, of 2^-42 of the bin's largest
  MKD_DEV unsigned long long weight(uint32_t key, float bin_top) const {
    return (unsigned long long)rint(mass_of(logit_of(key), bin_top, inv_t) * 0x1p42);
  }
  // The first member (by falling logit, equal ones by index) of `bin` at which the count
  // (by_count) or the integer mass reaches want >= 1; the last one if none does.
  MKD_DEV SmCut select(int bin, bool by_count, unsigned long long want, double mass_before) {
    stage(bin);
    const uint32_t kmax = s.kmax;
    const float bin_top = logit_of(kmax);
    const double unit = mass_of(bin_top, top, inv_t);
    uint32_t base = 0, range = kmax - s.kmin;   // distances kmax - key in [base, base + range]
    unsigned long long before = 0;              // mass in front of them
    const int x = threadIdx.x;
    uint32_t at_key;
    unsigned at_n;
    for (;;) {
      const int bits = range ? 32 - __clz(range) : 0, shift = bits > 10 ? bits - 10 : 0;
      s.sub_n[x] = 0;
      s.sub_mass[x] = 0;
      if (x == 0) s.found = -1;
      __syncthreads();
      for (unsigned m = x; m < n; m += kSmRow) {
        uint32_t key, index;
        member(m, key, index);
        const uint32_t d = kmax - key;
        if (d < base || d - base > range) continue;
        atomicAdd(&s.sub_n[(d - base) >> shift], 1u);
        atomicAdd(&s.sub_mass[(d - base) >> shift], weight(key, bin_top));
      }
      __syncthreads();
      const unsigned cn = s.sub_n[x];
      const unsigned long long cm = s.sub_mass[x];
      unsigned sn = cn;
      unsigned long long sm = cm;
      scan_n(s, sn);
      scan_m(s, sm);
      const unsigned long long upto = by_count ? sn : sm;
      // the sub-bin that reaches it, or the last one with members
      if (cn && upto >= want && (by_count ? sn - cn : sm - cm) < want) s.found = x;
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
      const unsigned long long front = by_count ? s.found_n : s.found_m;
      want = want > front ? want - front : 1;
      before += s.found_m;
      base += (uint32_t)hit << shift;
      at_n = s.sub_n[hit];
      __syncthreads();
      if (shift == 0) {
        at_key = kmax - base;
        break;
      }
      range = (1u << shift) - 1u;
    }
    const unsigned long long each = by_count ? 1ull : max(weight(at_key, bin_top), 1ull);
    const unsigned long long ties = min((want + each - 1) / each, (unsigned long long)at_n);
    SmCut c;
    c.bin = bin;
    c.key = at_key;
    c.ties = (uint32_t)max(ties, 1ull);
    c.mass = mass_before + (double)(before + c.ties * weight(at_key, bin_top)) * 0x1p-42 * unit;
    return c;
  }
  // the index that a cut names
  MKD_DEV int index_of(const SmCut& c) {
    stage(c.bin);
    const int x = threadIdx.x;
    if (x < nc) s.hits[x] = 0;
    if (x < kSmChunk / 32) s.bits[x] = 0;
    __syncthreads();
    for (unsigned m = x; m < n; m += kSmRow) {
      uint32_t key, index;
      member(m, key, index);
      if (key == c.key) atomicAdd(&s.hits[index / kSmChunk], 1u);
    }
    __syncthreads();
    unsigned v = x < nc ? s.hits[x] : 0, own = v;
    scan_n(s, v);
    if (x < nc && v >= c.ties && v - own < c.ties) {
      s.found = x;
      s.found_n = c.ties - (v - own);           // its rank in that chunk, from 1
    }
    __syncthreads();
    const int chunk = s.found;
    const unsigned rank = s.found_n;
    for (unsigned m = x; m < n; m += kSmRow) {
      uint32_t key, index;
      member(m, key, index);
      if (key == c.key && (int)(index / kSmChunk) == chunk)
        atomicOr(&s.bits[index % kSmChunk / 32], 1u << (index % 32));
    }
    __syncthreads();
    uint32_t word = x < kSmChunk / 32 ? s.bits[x] : 0;
    v = own = __popc(word);
    scan_n(s, v);
    if (v >= rank && v - own < rank) {
      for (unsigned k = rank - (v - own); k > 1; --k) word &= word - 1;
      s.token = chunk * kSmChunk + 32 * x + __ffs((int)word) - 1;
    }
    __syncthreads();
    return s.token;
  }
};

}  // namespace

template <bool BF>
__global__ void __launch_bounds__(kSmRow) sample_row_kernel(mkd_sample_args a, const SmRecord* rec, int nc) {
  __shared__ SmShared s;
  const int b = blockIdx.x, x = threadIdx.x;
  rec += (long long)b * nc;
  const SmSetting set = setting_of(a, b);
  // ---- the row's largest logit, each chunk's place and unit ----
  const float mine = x < nc ? rec[x].top : -INFINITY;
  float top = wave_max(mine);                   // (chunks are 256 at most: the first 4 waves)
  if ((x & 63) == 0) s.wave_d[x >> 6] = top;
  __syncthreads();
  top = -INFINITY;
  for (int q = 0; q < kSmRow / 64; ++q) top = fmaxf(top, (float)s.wave_d[q]);
  if (top == -INFINITY) {                       // nothing to choose
    if (x == 0) {
      a.tokens[b] = -1;
      if (a.logprobs) a.logprobs[b] = -INFINITY;
    }
    return;
  }
  if (x < nc) {
    const bool live = mine != -INFINITY;
    s.shift[x] = live ? bins_below(mine, top, set.inv_t) : kSmBins;
    s.factor[x] = live ? mass_of(mine, top, set.inv_t) * 0x1p-50 : 0.0;
  }
  __syncthreads();
  // ---- the row's bins: two threads each, even and odd chunks ----
  {
    const int j = x >> 1;
    unsigned cnt = 0;
    double m = 0.0;
    for (int c = x & 1; c < nc; c += 2) {
      const int k = j - s.shift[c];
      if (k < 0) continue;                      // (a chunk without tokens: its shift is past every bin)
      cnt += rec[c].start[k + 1] - rec[c].start[k];
      m += (double)rec[c].mass[k] * s.factor[c];
    }
    cnt += __shfl_xor(cnt, 1, 64);
    const double other = __shfl_xor(m, 1, 64);
    m = (x & 1) ? other + m : m + other;
    unsigned sn = (x & 1) ? 0 : cnt;
    double sm = (x & 1) ? 0.0 : m;
    scan_n(s, sn);
    scan_d(s, sm);
    if (!(x & 1)) {
      s.cum_n[j] = sn;
      s.cum[j] = sm;
    }
  }
  __syncthreads();
  SmRow<BF> row{a, s, rec, b, nc, top, set.inv_t};
  // the first bin that reaches a target; `last` if none does
  int last = kSmBins - 1;
  auto find_bin = [&](auto reached) {
    __syncthreads();
    if (x == 0) s.found = last;
    __syncthreads();
    if (x < kSmBins && reached(x)) atomicMin(&s.found, x);
    __syncthreads();
    const int j = s.found;
    __syncthreads();
    return j;
  };
  auto before = [&](int j) { return j > 0 ? s.cum[j - 1] : 0.0; };
  auto members = [&](int j) { return s.cum_n[j] - (j > 0 ? s.cum_n[j - 1] : 0u); };
  // integer mass of a bin's front part that holds t of the row's units
  auto in_bin = [&](int j, double t, bool past) -> unsigned long long {
    row.stage(j);
    const double v = t / mass_of(logit_of(s.kmax), top, set.inv_t) * 0x1p42;
    if (!(v > 0.0)) return 1;
    return v < 0x1p63 ? (past ? (unsigned long long)v + 1 : (unsigned long long)ceil(v)) : ~0ull >> 1;
  };
  last = find_bin([&](int i) { return s.cum_n[i] >= s.cum_n[kSmBins - 1]; });   // the last with members
  const double all = s.cum[kSmBins - 1];
  SmCut end{kSmBins, 0u, 0u, all};              // behind everything
  if (set.top_k > 0 && (unsigned)set.top_k < s.cum_n[kSmBins - 1]) {
    const unsigned k = set.top_k;
    const int j = find_bin([&](int i) { return s.cum_n[i] >= k; });
    end = row.select(j, true, k - (j > 0 ? s.cum_n[j - 1] : 0u), before(j));
  }
  if (set.top_p < 1.0) {
    const double t = set.top_p * end.mass;
    const int j = find_bin([&](int i) { return s.cum[i] >= t && members(i); });
    const SmCut c = row.select(j, false, in_bin(j, t - before(j), false), before(j));
    if (later(end, c)) end = c;
  }
  if (set.min_p > 0.0) {
    // the smallest logit whose mass is min_p at least, from its estimate by steps of one
    float cut = top;
    if (set.min_p < 1.0 && top != INFINITY) {
      cut = fminf((float)((double)top + log(set.min_p) / set.inv_t), top);
      if (cut == -INFINITY) cut = -3.402823466e38f;
      uint32_t k = key_of(cut);
      for (int i = 0; i < 64 && logit_of(k) < top && mass_of(logit_of(k), top, set.inv_t) < set.min_p; ++i) ++k;
      for (int i = 0; i < 64 && mass_of(logit_of(k - 1), top, set.inv_t) >= set.min_p; ++i) --k;
      cut = logit_of(k);
    }
    const int j = bins_below(cut, top, set.inv_t);
    if (j < end.bin || (j == end.bin && key_of(cut) > end.key)) {
      // the members of bin j at least as large: a selection by their number
      row.stage(min(j, kSmBins - 1));
      if (x == 0) s.found_n = 0;
      __syncthreads();
      unsigned hits = 0;
      if (j < kSmBins)
        for (unsigned m = x; m < row.n; m += kSmRow) {
          uint32_t key, index;
          row.member(m, key, index);
          hits += key >= key_of(cut);
        }
      if (hits) atomicAdd(&s.found_n, hits);
      __syncthreads();
      hits = s.found_n;
      __syncthreads();
      if (hits) {
        end = row.select(j, true, hits, before(j));
      } else if (j < kSmBins) {                 // everything in front of the bin
        const double m = before(j);
        const int i = find_bin([&](int q) { return s.cum_n[q] >= (j > 0 ? s.cum_n[j - 1] : 0u); });
        end = SmCut{i, 0u, 0xffffffffu, m};     // (a place behind the bin's last member)
      }
    }
  }
  // ---- the token: the first whose cumulative mass passes u times the kept ----
  const double t = set.u * end.mass;
  int j = find_bin([&](int i) { return s.cum[i] > t && members(i); });
  if (j > end.bin) j = end.bin;
  SmCut pick = row.select(j, false, in_bin(j, t - before(j), true), before(j));
  if (later(pick, end)) pick = end;
  const int token = row.index_of(pick);
  if (x == 0) {
    a.tokens[b] = token;
    if (a.logprobs) a.logprobs[b] = (float)log(mass_of(logit_of(pick.key), top, set.inv_t) / end.mass);
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
