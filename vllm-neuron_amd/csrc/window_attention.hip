// window_attention.hip — attention over a paged cache with a sliding window and
// a few first tokens that stay visible, bf16 MFMA on gfx950.
//
// Mathematics.  The query at position p sees key t where t <= p and (t < first or t > p -
// window): out = sum exp(s_t - m) v_t / (sum exp(s_t - m) + exp(sink - m)), s_t = scale
// q.k_t, tile by tile with a running maximum m and sum in fp32.  Codes of an 8-bit
// cache are exact in bf16: a key's scale multiplies its score, its value's the
// probability.
//
// Keys.  Only those that a row tile sees are read: groups of 16 keys (one block, one
// table entry), the first tokens' and then the window's, end to end.  Blocks between
// them may be freed; what lies in unseen places of a group reaches nothing (scores
// replaced by -inf, values by zeros).
//
// Forms, by the rows of a sequence and kv head (query tokens x heads of the group):
//   tall  128 rows a workgroup, 32 per wave, 64-key tiles of K and V through two LDS
//         stages (v_mfma_f32_32x32x16_bf16), probabilities rounded to bf16.  Bound by power
//         and issue: 8191 tokens, 32 heads of d = 128, window 2048: 277-293 us by card,
//         840-890 TFLOP/s, matrix units and vector instructions busy 45 % of the
//         cycles each, the clock at 1.8 GHz.  Eight waves in two groups, one in its
//         products while the other is in its softmax, took 294; the next tile's scores between
//         this one's exponentials 345; fragments read 4 or 6 ahead instead of 2 the same.
//         Short windows: 2183 tokens of 64 heads, d = 64, window 128: 23.4 us, two
//         thirds of it start, loads' latency and stores.
//   thin  16 or 32 rows: each wave streams 32-key tiles of its own, K straight to
//         operands, V through LDS (v_mfma_f32_16x16x32_bf16).  Probabilities go in two
//         bf16 parts (the second product is free here), so that the result is as exact
//         as the bf16 output.  Bound by HBM: 64 tokens over 4100 keys, 32 heads, d = 128:
//         178 us, 5.8 TB/s; 128 over 528 int8 keys, d = 64: 19.3-20.6 us, 3.5-3.7 TB/s.
//         Few rows: by the chain lengths, table, keys, values, join (4 tokens over 1028 keys
//         9.8-10.5 us).
#include <algorithm>

#include "attn_tile.h"

namespace mia {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = 128;     // query rows of a tall workgroup (4 waves x 32)
constexpr int kTallKeys = 64;  // keys per tall tile
constexpr int kThinKeys = 32;  // keys per thin tile
constexpr int kAhead = 2;      // tall: operand fragments read ahead of their product

struct WindowParams {
  const uint16_t *q;
  int64_t qs_t, qs_h;
  uint16_t *out;
  int64_t os_t, os_h;
  int num_tokens, n_seq;
  const int32_t *cu;   // [n_seq + 1] first query tokens, or NULL: one each
  const int32_t *len;  // [n_seq] keys
  int tok_max;         // query tokens of a sequence at most
  int zero_rest;       // rows that nothing computes are cleared
  int cap;             // keys a table row can hold
  int window, first;
  int G, Hkv, d;
  FastDiv g_div;
  const int32_t *bt;
  int64_t bt_s, bt_j;
  const uint8_t *k_cache, *v_cache;
  uint32_t kc_blk16, vc_blk16;     // block strides in 16-byte units
  int64_t kc_h, vc_h;              // bytes
  uint32_t kc_t, vc_t;
  const float *k_sc, *v_sc;        // per-key scales or NULL
  uint32_t ks_blk, ks_t, vs_blk, vs_t;  // elements
  int64_t ks_h, vs_h;
  const float *k_deq, *v_deq;      // per-head scales or NULL
  const float *sink;
  int nb, bs;
  FastDiv bs_div;
  float scale_log2;
  int rt_max;     // row tiles of a sequence at most
  int split;      // pieces of a row tile's keys
  FastDiv rt_div, split_div, seq_div;
  int part_rows;  // rows of a partial
  float *part_o;  // [piece][part_rows][D]
  float2 *part_ml;
};

// The keys that a row tile sees: those of a sequence's rows [r0, r1), whose
// first and last query stand at p_lo and p_hi: [0, min(first, hi)) and [lo, hi).
// They are taken in groups of 16, the first tokens' and then the window's, end to
// end, and a tile is the next 2 or 4 groups of that list: 128 keys behind 4 first
// ones fill three tiles of 64, where tiles that start at multiples of 64 are five.
struct Tiles {
  int tok0, rows;      // first query token, rows of the sequence
  int pos0;            // position of its first query
  int p_lo, p_hi, lo, hi;
  int n_first, g_lo;   // groups of first tokens, first group of the window
  int n;               // tiles

  template <int T>
  MIA_DEV bool set(const WindowParams &p, int i, int r0, int rows_tile) {
    int a = i, b = i + 1;
    if (p.cu) {
      a = min(max(scalar_load(p.cu, i), 0), p.num_tokens);
      b = min(max(scalar_load(p.cu, i + 1), a), p.num_tokens);
    }
    tok0 = a;
    rows = min(b - a, p.tok_max) * p.G;
    if (r0 >= rows) return false;
    const int len = min(max(scalar_load(p.len, i), 0), p.cap);
    pos0 = len - (b - a);
    const int r1 = min(r0 + rows_tile, rows);
    p_lo = pos0 + (int)fdiv((uint32_t)r0, p.g_div);
    p_hi = pos0 + (int)fdiv((uint32_t)(r1 - 1), p.g_div);
    hi = max(p_hi + 1, 0);
    lo = min(max(p_lo - p.window + 1, 0), hi);
    g_lo = lo / 16;
    n_first = min((min(p.first, hi) + 15) / 16, g_lo);
    n = (n_first + (hi + 15) / 16 - g_lo + T / 16 - 1) / (T / 16);
    return true;
  }
  // first key of group g of the list (past its end: keys that no row sees)
  MIA_DEV int key(int g) const { return (g < n_first ? g : g - n_first + g_lo) * 16; }
  // does any row of the tile see key k?
  MIA_DEV bool any(int k, int first) const { return k < hi && (k < first || k >= lo); }
  // are there keys among the 16 from k on that none sees?
  MIA_DEV bool edge(int k, int first) const {
    return k + 16 > hi || (k < lo && k + 16 > first);
  }
};
// Do the rows from position lo to hi all see every key of [k0, k1)?
MIA_DEV bool see_all(const WindowParams &p, int lo, int hi, int k0, int k1) {
  return k1 - 1 <= lo && (k1 <= p.first || k0 > hi - p.window);
}

// Where a head's keys lie (wave-uniform).
struct Keys {
  const int32_t *bt;
  const uint8_t *k, *v;
  const float *ks, *vs;
  MIA_DEV void set(const WindowParams &p, int i, int h) {
    bt = p.bt + (int64_t)i * p.bt_s;
    k = p.k_cache + (int64_t)h * p.kc_h;
    v = p.v_cache + (int64_t)h * p.vc_h;
    ks = p.k_sc + (int64_t)h * p.ks_h;
    vs = p.v_sc + (int64_t)h * p.vs_h;
  }
  // first key of the 16-key group at k0, kept inside the table
  MIA_DEV int first(const WindowParams &p, int k0) const { return min(k0, p.cap - 16); }
  MIA_DEV int entry(const WindowParams &p, int k0) const {
    return scalar_load(bt, (int64_t)fdiv((uint32_t)first(p, k0), p.bs_div) * p.bt_j);
  }
};

// A 16-key group: its block and its first key inside the block, both inside
// the pool whatever the table holds.
struct Group {
  uint32_t blk, off;
  const uint8_t *k, *v;
  MIA_DEV void set(const WindowParams &p, const Keys &s, int k0, int entry) {
    const int k16 = s.first(p, k0);
    blk = min(max(entry, 0), p.nb - 1);
    off = k16 - (int)fdiv((uint32_t)k16, p.bs_div) * p.bs;
    k = s.k + (((uint64_t)blk * p.kc_blk16) << 4) + (uint64_t)off * p.kc_t;
    v = s.v + (((uint64_t)blk * p.vc_blk16) << 4) + (uint64_t)off * p.vc_t;
  }
  MIA_DEV const float *ks(const WindowParams &p, const Keys &s) const {
    return s.ks + (uint64_t)blk * p.ks_blk + (uint64_t)off * p.ks_t;
  }
  MIA_DEV const float *vs(const WindowParams &p, const Keys &s) const {
    return s.vs + (uint64_t)blk * p.vs_blk + (uint64_t)off * p.vs_t;
  }
};

// Keys that a lane's row does not see, a bit for each of its scores.  A lane
// holds four consecutive keys of every STEP, from its first one on, N in all, in
// the order of the keys: those at a distance of at most d behind the first are
// its first count(d) scores.
template <int STEP, int N>
MIA_DEV uint32_t hidden(const WindowParams &p, int pos, int k0) {
  auto count = [](int d) {
    d = min(max(d, -1), N / 4 * STEP - 1);
    constexpr int SH = STEP == 8 ? 3 : 4;
    return (d >> SH) * 4 + min((d & (STEP - 1)) + 1, 4);
  };
  auto bits = [](int n) { return n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  const int dist = pos - k0;
  const uint32_t behind = bits(count(dist));  // at or before the row's position
  const uint32_t old = bits(count(dist - p.window));
  const uint32_t first = bits(count(p.first - 1 - k0));
  return ~(behind & (~old | first));
}
MIA_DEV float hide(float x, uint32_t hid, int bit) {
  const uint32_t t = (uint32_t)__builtin_amdgcn_sbfe((int)hid, bit, 1);
  return __uint_as_float((t & 0xff800000u) | (~t & __float_as_uint(x)));
}

// log2(e) x softmax scale x per-head scale of K: its magnitude; a negative
// factor goes to q (sign bits), so that the largest product is the largest
// score.
MIA_DEV float score_factor(const WindowParams &p, int h, uint32_t &neg) {
  float c1 = p.scale_log2;
  if (p.k_deq) c1 *= p.k_deq[h];
  neg = c1 < 0.f ? 0x80008000u : 0u;
  const float c2 = fabsf(c1);
  return c2 == 0.f ? 1e-37f : c2;  // masked scores (-inf) stay masked
}

// Factor of a finished row's accumulators: 1 / (sum of its exponentials and
// its sink's), times the per-head scale of V; 0 where it saw no key.
MIA_DEV float row_factor(const WindowParams &p, int h, int hq, float m, float l) {
  if (m == -INFINITY) return 0.f;
  if (p.sink) l += __builtin_amdgcn_exp2f(fmaf(p.sink[hq], kLog2e, -m));
  float f = l == 0.f ? 0.f : 1.f / l;
  if (p.v_deq) f *= p.v_deq[h];
  return f;
}

// Workgroup -> (head, sequence, row tile, piece).  Workgroups go round robin
// over the 8 XCDs: each takes a contiguous run of the list, ordered by head,
// sequence and row tile, so that row tiles that share keys share an L2.
struct Work {
  int h, i, rt, s;
  int64_t piece;
  // Zeros in the rows of tokens that no sequence computes: those behind the
  // longest allowed of this one, before the first and behind the last one,
  // shared by the workgroups of the sequence and head.
  MIA_DEV void clear_rest(const WindowParams &p) const {
    if (!p.zero_rest || s) return;
    int a = i, b = i + 1;
    if (p.cu) {
      a = min(max(scalar_load(p.cu, i), 0), p.num_tokens);
      b = min(max(scalar_load(p.cu, i + 1), a), p.num_tokens);
    }
    auto clear = [&](int t0, int t1) {
      const int c4 = p.d / 4, row = p.G * c4;
      for (int t = t0 + rt; t < t1; t += p.rt_max)
        for (int x = threadIdx.x; x < row; x += blockDim.x) {
          const int g = x / c4;
          *reinterpret_cast<u32x2_t *>(p.out + (int64_t)t * p.os_t +
                                       (int64_t)(h * p.G + g) * p.os_h + (x - g * c4) * 4) =
              u32x2_t{0u, 0u};
        }
    };
    if (b - a > p.tok_max) clear(a + p.tok_max, b);
    if (i == 0) clear(0, a);
    if (i == p.n_seq - 1) clear(b, p.num_tokens);
  }
  MIA_DEV void set(const WindowParams &p) {
    const int total = gridDim.x, b = blockIdx.x;
    const int full = total / 8, rem = total % 8, x = b % 8;
    int id = x * full + min(x, rem) + b / 8;
    piece = id;
    int next = (int)fdiv((uint32_t)id, p.split_div);
    s = id - next * p.split;
    id = next;
    next = (int)fdiv((uint32_t)id, p.rt_div);
    rt = id - next * p.rt_max;
    h = (int)fdiv((uint32_t)next, p.seq_div);
    i = next - h * p.n_seq;
  }
  // the piece's tiles [x, y) of n (at most 2^25, of at most 32 pieces)
  MIA_DEV int2 share(const WindowParams &p, int n) const {
    if (p.split == 1) return make_int2(0, n);
    return make_int2((int)fdiv((uint32_t)(n * s), p.split_div),
                     (int)fdiv((uint32_t)(n * (s + 1)), p.split_div));
  }
};

// ---------------------------------------------------------------------------
// tall form
// ---------------------------------------------------------------------------
template <int D, int CT, bool SC>
struct TallLds {
  static constexpr int TILEB = kTallKeys * D * 2;
  uint8_t kv[2][2][TILEB];             // [stage][K, V]
  float sc[2][2][SC ? kTallKeys : 4];  // [stage][K, V]
};

// DU <= D: the products stop there (a head dim of at most DU; channels past
// the head dim are zero).
template <int D, int CT, bool SC, int DU>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void window_tall_kernel(WindowParams p) {
  constexpr bool DMA = CT == kBf16;  // else through registers, widened
  constexpr int EB = CT == kBf16 ? 2 : 1;
  constexpr int CE = 16 / EB;        // elements per 16-byte load
  constexpr int LPR = D / CE;        // lanes per key row
  constexpr int RPW = 64 / LPR;      // key rows per wave and load
  constexpr int NP = 16 / RPW;       // loads per thread and tile (K, V each)
  constexpr int ROWB = D * 2;
  constexpr int TILEB = kTallKeys * ROWB;
  constexpr int KSTEPS = DU / 16;
  constexpr int DBLK = DU / 32;
  __shared__ __attribute__((aligned(1024))) TallLds<D, CT, SC> lds;

  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int rl = lane & 31;
  lds_u8_t *const base = (lds_u8_t *)&lds.kv[0][0][0];
  lds_f32_t *const scb = (lds_f32_t *)&lds.sc[0][0][0];

  Work wk;
  wk.set(p);
  wk.clear_rest(p);
  Tiles tl;
  const int r0 = wk.rt * kRows;
  if (!tl.set<kTallKeys>(p, wk.i, r0, kRows)) return;
  const int2 share = wk.share(p, tl.n);
  const int x0 = share.x, x1 = share.y;

  // (the first table entry is under way while the rows are loaded)
  Keys keys;
  keys.set(p, wk.i, wk.h);
  int ent = 0;  // the wave's table entry of a tile, loaded one tile ahead
  auto load_entry = [&](int x) { ent = keys.entry(p, tl.key(4 * x + wave)); };
  if (x0 < x1) load_entry(x0);

  // ---- the rows
  const int rloc = wave * 32 + rl;
  const int r = r0 + rloc;
  const bool ok = r < tl.rows;
  const bool live = r0 + wave * 32 < tl.rows;
  const int j = (int)fdiv((uint32_t)(ok ? r : 0), p.g_div);
  const int hq = wk.h * p.G + (ok ? r - j * p.G : 0);
  const int pos = tl.pos0 + j;
  u32x4_t qw[KSTEPS];
  {
    const uint16_t *qp = p.q + (int64_t)(tl.tok0 + j) * p.qs_t + (int64_t)hq * p.qs_h;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      qw[ks] = u32x4_t{0u, 0u, 0u, 0u};
      const int d0 = ks * 16 + half * 8;
      if (ok && d0 < p.d) qw[ks] = *reinterpret_cast<const u32x4_t *>(qp + d0);
    }
  }

  // ---- loads of a tile: wave w takes the 16 keys 16 w .. (one block: one
  // table entry), thread -> row jj * RPW + lr of them, chunk lc
  const int lr = lane / LPR;
  const int lc = lane % LPR;
  const bool ch_ok = lc * CE < p.d;
  constexpr int NR = DMA ? 1 : NP;
  u32x4_t kr[NR], vr[NR];
  float sr[NR];
  // the chunk a lane loads: for copies the one that the swizzle puts in its
  // slot, else its own (past the head dim: the first, stored nowhere)
  auto k_chunk = [&](int jj) { return DMA ? lc ^ k_swz<D>(jj * RPW + lr) : ch_ok ? lc : 0; };
  auto v_chunk = [&](int jj) { return DMA ? lc ^ v_swz<D>(jj * RPW + lr) : ch_ok ? lc : 0; };
  uint32_t ko[NP], vo[NP];  // a lane's bytes from its group's first row
#pragma unroll
  for (int jj = 0; jj < NP; ++jj) {
    ko[jj] = (uint32_t)(jj * RPW + lr) * p.kc_t + k_chunk(jj) * 16;
    vo[jj] = (uint32_t)(jj * RPW + lr) * p.vc_t + v_chunk(jj) * 16;
  }
  auto load_tile = [&](int x, int st) {
    const int k0 = tl.key(4 * x + wave);
    Group g;
    g.set(p, keys, k0, ent);
    if constexpr (DMA) {
      const uint32_t dst = (uint32_t)(uintptr_t)base + (st * 2) * TILEB + wave * 16 * ROWB;
      if (p.d == D) {
        copy16<NP>(g.k, ko, dst);
      } else {
#pragma unroll
        for (int jj = 0; jj < NP; ++jj)
          if (k_chunk(jj) * CE < p.d) copy1(g.k, ko[jj], dst + jj * 1024);
      }
      if (p.d == D && !tl.edge(k0, p.first)) {
        copy16<NP>(g.v, vo, dst + TILEB);
      } else {
        // values that no row sees are zeros: 0 * NaN would reach the sums (and
        // channels past d stay the zeros they are)
#pragma unroll
        for (int jj = 0; jj < NP; ++jj) {
          if (!tl.any(k0 + jj * RPW + lr, p.first))
            *(lds_u32x4_t *)(base + (st * 2 + 1) * TILEB + wave * 16 * ROWB + jj * 1024 +
                             lane * 16) = u32x4_t{0u, 0u, 0u, 0u};
          else if (v_chunk(jj) * CE < p.d)
            copy1(g.v, vo[jj], dst + TILEB + jj * 1024);
        }
      }
    } else {
#pragma unroll
      for (int jj = 0; jj < NP; ++jj) {
        kr[jj] = *reinterpret_cast<const u32x4_t *>(g.k + ko[jj]);
        vr[jj] = *reinterpret_cast<const u32x4_t *>(g.v + vo[jj]);
        if constexpr (SC) {
          // even lanes of a row its K scale, odd ones its V scale
          const float *sp = lc & 1 ? g.vs(p, keys) : g.ks(p, keys);
          sr[jj] = sp[(uint64_t)(jj * RPW + lr) * (lc & 1 ? p.vs_t : p.ks_t)];
        }
      }
    }
    if (x + 1 < x1) load_entry(x + 1);
  };
  // 8-bit caches: the loaded tile widened into stage st
  auto store_tile = [&](int x, int st) {
    const int k0 = tl.key(4 * x + wave);
    lds_u8_t *const kb = base + (st * 2) * TILEB;
    lds_u8_t *const vb = base + (st * 2 + 1) * TILEB;
#pragma unroll
    for (int jj = 0; jj < NR; ++jj) {
      const int row = wave * 16 + jj * RPW + lr;
      // values that no row sees are cleared: 0 * NaN would reach the sums
      const bool in = tl.any(k0 + jj * RPW + lr, p.first);
      const u32x4_t v = in ? vr[jj] : u32x4_t{0u, 0u, 0u, 0u};
      if (ch_ok)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        *(lds_u32x4_t *)(kb + row * ROWB + (((2 * lc + y) ^ k_swz<D>(row)) << 4)) =
            widen8<CT>(kr[jj][2 * y], kr[jj][2 * y + 1]);
        *(lds_u32x4_t *)(vb + row * ROWB + (((2 * lc + y) ^ v_swz<D>(row)) << 4)) =
            widen8<CT>(v[2 * y], v[2 * y + 1]);
        // converted a chunk at a time: all of them at once spill
        if constexpr (CT == kI8) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (SC) {
        if (lc < 2) scb[(st * 2 + lc) * kTallKeys + row] = in ? sr[jj] : 0.f;
      }
    }
  };

  uint32_t neg;
  const float c2 = score_factor(p, wk.h, neg);
  bf16x8_t qf[KSTEPS];
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks)
    qf[ks] = __builtin_bit_cast(bf16x8_t, qw[ks] ^ u32x4_t{neg, neg, neg, neg});
  f32x16_t acc[DBLK];
#pragma unroll
  for (int i = 0; i < DBLK; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  // transposed reads of V: within a 16-lane group, result lane k gets element
  // k % 4 of the 8 bytes read by lane 4j + k/4
  const int tr_k = lane & 15;
  const int tr_col = ((lane >> 4) & 1) * 16 + 4 * (tr_k & 3);
  const int tr_row = half * 4 + (tr_k >> 2);

  // positions of the wave's first and last row
  const int w_lo = tl.pos0 + (int)fdiv((uint32_t)min(r0 + wave * 32, tl.rows - 1), p.g_div);
  const int w_hi = tl.pos0 + (int)fdiv((uint32_t)min(r0 + wave * 32 + 31, tl.rows - 1), p.g_div);
  auto compute = [&](int x, int st) {
    // first key of the tile, and whether its groups follow each other
    const int kt = tl.key(4 * x);
    const bool row = 4 * x >= tl.n_first || 4 * x + 4 <= tl.n_first;
    if (row && (kt > w_hi || (kt >= p.first && kt + kTallKeys - 1 <= w_lo - p.window))) return;
    const lds_u8_t *kb = base + (st * 2) * TILEB;
    const lds_u8_t *vb = kb + TILEB;
    const lds_f32_t *ksb = scb + (st * 2) * kTallKeys;
    const lds_f32_t *vsb = ksb + kTallKeys;
    // S^T = K . Q^T: lane = row rl, value e of block b: key b*32 + (e/4)*8 +
    // half*4 + e%4
    f32x16_t s[2];
    auto read_k = [&](int b, int ks) {
      const int row = b * 32 + rl;
      return __builtin_bit_cast(
          bf16x8_t,
          *(const lds_u32x4_t *)(kb + row * ROWB + (((ks * 2 + half) ^ k_swz<D>(row)) << 4)));
    };
    auto read_v = [&](int k2, int db) {
      u32x2_t t2[2];
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int row = k2 * 16 + rr * 8 + tr_row;
        const int dd = db * 32 + tr_col;
        const int off = row * ROWB + (((dd >> 3) ^ v_swz<D>(row)) << 4) + ((dd & 7) << 1);
        t2[rr] = __builtin_bit_cast(
            u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vb + off)));
      }
      return __builtin_bit_cast(bf16x8_t, u32x4_t{t2[0][0], t2[0][1], t2[1][0], t2[1][1]});
    };
    // (fragments are read kAhead products ahead, an order held by the
    // scheduling barriers)
    __builtin_amdgcn_s_setprio(0);
    {
      constexpr int AHEAD = kAhead, N = 2 * KSTEPS;
      bf16x8_t kf[AHEAD + 1];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) kf[n] = read_k(n & 1, n >> 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n + AHEAD < N)
          kf[(n + AHEAD) % (AHEAD + 1)] = read_k((n + AHEAD) & 1, (n + AHEAD) >> 1);
        s[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            kf[n % (AHEAD + 1)], qf[n >> 1], n > 1 ? s[n & 1] : f32x16_t{}, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(1);
    if constexpr (SC) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_t ks4 = *(const lds_f32x4_t *)(ksb + b * 32 + g * 8 + half * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[b][g * 4 + i] *= ks4[i];
        }
    }
    if (!row || !see_all(p, w_lo, w_hi, kt, kt + kTallKeys)) {
      uint32_t hid = 0;
      if (row) {
        hid = hidden<8, 32>(p, pos, kt + half * 4);
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          hid |= (hidden<8, 8>(p, pos, tl.key(4 * x + g) + half * 4) & 0xffu) << (8 * g);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = hide(s[b][e], hid, b * 16 + e);
    }
    // online softmax; the maximum moves only when a score passes it by more
    // than 8 (log2 units): probabilities stay below 2^8, the accumulators are
    // rescaled on few tiles
    uint32_t pk[2][8];
    auto exps = [&]() {
      const float nm = m_run == -INFINITY ? 0.f : -m_run;
      float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float pr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            pr[i] = __builtin_amdgcn_exp2f(fmaf(s[b][g * 4 + i], c2, nm));
            ps[i] += pr[i];
          }
          if constexpr (SC) {
            const f32x4_t vs4 = *(const lds_f32x4_t *)(vsb + b * 32 + g * 8 + half * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[i] *= vs4[i];
          }
          // probabilities rounded to bf16 for the MFMA (half a step, 2^-8 of
          // each); their sum keeps the unrounded ones
          pk[b][g * 2] = pack2_bf16(pr[0], pr[1]);
          pk[b][g * 2 + 1] = pack2_bf16(pr[2], pr[3]);
        }
      return (ps[0] + ps[1]) + (ps[2] + ps[3]);
    };
    auto tile_max = [&]() {
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[b][e]);
      return max32(mx) * c2;
    };
    auto raise = [&](bool bump, float mx) {
      const float m_new = bump ? mx : m_run;
      const float alpha = m_run == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < DBLK; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= alpha;
    };
    const float mx = tile_max();
    const bool bump = mx > m_run + 8.f || (m_run == -INFINITY && mx > -INFINITY);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(bump) != 0, 0)) raise(bump, mx);
    const float psum = exps();
    l_run += psum;
    // O^T += V^T . P^T
    __builtin_amdgcn_s_setprio(0);
    {
      constexpr int AHEAD = kAhead, N = 4 * DBLK;
      bf16x8_t vf[AHEAD + 1];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) vf[n] = read_v(n / DBLK, n % DBLK);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n + AHEAD < N)
          vf[(n + AHEAD) % (AHEAD + 1)] = read_v((n + AHEAD) / DBLK, (n + AHEAD) % DBLK);
        const int k2 = n / DBLK, b = k2 >> 1, kh = k2 & 1;
        const u32x4_t bw = {pk[b][kh * 4], pk[b][kh * 4 + 1], pk[b][kh * 4 + 2], pk[b][kh * 4 + 3]};
        acc[n % DBLK] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            vf[n % (AHEAD + 1)], __builtin_bit_cast(bf16x8_t, bw), acc[n % DBLK], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(1);
  };

  // ---- the tiles
  if (x0 < x1) {
    if (p.d < D) {  // channels past d: zero in both stages, never written again
      for (int o = tid * 16; o < 4 * TILEB; o += kThreads * 16)
        *(lds_u32x4_t *)(base + o) = u32x4_t{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    load_tile(x0, 0);
    int st = 0;
    if constexpr (DMA) {
      for (int x = x0; x < x1; ++x) {
        // own copies of this tile have landed; the barrier makes every thread's
        // visible and the other stage free
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (x + 1 < x1) load_tile(x + 1, st ^ 1);
        if (live) compute(x, st);
        st ^= 1;
      }
    } else {
      store_tile(x0, 0);
      if (x0 + 1 < x1) load_tile(x0 + 1, 0);
      __syncthreads();
      for (int x = x0; x < x1; ++x) {
        if (live) compute(x, st);
        if (x + 1 < x1) store_tile(x + 1, st ^ 1);
        if (x + 2 < x1) load_tile(x + 2, 0);
        __syncthreads();
        st ^= 1;
      }
    }
  }

  // ---- final rows, or a partial
  const float l = sum32(l_run);
  if (p.split == 1) {
    // Through LDS, so that rows are stored in whole lines: a lane's own channels
    // come in pieces of 8 bytes, 16 of a row at a time, and L2 takes a request for
    // each (2183 tokens of 64 heads, d = 64, window 128: 24.8 against 23.4 us; 8191 of
    // 32 heads, d = 128: 73 against 67).
    const float f = ok ? row_factor(p, wk.h, hq, m_run, l) : 0.f;
    constexpr int PITCH = ROWB + 16, CPR = DU / 8, RPS = 64 / CPR;  // chunks of a row, rows a store
    static_assert(kWaves * 32 * PITCH <= 4 * TILEB, "the rows fit");
    __syncthreads();  // (the last tile has been read)
    lds_u8_t *const rows = base + wave * 32 * PITCH;
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(lds_u32x2_t *)(rows + rl * PITCH + (i * 32 + g * 8 + half * 4) * 2) =
            u32x2_t{pack2_bf16(acc[i][g * 4] * f, acc[i][g * 4 + 1] * f),
                    pack2_bf16(acc[i][g * 4 + 2] * f, acc[i][g * 4 + 3] * f)};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    typedef u32x4_t __attribute__((aligned(8))) u32x4_a8;  // (rows of out start at 8 bytes)
    const int c = lane % CPR;
    for (int y = lane / CPR; y < 32; y += RPS) {
      const int ro = r0 + wave * 32 + y;
      if (ro >= tl.rows) break;
      const int jo = (int)fdiv((uint32_t)ro, p.g_div);
      uint16_t *op = p.out + (int64_t)(tl.tok0 + jo) * p.os_t +
                     (int64_t)(wk.h * p.G + ro - jo * p.G) * p.os_h + c * 8;
      const u32x4_t v = *(const lds_u32x4_t *)(rows + y * PITCH + c * 16);
      if (lane < CPR * RPS && c * 8 < p.d) *reinterpret_cast<u32x4_a8 *>(op) = v;
    }
    return;
  }
  if (!ok) return;
  const int64_t pr = wk.piece * p.part_rows + rloc;
  float *po = p.part_o + pr * D;
#pragma unroll
  for (int i = 0; i < DBLK; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4_t *>(po + i * 32 + g * 8 + half * 4) =
          f32x4_t{acc[i][g * 4], acc[i][g * 4 + 1], acc[i][g * 4 + 2], acc[i][g * 4 + 3]};
  if (half == 0) p.part_ml[pr] = make_float2(m_run, l);
}

// ---------------------------------------------------------------------------
// thin form: at most 16 NC rows, each wave streams tiles of its own
// ---------------------------------------------------------------------------
template <int D, bool SC, int NC, int WAVES>
struct ThinLds {
  union {
    struct {
      uint8_t v[WAVES][kThinKeys * D * 2];
      float sc[WAVES][SC ? 2 * kThinKeys : 4];
    };
    float o[WAVES][NC * 16][D + 4];  // the waves' sums, joined at the end
  };
  float2 ml[WAVES][NC * 16];
};

template <int D, int CT, bool SC, int DU, int NC, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void window_thin_kernel(WindowParams p) {
  constexpr int THREADS = WAVES * 64;
  // (8-bit k-steps come in pairs: all of D)
  constexpr int EB = CT == kBf16 ? 2 : 1;
  constexpr int KSTEPS = (CT == kBf16 ? DU : D) / 32;
  constexpr int VE = 16 / EB;         // V elements per 16-byte load
  constexpr int DS = D / VE;          // lanes per V row
  constexpr int TL = 64 / DS;         // V rows per load
  constexpr int NV = kThinKeys / TL;  // V loads per tile
  static_assert(TL <= 16, "a V load's rows lie in one 16-key group");
  // K: bf16 k-step ks of lane group kg holds channels 32 ks + 8 kg; 8-bit
  // k-steps 2u and 2u + 1 channels 64 u + 16 kg and + 8 (one 16-byte load)
  constexpr int NK = CT == kBf16 ? KSTEPS : KSTEPS / 2;  // K loads per 16 keys
  constexpr int ROWB = D * 2;
  constexpr int VNCH = D / 8;
  constexpr int DB16 = DU / 16;
  __shared__ __attribute__((aligned(1024))) ThinLds<D, SC, NC, WAVES> lds;

  const int wave = readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 15;
  const int kg = lane >> 4;
  lds_u8_t *const vw = (lds_u8_t *)&lds.v[wave][0];
  lds_f32_t *const sw = (lds_f32_t *)&lds.sc[wave][0];

  Work wk;
  wk.set(p);
  wk.clear_rest(p);
  Tiles tl;
  if (!tl.set<kThinKeys>(p, wk.i, 0, NC * 16)) return;
  // the piece's tiles, which the waves take in turn
  const int2 share = wk.share(p, tl.n);
  const int x0 = share.x, x1 = share.y;

  auto k_chan = [](int j, int g) { return CT == kBf16 ? j * 32 + g * 8 : j * 64 + g * 16; };
  const int vds = lane % DS, vtl = lane / DS;
  // A tile's loads are in flight while the tile before is computed.  (Two tiles
  // ahead take registers that cost a resident workgroup: 128 x 528 int8 keys,
  // d = 64, 24.6 against 22.6 us, bf16 37 against 31.)
  struct Slot {
    u32x4_t k[2][NK], v[NV];
    float s;
    Group g[2];
    int ent[2];  // the table entries of the tile behind
  } slot;
  // bytes of a lane's chunks in a row; past the head dim the first chunk: K is
  // cleared at its use, what V gives there is stored nowhere
  uint32_t kch[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j)
    kch[j] = (k_chan(j, kg) < p.d ? k_chan(j, kg) * EB : 0) + (uint32_t)col * p.kc_t;
  const uint32_t vch = vds * VE < p.d ? vds * 16 : 0;
  const bool narrow = p.d < D;
  Keys keys;
  keys.set(p, wk.i, wk.h);
  auto load_entries = [&](Slot &t, int x) {
    t.ent[0] = keys.entry(p, tl.key(2 * x));
    t.ent[1] = keys.entry(p, tl.key(2 * x + 1));
  };
  // the places of tile x (its entries are loaded), and the entries of the tile
  // behind
  auto locate = [&](Slot &t, int x) {
    t.g[0].set(p, keys, tl.key(2 * x), t.ent[0]);
    t.g[1].set(p, keys, tl.key(2 * x + 1), t.ent[1]);
    if (x + WAVES < x1) load_entries(t, x + WAVES);
  };
  auto load_k = [&](Slot &t) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < NK; ++j)
        t.k[b][j] = *reinterpret_cast<const u32x4_t *>(t.g[b].k + kch[j]);
  };
  auto load_v = [&](Slot &t) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      t.v[j] = *reinterpret_cast<const u32x4_t *>(
          t.g[j * TL / 16].v + ((uint32_t)(j * TL % 16 + vtl) * p.vc_t + vch));
  };
  // lane l: scale of key l (K), of key l - 32 (V)
  auto load_s = [&](Slot &t) {
    if constexpr (SC) {
      const int k = lane & 31;
      const bool up = k >= 16;
      const float *ks = up ? t.g[1].ks(p, keys) : t.g[0].ks(p, keys);
      const float *vs = up ? t.g[1].vs(p, keys) : t.g[0].vs(p, keys);
      const float *sp = lane < 32 ? ks : vs;
      t.s = sp[(uint64_t)(k & 15) * (lane < 32 ? p.ks_t : p.vs_t)];
    }
  };

  // ---- the rows
  uint32_t neg;
  const float c2 = score_factor(p, wk.h, neg);
  bf16x8_t qf[NC][KSTEPS];
  f32x4_t acc[NC][DB16];
  float m_run[NC], l_run[NC];
  int pos[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int r = n * 16 + col;
    const bool ok = r < tl.rows;
    const int j = (int)fdiv((uint32_t)(ok ? r : 0), p.g_div);
    const int hq = wk.h * p.G + (ok ? r - j * p.G : 0);
    const uint16_t *qp = p.q + (int64_t)(tl.tok0 + j) * p.qs_t + (int64_t)hq * p.qs_h;
    pos[n] = tl.pos0 + j;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const int d0 = CT == kBf16 ? k_chan(ks, kg) : k_chan(ks >> 1, kg) + (ks & 1) * 8;
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (ok && d0 < p.d) w = *reinterpret_cast<const u32x4_t *>(qp + d0);
      qf[n][ks] = __builtin_bit_cast(bf16x8_t, w ^ u32x4_t{neg, neg, neg, neg});
    }
#pragma unroll
    for (int i = 0; i < DB16; ++i) acc[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[n] = -INFINITY;
    l_run[n] = 0.f;
  }

  // V^T operand of 16 channels: k index j of lane group kg is key 4 kg + j
  // (j < 4), 16 + 4 kg + j - 4 (else), the keys whose scores the lane holds;
  // source lane s of a 16-lane group addresses key 4 kg + s/4, channels 4 (s%4)
  const int tr_s = lane & 15;
  const int tr_row = 4 * kg + (tr_s >> 2);
  const int tr_x = tr_row & (VNCH - 1);

  f32x4_t s[NC][2];
  // (the conversions of codes stay behind this: drawn to the loads, over the
  // loop's edge, four registers would be held for each)
  auto here = [](u32x4_t &x) {
    if constexpr (CT == kI8) asm volatile("" : "+v"(x));
  };
  auto scores = [&](Slot &t) {
    auto &kr = t.k;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < NK; ++j) here(kr[b][j]);
    if (narrow) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < NK; ++j)
          if (k_chan(j, kg) >= p.d) kr[b][j] = u32x4_t{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < NC; ++n) s[n][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        u32x4_t w;
        if constexpr (CT == kBf16) w = kr[b][ks];
        else w = widen8<CT>(kr[b][ks >> 1][(ks & 1) * 2], kr[b][ks >> 1][(ks & 1) * 2 + 1]);
#pragma unroll
        for (int n = 0; n < NC; ++n)
          s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w),
                                                            qf[n][ks], s[n][b], 0, 0, 0);
        if constexpr (CT == kI8) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto store_v = [&](Slot &sl, const int (&k0)[2], bool whole) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int t = j * TL + vtl;
      here(sl.v[j]);
      // values that no row sees are cleared: 0 * NaN would reach the sums
      const u32x4_t v =
          whole || tl.any(k0[j * TL / 16] + (t & 15), p.first) ? sl.v[j] : u32x4_t{0u, 0u, 0u, 0u};
      if constexpr (CT == kBf16) {
        *(lds_u32x4_t *)(vw + t * ROWB + ((vds ^ (t & (VNCH - 1))) << 4)) = v;
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *(lds_u32x4_t *)(vw + t * ROWB + (((2 * vds + x) ^ (t & (VNCH - 1))) << 4)) =
              widen8<CT>(v[2 * x], v[2 * x + 1]);
        if constexpr (CT == kI8) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // probabilities as the sum of two bf16 values (2^-17 of each is left): the
  // products are few beside the keys' bytes, and one alone would be the largest
  // error of the output but its own rounding
  u32x4_t pk[NC], pl[NC];
  auto softmax = [&](const int (&k0)[2], bool whole) {
    f32x4_t ks4[2], vs4[2];
    if constexpr (SC) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        ks4[b] = *(const lds_f32x4_t *)(sw + b * 16 + kg * 4);
        vs4[b] = *(const lds_f32x4_t *)(sw + 32 + b * 16 + kg * 4);
      }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if constexpr (SC) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][b][i] *= ks4[b][i];
      }
      if (!whole) {
        const uint32_t hid = (hidden<16, 4>(p, pos[n], k0[0] + kg * 4) & 15u) |
                             hidden<16, 4>(p, pos[n], k0[1] + kg * 4) << 4;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][b][i] = hide(s[n][b][i], hid, b * 4 + i);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[n][b][i]);
      mx = max32(max16(mx)) * c2;
      const bool bump = mx > m_run[n] + 8.f || (m_run[n] == -INFINITY && mx > -INFINITY);
      if (__builtin_amdgcn_ballot_w64(bump)) {
        const float m_new = bump ? mx : m_run[n];
        const float alpha =
            m_run[n] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
        m_run[n] = m_new;
        l_run[n] *= alpha;
#pragma unroll
        for (int i = 0; i < DB16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][i][e] *= alpha;
      }
      const float nm = m_run[n] == -INFINITY ? 0.f : -m_run[n];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[i] = __builtin_amdgcn_exp2f(fmaf(s[n][b][i], c2, nm));
          l_run[n] += pr[i];
          if constexpr (SC) pr[i] *= vs4[b][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w = pack2_bf16(pr[2 * i], pr[2 * i + 1]);
          pk[n][2 * b + i] = w;
          pl[n][2 * b + i] = pack2_bf16(pr[2 * i] - bf16lo(w), pr[2 * i + 1] - bf16hi(w));
        }
      }
    }
  };
  auto values = [&]() {
#pragma unroll
    for (int blk = 0; blk < DB16; ++blk) {
      const uint32_t off = tr_row * ROWB + (((blk * 2 + ((tr_s >> 1) & 1)) ^ tr_x) << 4) +
                           ((tr_s & 1) << 3);
      // row + 16 has the same swizzle (VNCH divides 16)
      const u32x2_t t0 = __builtin_bit_cast(
          u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vw + off)));
      const u32x2_t t1 = __builtin_bit_cast(
          u32x2_t,
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vw + off + 16 * ROWB)));
      const u32x4_t v = {t0[0], t0[1], t1[0], t1[1]};
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        acc[n][blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, pk[n]), acc[n][blk], 0,
            0, 0);
        acc[n][blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, pl[n]), acc[n][blk], 0,
            0, 0);
      }
    }
  };

  // ---- the stream: K (V) of the next tile is issued once this tile's
  // product (copy to LDS) has freed the registers
  int x = x0 + wave;
  if (x < x1) {
    load_entries(slot, x);
    locate(slot, x);
    load_k(slot);
    load_s(slot);
    load_v(slot);
  }
  for (; x < x1; x += WAVES) {
    const int k0[2] = {tl.key(2 * x), tl.key(2 * x + 1)};
    const bool whole = see_all(p, tl.p_lo, tl.p_hi, k0[0], k0[0] + 16) &&
                       see_all(p, tl.p_lo, tl.p_hi, k0[1], k0[1] + 16);
    const bool go = x + WAVES < x1;
    if (go) locate(slot, x + WAVES);
    scores(slot);
    if constexpr (SC) {
      const int k = (lane & 16 ? k0[1] : k0[0]) + (lane & 15);
      sw[lane] = whole || tl.any(k, p.first) ? slot.s : 0.f;
    }
    if (go) {
      load_k(slot);
      load_s(slot);
    }
    softmax(k0, whole);
    store_v(slot, k0, whole);
    if (go) load_v(slot);
    values();
  }

  // ---- the waves' sums joined, thread -> rows and four channels
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float l = sum32(sum16(l_run[n]));
#pragma unroll
    for (int i = 0; i < DB16; ++i)
      *reinterpret_cast<f32x4_t *>(&lds.o[wave][n * 16 + col][i * 16 + kg * 4]) = acc[n][i];
    if (kg == 0) lds.ml[wave][n * 16 + col] = make_float2(m_run[n], l);
  }
  __syncthreads();
  constexpr int C4 = D / 4;
  const int c = threadIdx.x % C4 * 4;
  if (c >= p.d) return;
#pragma unroll
  for (int k = 0; k < (NC * 16 * C4 + THREADS - 1) / THREADS; ++k) {
    const int r = k * (THREADS / C4) + (int)threadIdx.x / C4;
    if (r >= tl.rows) return;
    float m = -INFINITY, l = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(&lds.o[w][r][c]);
      add_piece(m, l, o, lds.ml[w][r].x, lds.ml[w][r].y, v);
    }
    if (p.split > 1) {
      const int64_t pr = wk.piece * p.part_rows + r;
      *reinterpret_cast<f32x4_t *>(p.part_o + pr * D + c) = o;
      if (c == 0) p.part_ml[pr] = make_float2(m, l);
      continue;
    }
    const int j = (int)fdiv((uint32_t)r, p.g_div);
    const int hq = wk.h * p.G + r - j * p.G;
    const float f = row_factor(p, wk.h, hq, m, l);
    *reinterpret_cast<u32x2_t *>(p.out + (int64_t)(tl.tok0 + j) * p.os_t +
                                 (int64_t)hq * p.os_h + c) =
        u32x2_t{pack2_bf16(o[0] * f, o[1] * f), pack2_bf16(o[2] * f, o[3] * f)};
  }
}

// ---------------------------------------------------------------------------
// join of the pieces: D / 4 lanes per row
// ---------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(256) void window_join_kernel(WindowParams p, int tile_rows) {
  constexpr int C4 = D / 4, RPB = 256 / C4;
  const int c = threadIdx.x % C4 * 4;
  // workgroup -> (row tile of a sequence and head, rows)
  const int per = (p.part_rows + RPB - 1) / RPB;
  int id = blockIdx.x / per;
  const int rloc = (blockIdx.x % per) * RPB + (int)threadIdx.x / C4;
  const int64_t piece0 = (int64_t)id * p.split;
  const int rt = id % p.rt_max;
  id /= p.rt_max;
  const int i = id % p.n_seq, h = id / p.n_seq;
  int a = i, b = i + 1;
  if (p.cu) {
    a = min(max(scalar_load(p.cu, i), 0), p.num_tokens);
    b = min(max(scalar_load(p.cu, i + 1), a), p.num_tokens);
  }
  const int r = rt * tile_rows + rloc;
  if (rloc >= p.part_rows || r >= min(b - a, p.tok_max) * p.G || c >= p.d) return;
  float m = -INFINITY, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < p.split; s0 += 4) {
    float2 ml[4];
    f32x4_t v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t pr = (piece0 + min(s0 + u, p.split - 1)) * p.part_rows + rloc;
      ml[u] = p.part_ml[pr];
      v[u] = *reinterpret_cast<const f32x4_t *>(p.part_o + pr * D + c);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + u < p.split) add_piece(m, l, o, ml[u].x, ml[u].y, v[u]);
  }
  const int j = (int)fdiv((uint32_t)r, p.g_div);
  const int hq = h * p.G + r - j * p.G;
  const float f = row_factor(p, h, hq, m, l);
  *reinterpret_cast<u32x2_t *>(p.out + (int64_t)(a + j) * p.os_t + (int64_t)hq * p.os_h + c) =
      u32x2_t{pack2_bf16(o[0] * f, o[1] * f), pack2_bf16(o[2] * f, o[3] * f)};
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

struct Plan {
  bool thin;
  int tile_rows;  // rows of a workgroup
  int waves;      // of a thin workgroup
  int64_t blocks;
  size_t o, total;  // byte offset of the sums, size
};

Plan plan_window(WindowParams &p) {
  Plan w;
  const int D = p.d <= 64 ? 64 : 128;
  const int64_t seq_rows = (int64_t)p.tok_max * p.G;
  w.thin = seq_rows <= 32;
  const int tile_rows = w.tile_rows = seq_rows <= 16 ? 16 : seq_rows <= 32 ? 32 : kRows;
  p.rt_max = (int)((seq_rows + tile_rows - 1) / tile_rows);
  p.part_rows = (int)std::min<int64_t>(seq_rows, tile_rows);
  // tiles of a row tile at most, row tiles that have rows at most
  const int T = w.thin ? kThinKeys : kTallKeys;
  const int64_t span = (int64_t)p.window + tile_rows / p.G + 1;
  const int64_t tiles =
      std::min<int64_t>((p.cap + T - 1) / T, ((p.first + 15) / 16 + (span + 30) / 16) * 16 / T + 1);
  const int64_t busy =
      std::min<int64_t>((int64_t)p.n_seq * p.rt_max,
                        (int64_t)p.num_tokens * p.G / tile_rows + p.n_seq) * p.Hkv;
  // Thin workgroups of eight waves where every CU has one at most (and there is more
  // than a tile for each of four): half the tiles one after the other.  us at 1024
  // keys, d = 128, bf16, 4 / 8 waves: 256 workgroups 32.5 / 28.9, int8 22.7 / 18.6;
  // 320 workgroups 41.0 / 43.8, 512 52.3 / 54.9.
  w.waves = w.thin && busy <= cu_count() && tiles > 4 ? 8 : 4;
  // Keys are cut where workgroups are few, to pieces of `least` tiles at least.  A
  // cut costs a second launch (2 us, 4 of host time where calls are not captured),
  // which up to 40 tiles at d = 64 (20 at 128) it does not earn back: us uncut / cut,
  // captured, bf16, 4 x 8 heads, d = 64: 512 keys 7.4 / 8.5, 1024 10.6 / 10.3, 2048
  // 15.4 / 12.1; 16 x 8 heads: 1024 11.1 / 13.0, 2048 17.2 / 17.9; d = 128, 8 x 8
  // heads: 512 11.2 / 12.0, 1024 15.9 / 14.0.
  const int64_t slots = (int64_t)cu_count() * 8 / w.waves;
  const int64_t least = w.thin ? 8 : 6;
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>({slots / busy, tiles / least, 32}));
  if (w.waves == 8 && tiles * D <= 40 * 64) p.split = 1;
  // (slots for partials are by the longest sequence: many short ones beside it
  // would take gigabytes that nothing writes)
  const int64_t tiles_all = (int64_t)p.n_seq * p.rt_max * p.Hkv;
  const int64_t piece = (int64_t)p.part_rows * (D * 4 + 8);
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>(p.split, (128 << 20) / (tiles_all * piece)));
  w.blocks = tiles_all * p.split;
  p.rt_div = make_fastdiv(p.rt_max);
  p.split_div = make_fastdiv(p.split);
  p.seq_div = make_fastdiv(p.n_seq);
  w.o = w.total = 0;
  if (p.split > 1) {
    w.o = (size_t)up(w.blocks * p.part_rows * 8, 256);
    w.total = w.o + (size_t)w.blocks * p.part_rows * D * 4;
  }
  return w;
}

WindowParams window_params(const mia_window_args &a) {
  WindowParams p = {};
  const int eb = a.cache_dtype == MIA_DTYPE_BF16 ? 2 : 1;
  p.q = (const uint16_t *)a.q, p.out = (uint16_t *)a.out;
  p.qs_t = a.q_stride[0], p.qs_h = a.q_stride[1];
  p.os_t = a.out_stride[0], p.os_h = a.out_stride[1];
  p.num_tokens = a.num_tokens, p.n_seq = a.num_seqs;
  p.cu = a.cu_seqlens_q, p.len = a.seq_lens;
  p.zero_rest = a.zero_rest;
  p.tok_max = a.cu_seqlens_q ? std::min(a.max_seqlen_q, a.num_tokens) : 1;
  p.cap = a.blocks_per_seq * a.block_size;
  p.window = a.window, p.first = a.first_tokens;
  p.G = a.num_q_heads / a.num_kv_heads, p.Hkv = a.num_kv_heads, p.d = a.head_dim;
  p.g_div = make_fastdiv(p.G);
  p.bt = a.block_table, p.bt_s = a.bt_stride[0], p.bt_j = a.bt_stride[1];
  p.k_cache = (const uint8_t *)a.k_cache, p.v_cache = (const uint8_t *)a.v_cache;
  p.kc_blk16 = (uint32_t)(a.k_cache_stride[0] * eb / 16);
  p.vc_blk16 = (uint32_t)(a.v_cache_stride[0] * eb / 16);
  p.kc_h = a.k_cache_stride[1] * eb, p.kc_t = (uint32_t)(a.k_cache_stride[2] * eb);
  p.vc_h = a.v_cache_stride[1] * eb, p.vc_t = (uint32_t)(a.v_cache_stride[2] * eb);
  p.k_sc = a.k_scales, p.v_sc = a.v_scales;
  p.ks_blk = (uint32_t)a.k_scale_stride[0], p.ks_t = (uint32_t)a.k_scale_stride[2];
  p.vs_blk = (uint32_t)a.v_scale_stride[0], p.vs_t = (uint32_t)a.v_scale_stride[2];
  p.ks_h = a.k_scale_stride[1], p.vs_h = a.v_scale_stride[1];
  p.k_deq = a.k_dequant, p.v_deq = a.v_dequant;
  p.sink = a.sink;
  p.nb = a.num_blocks, p.bs = a.block_size;
  p.bs_div = make_fastdiv(a.block_size);
  p.scale_log2 = a.softmax_scale * kLog2e;
  return p;
}

template <int D, int CT, bool SC, int DU, int NC>
void launch_thin(const WindowParams &p, const Plan &w, hipStream_t s) {
  const unsigned n = (unsigned)w.blocks;
  if (w.waves == 8) window_thin_kernel<D, CT, SC, DU, NC, 8><<<n, 512, 0, s>>>(p);
  else window_thin_kernel<D, CT, SC, DU, NC, 4><<<n, 256, 0, s>>>(p);
}

template <int D, int CT, bool SC, int DU>
void launch_form(const WindowParams &p, const Plan &w, hipStream_t s) {
  if (!w.thin) window_tall_kernel<D, CT, SC, DU><<<(unsigned)w.blocks, kThreads, 0, s>>>(p);
  else if (w.tile_rows == 16) launch_thin<D, CT, SC, DU, 1>(p, w, s);
  else launch_thin<D, CT, SC, DU, 2>(p, w, s);
}

template <int D, int DU>
void launch_cache(const WindowParams &p, const Plan &w, int dtype, hipStream_t s) {
  if (dtype == MIA_DTYPE_BF16) launch_form<D, kBf16, false, DU>(p, w, s);
  else if (dtype == MIA_DTYPE_I8) launch_form<D, kI8, true, DU>(p, w, s);
  else if (p.k_sc) launch_form<D, kFp8, true, DU>(p, w, s);
  else launch_form<D, kFp8, false, DU>(p, w, s);
}

}  // namespace

size_t window_workspace(const mia_window_args &a) {
  WindowParams p = window_params(a);
  return plan_window(p).total;
}

int launch_window(const mia_window_args &a, hipStream_t s) {
  WindowParams p = window_params(a);
  const Plan w = plan_window(p);
  p.part_ml = (float2 *)a.workspace;
  p.part_o = (float *)((uint8_t *)a.workspace + w.o);
  if (p.d <= 64) launch_cache<64, 64>(p, w, a.cache_dtype, s);
  else if (p.d <= 96) launch_cache<128, 96>(p, w, a.cache_dtype, s);
  else launch_cache<128, 128>(p, w, a.cache_dtype, s);
  if (p.split > 1) {
    const int D = p.d <= 64 ? 64 : 128, rpb = 256 / (D / 4);
    const unsigned n = (unsigned)(w.blocks / p.split * ((p.part_rows + rpb - 1) / rpb));
    if (D == 64) window_join_kernel<64><<<n, 256, 0, s>>>(p, w.tile_rows);
    else window_join_kernel<128><<<n, 256, 0, s>>>(p, w.tile_rows);
  }
  return check_hip(hipGetLastError(), "window_attention");
}

}  // namespace mia
