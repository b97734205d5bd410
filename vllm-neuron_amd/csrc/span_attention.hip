// span_attention.hip — attention of query rows over spans of keys of another
// length, bf16 MFMA on gfx950: cross attention (ragged queries over ragged
// encoder keys) and decode attention of a batch that shares a long prefix
// (one span for all rows, and each row's own span).
//
// Mathematics.  Every row of a (sequence, kv head) sees every key of its
// span: out = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m), s_k = scale q.k_k,
// accumulated tile by tile with a running maximum m and sum l in fp32.  Spans
// of the same row are joined by their (m, l, o).  Codes of a quantised cache
// are exact in bf16, so they go to the MFMA as they are: the scale of a key
// multiplies its score, the scale of its value the probability.
//
// Rows.  The query rows of one kv head are packed GQA-first: row r = pos * G
// + g is query token `pos` and q head h * G + g.
//
// Two forms of a tile, chosen by the rows that share a span (list.thin):
//   tall  a workgroup takes 128 rows, 32 per wave; 64-key tiles of K and V go
//         through LDS and serve all four waves (v_mfma_f32_32x32x16_bf16).
//         Bound by the MFMAs and exponentials.  K and V of the next tile arrive
//         in the other of two LDS stages meanwhile.  2048 tokens of 32 heads
//         over 6404 keys, d = 128: 205-216 us by card, 1.0-1.05 PFLOP/s; the
//         matrix units are busy 53 % of the cycles, vector instructions issue
//         in 50 %, at a clock that falls to 1.9 GHz.
//   thin  at most 16 or 32 rows: each wave streams 32-key tiles of its own, K
//         straight into MFMA operands, V through a piece of LDS of the wave
//         (v_mfma_f32_16x16x32_bf16).  Bound by HBM behind a start of 7 us
//         (launch, plan, table, first keys): one token of 16 heads each over
//         32 x 100-1500 keys, d = 64 (106 MB) 25 us, 4.2 TB/s, 6 without the
//         start.
// Both compute S^T = K Q^T and O^T = V^T P^T, so a lane holds scores of one
// row, and its probabilities are the second product's operand as they are.
//
// Work split.  The tiles of all segments ((sequence, kv head, row tile)) of
// a form are laid end to end and cut into equal shares, one per workgroup
// (tall) or wave (thin), whatever the lengths: every workgroup computes its
// share from the lengths on the device (a block scan, 3 us), so a captured
// call follows its tensors.  A share begins and ends inside a segment; pieces
// of cut segments go to the workspace as fp32 (o, m, l) and a second kernel
// joins them.  A call with both forms (shared prefix) gives them workgroups in
// proportion to their tiles' costs, side by side in one launch: the prefix's
// products run beside the own spans' HBM streams.
#include <algorithm>

#include "attn_tile.h"

namespace mia {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = 128;    // query rows of a tall segment (4 waves x 32)
constexpr int kTallKeys = 64;  // keys per tall tile
constexpr int kThinKeys = 32;  // keys per thin tile
// Tall: operand fragments read from LDS ahead of their product.  Left alone
// the compiler reads each right before it: 2048 tokens of 32 heads over 6404
// keys (d = 128) 246 us, 230 with 2 or 3 ahead.
constexpr int kAhead = 2;
// Tall waves issue their products at a lower priority than the rest, so that
// of a SIMD's two waves the one in its softmax is not held up by the other's
// products: the same call, eager on one card, 220 us at one priority, 211 with
// the products above the rest and 210 with them below.

// One list of sequences and their key spans.
struct SpanList {
  int n;              // sequences
  int thin;           // form of its tiles
  const int32_t *cu;  // [n + 1] first query tokens, or NULL: tok_per each
  int tok_per;
  int tok_max;        // query tokens of a sequence at most
  const int32_t *len; // [n] keys
  int len_sub;        // subtracted from len
  int len_cap;        // keys the table (or the dense rows) can hold
  const int32_t *bt;  // block table, or NULL: block = sequence
  int64_t bt_s, bt_j;
  int part_rows;      // rows of a partial
  int64_t part0;      // first partial row
};

struct SpanParams {
  const uint16_t *q;
  int64_t qs_b, qs_s, qs_h;  // token t: b = t / S, s = t % S
  uint16_t *out;
  int64_t os_b, os_s, os_h;
  FastDiv s_div, g_div;
  int num_tokens, S;
  int G, Hkv, d;
  const uint8_t *k_cache, *v_cache;
  uint32_t kc_blk16, vc_blk16;       // block strides in 16-byte units
  int64_t kc_h, kc_t, vc_h, vc_t;    // bytes
  const float *k_sc, *v_sc;  // per-key scales or NULL
  uint32_t ks_blk, ks_t, vs_blk, vs_t;  // elements
  int64_t ks_h, vs_h;
  const float *k_deq, *v_deq;  // per-head scales or NULL
  const float *sink;
  int nb, bs;
  FastDiv bs_div;
  float scale_log2;
  SpanList list[2];
  int join;        // every piece goes to the workspace (rows have several spans)
  int zero_rest;   // cross attention: rows that nothing computes are cleared
  float cost[2];   // time of a tall tile per workgroup, of a thin one per wave
  int over[2];     // cost of a segment's start in tiles (stores, query rows, table)
  int least[2];    // units of a share at least
  int *hdr;        // see plan()
  float *part_o;   // [partial row][D]
  float2 *part_ml; // [partial row]
};

// The launch's parameters (the first kernel argument) read anew from the
// kernel's argument segment: what a piece's start or end needs is not kept in
// scalar registers through the tile loops (kept, the 128-wide kernels
// spilled over 100 of them to scratch).
MIA_DEV const SpanParams &fresh() {
  auto *k = (const __attribute__((address_space(4))) SpanParams *)
      __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  return *(const SpanParams *)k;
}

MIA_DEV int list_len(const SpanList &l, int i) {
  const int n = scalar_load(l.len, i);  // (any int32: no difference below zero)
  return n > l.len_sub ? min(n - l.len_sub, l.len_cap) : 0;
}
// first query token and token count of sequence i
MIA_DEV int2 list_tokens(const SpanList &l, int i, int num_tokens) {
  int a, b;
  if (l.cu) {
    a = min(max(scalar_load(l.cu, i), 0), num_tokens);
    b = min(max(scalar_load(l.cu, i + 1), a), num_tokens);
  } else {
    a = min(i * l.tok_per, num_tokens);
    b = min(a + l.tok_per, num_tokens);
  }
  return make_int2(a, min(b - a, l.tok_max));
}
MIA_DEV int row_tiles(const SpanList &l, int rows) {
  return l.thin ? (rows > 0) : (rows + kRows - 1) / kRows;
}
MIA_DEV int key_tiles(const SpanList &l, int len) {
  return l.thin ? (len + kThinKeys - 1) / kThinKeys : (len + kTallKeys - 1) / kTallKeys;
}

// A form's segments laid end to end: `over` units for the start of a segment,
// then one per tile.  N units are cut into W shares: the first `rem` hold
// base + 1, the others base.
struct Cut {
  int base, rem;
};
MIA_DEV int cut_start(Cut c, int w) { return w * c.base + min(w, c.rem); }
MIA_DEV int cut_of(Cut c, int x) {  // the share that holds unit x
  const int head = c.rem * (c.base + 1);
  return x < head ? x / (c.base + 1) : c.rem + (x - head) / c.base;
}

// Workspace header.  Joined calls: [0..3] the cuts of both forms, [8 + u] the
// first unit of joined sequence u in its form's stream.  Cross attention: 8
// ints per share: pieces of the cut segment that starts in it (0: none), its
// first query token, rows, row tile, head.
constexpr int kHdr = 8;

// Where a share starts.
struct Share {
  Cut cut;
  int w;       // number of the share
  int x0, x1;  // its units
  int u;       // sequence of unit x0
  int xu;      // first unit of that sequence
  int len, tok0, rows;  // its keys, first query token and rows
};

struct PlanLds {
  int tot[2][kWaves];
  int seq[kWaves], first[kWaves], len[kWaves], tok0[kWaves], rows[kWaves];
};

// Inclusive scan over the wave: shifts inside rows of 16 lanes, then the row
// totals broadcast (DPP: a few cycles a step, where a shuffle through LDS
// takes over a hundred).
MIA_DEV int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Zeros in the output rows of tokens [t0, t1); a wave calls it.
MIA_DEV void zero_rows(const SpanParams &p, int t0, int t1) {
  const int lane = threadIdx.x & 63;
  const int c8 = p.d / 8, heads = 64 / c8;  // 16-byte chunks of a head, heads at once
  const int h0 = lane / c8, c = lane - h0 * c8;
  for (int t = t0; t < t1; ++t) {
    const int b = (int)fdiv((uint32_t)t, p.s_div);
    uint16_t *op = p.out + (int64_t)b * p.os_b + (int64_t)(t - b * p.S) * p.os_s + c * 8;
    if (h0 < heads)
      for (int h = h0; h < p.Hkv * p.G; h += heads) {
        u32x2_t *x = reinterpret_cast<u32x2_t *>(op + (int64_t)h * p.os_h);
        x[0] = u32x2_t{0u, 0u};
        x[1] = u32x2_t{0u, 0u};
      }
  }
}

// The plan of a launch, in every workgroup: a block scan of the sequences'
// tiles (each thread a contiguous run of the joined lists), the workgroups of
// each form, and this workgroup's (tall) or wave's (thin) share.  Returns 0
// for a tall share, 1 for a thin one, -1 for none; uniform in the workgroup (a
// share may hold no tile).
MIA_DEV int plan(const SpanParams &p, PlanLds &lds, Share &sh) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = readfirstlane(tid >> 6);
  const int grid = gridDim.x;
  const int b = blockIdx.x;
  const int n0 = p.list[0].n;
  const int n_seq = n0 + p.list[1].n;
  const int per = (n_seq + kThreads - 1) / kThreads;
  const int u0 = min(tid * per, n_seq), u1 = min(u0 + per, n_seq);
  struct Seq {
    int thin, len, tok0, rows, units;
  };
  auto seq_of = [&](int u) {
    const int li = u < n0 ? 0 : 1;
    const SpanList &l = p.list[li];
    const int i = li ? u - n0 : u;
    const int2 tk = list_tokens(l, i, p.num_tokens);
    Seq q;
    q.thin = l.thin;
    q.len = list_len(l, i);
    q.tok0 = tk.x;
    q.rows = tk.y * p.G;
    const int kt = key_tiles(l, q.len);
    q.units = kt ? (kt + p.over[l.thin]) * row_tiles(l, q.rows) * p.Hkv : 0;
    return q;
  };
  // This workgroup's part of tokens [x, y): equal runs over the launch, from
  // workgroup `at` (below grid) on.
  auto part = [&](int x, int y, int at) {
    const int n = max(y - x, 0);
    const int each = n <= grid ? 1 : (n + grid - 1) / grid;
    const int k = b < at ? b - at + grid : b - at;
    return make_int2(x + min(k * each, n), x + min((k + 1) * each, n));
  };
  // The tokens of sequence u that it clears (cross attention): those of a
  // sequence without any key and, with zero_rest, those up to the next sequence
  // that nothing computes.
  auto cleared = [&](int u, int at, const Seq &q) {
    int2 t = {0, 0};
    if (p.join) return t;
    const SpanList &l = p.list[1];
    const int i = u - n0;
    t.y = q.tok0 + (int)fdiv((uint32_t)q.rows, p.g_div);
    t.x = q.len == 0 ? q.tok0 : t.y;
    if (p.zero_rest) {
      if (i == l.n - 1) t.y = p.num_tokens;
      else if (l.cu) t.y = min(max(scalar_load(l.cu, i + 1), t.y), p.num_tokens);
    }
    return t.x < t.y ? part(t.x, t.y, at) : t;
  };
  // (calls of up to 256 sequences: one per thread, kept)
  Seq mine = {0, 0, 0, 0, 0};
  int sum[2] = {0, 0};
  int2 zero = {0, 0};  // tokens to be cleared, of the last such sequence
  bool more = false, bad = false;
  int at = u0 < grid ? u0 : u0 % grid;
#pragma nounroll
  for (int u = u0; u < u1; ++u) {
    mine = seq_of(u);
    if (u >= n0 && p.list[1].cu) {
      const int32_t *cu = p.list[1].cu + (u - n0);
      bad |= scalar_load(cu, 1) < scalar_load(cu, 0);
    }
    sum[0] += mine.thin ? 0 : mine.units;
    sum[1] += mine.thin ? mine.units : 0;
    const int2 t = cleared(u, at, mine);
    if (t.x < t.y) {
      more |= zero.x < zero.y;
      zero = t;
    }
    at = at + 1 == grid ? 0 : at + 1;
  }
  // (first tokens that decrease would let sequences share tokens: more units
  // than the host counted, rows written twice; the call then has no tiles)
  bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  int inc[2], n[2], base[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    inc[f] = wave_scan(sum[f]);
    if (lane == 63) lds.tot[f][wave] = bad ? -1 : inc[f];
  }
  __syncthreads();
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    n[f] = 0;
    base[f] = inc[f] - sum[f];
    bad = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      base[f] += w < wave ? lds.tot[f][w] : 0;
      n[f] += lds.tot[f][w];
      bad |= lds.tot[f][w] < 0;
    }
    n[f] = bad ? 0 : readfirstlane(n[f]);
  }
  // workgroups of each form: in proportion to the costs, whole multiples of
  // the 8 XCDs where there are enough
  const int most_t = n[0] ? max(1, n[0] / p.least[0]) : 0;
  const int most_s = n[1] ? max(1, n[1] / (kWaves * p.least[1])) : 0;
  int wt = most_t, ws = most_s;
  if (wt + ws > grid) {
    const float ca = (float)n[0] * p.cost[0], cb = (float)n[1] * p.cost[1];
    const int share = readfirstlane((int)((float)grid * (ca / (ca + cb)) + 0.5f));
    wt = n[0] == 0 ? 0 : n[1] == 0 ? grid : min(min(max(share, 1), grid - 1), most_t);
    ws = n[1] == 0 ? 0 : min(grid - wt, most_s);
  }
  if (wt > 8) wt &= ~7;
  const int form = b < wt ? 0 : b < wt + ws ? 1 : -1;
  const int wv = ws * kWaves;
  Cut cut[2];
  cut[0].base = wt ? n[0] / wt : 0;
  cut[0].rem = n[0] - cut[0].base * wt;
  cut[1].base = wv ? n[1] / wv : 0;
  cut[1].rem = n[1] - cut[1].base * wv;
  const bool lists = p.join && b == 0;  // this workgroup writes the header
  if (lists && tid == 0) {
    p.hdr[0] = cut[0].base, p.hdr[1] = cut[0].rem;
    p.hdr[2] = cut[1].base, p.hdr[3] = cut[1].rem;
  }
  // workgroups go round-robin over the 8 XCDs: neighbouring tall shares (the
  // row tiles of one head over the same keys) stay on one XCD's L2
  const int w = form == 1 ? (b - wt) * kWaves
                : wt >= 8 && wt % 8 == 0 ? (b % 8) * (wt / 8) + b / 8 : b;
  if (!p.join && lane == 0) {
    // (one form only) no cut segment starts in a share unless it says so: the
    // header is cleared by the thread that may set it
    if (p.list[1].thin) p.hdr[kHdr * (b * kWaves + wave)] = 0;
    else if (wave == 0) p.hdr[kHdr * (form == 0 ? w : b)] = 0;
  }
  // the sequences of this workgroup's first units
  const Cut mycut = form == 1 ? cut[1] : cut[0];
  const int shares = form < 0 ? 0 : form == 1 ? kWaves : 1;
  const int x_lo = cut_start(mycut, w), x_hi = cut_start(mycut, w + shares);
  int x[2] = {base[0], base[1]};
  const bool find = form == 1 ? x_lo < x[1] + sum[1] && x_hi > x[1]
                              : form == 0 && x_lo < x[0] + sum[0] && x_hi > x[0];
  if (lists || find) {
#pragma nounroll
    for (int u = u0; u < u1; ++u) {
      const Seq q = per == 1 ? mine : seq_of(u);
      const int xu = q.thin ? x[1] : x[0];
      if (lists) p.hdr[kHdr + u] = xu;
      if (find && q.thin == form) {
#pragma nounroll
        for (int k = 0; k < shares; ++k) {
          const int xs = cut_start(mycut, w + k);
          if (xs < xu || xs >= xu + q.units) continue;
          lds.seq[k] = u;
          lds.first[k] = xu;
          lds.len[k] = q.len;
          lds.tok0[k] = q.tok0;
          lds.rows[k] = q.rows;
        }
      }
      x[0] += q.thin ? 0 : q.units;
      x[1] += q.thin ? q.units : 0;
    }
  }
  __syncthreads();
  // (2048 tokens of 32 heads, d = 128, beside 16 with keys: 32 us, by one
  // workgroup 705)
  auto clear = [&](int2 t) {
    uint64_t left = __builtin_amdgcn_ballot_w64(t.x < t.y);
    while (left) {
      const int src = __builtin_ctzll(left);
      left &= left - 1;
      zero_rows(p, __builtin_amdgcn_readlane(t.x, src), __builtin_amdgcn_readlane(t.y, src));
    }
  };
  if (p.zero_rest && wave == 0) {  // tokens before the first sequence, or all
    const int head = bad ? p.num_tokens
                         : p.list[1].cu ? min(max(scalar_load(p.list[1].cu, 0), 0), p.num_tokens) : 0;
    const int2 t = part(0, head, 0);
    if (t.x < t.y) zero_rows(p, t.x, t.y);
  }
  if (!bad) {
    clear(zero);
    if (__builtin_amdgcn_ballot_w64(more)) {  // (a thread of several sequences)
      at = u0 < grid ? u0 : u0 % grid;
#pragma nounroll
      for (int u = u0; u < u0 + per; ++u) {
        clear(u < u1 ? cleared(u, at, seq_of(u)) : int2{0, 0});
        at = at + 1 == grid ? 0 : at + 1;
      }
    }
  }
  if (form < 0) return -1;
  const int k = form == 1 ? wave : 0;
  sh.cut = mycut;
  sh.w = w + k;
  sh.x0 = cut_start(mycut, sh.w);
  sh.x1 = cut_start(mycut, sh.w + 1);
  sh.u = readfirstlane(lds.seq[k]);
  sh.xu = readfirstlane(lds.first[k]);
  sh.len = readfirstlane(lds.len[k]);
  sh.tok0 = readfirstlane(lds.tok0[k]);
  sh.rows = readfirstlane(lds.rows[k]);
  return form;
}

// A piece: consecutive tiles of one segment in a share (wave-uniform).
struct Piece {
  int li, i;          // list, sequence
  int tok0, rows;     // first query token, rows (tokens x G)
  int len, tiles;     // keys, tiles of the segment
  int rt_n, rt, h;    // row tiles, this one, kv head
  int t, n;           // its tiles [t, t + n)
  int x;              // unit of tile t
  int over;           // units before a segment's first tile
  MIA_DEV bool whole() const { return t == 0 && n == tiles; }
};

MIA_DEV void load_seq(const SpanParams &p, Piece &c) {
  const SpanList &l = p.list[c.li];
  const int2 tk = list_tokens(l, c.i, p.num_tokens);
  c.tok0 = readfirstlane(tk.x);
  c.rows = readfirstlane(tk.y * p.G);
  c.len = readfirstlane(list_len(l, c.i));
  c.tiles = key_tiles(l, c.len);
  c.rt_n = row_tiles(l, c.rows);
}

// The share's first piece; false if it has no tile.
MIA_DEV bool first_piece(const SpanParams &p, const Share &sh, Piece &c) {
  if (sh.x0 >= sh.x1) return false;
  c.li = sh.u < p.list[0].n ? 0 : 1;
  c.i = c.li ? sh.u - p.list[0].n : sh.u;
  const SpanList &l = p.list[c.li];
  c.len = sh.len;
  c.tok0 = sh.tok0;
  c.rows = sh.rows;
  c.tiles = key_tiles(l, c.len);
  c.rt_n = row_tiles(l, c.rows);
  c.over = p.over[l.thin];
  const int k = sh.x0 - sh.xu;  // unit of the sequence
  const int seg = k / (c.tiles + c.over);
  c.t = k - seg * (c.tiles + c.over) - c.over;
  c.x = sh.x0;
  if (c.t < 0) {  // among the units of a segment's start
    c.x -= c.t;
    c.t = 0;
  }
  c.h = seg / c.rt_n;
  c.rt = seg - c.h * c.rt_n;
  c.n = min(c.tiles - c.t, sh.x1 - c.x);
  return c.n > 0;
}

// To the piece behind c, over sequences without tiles and lists of the other
// form; false at the end of the share.
MIA_DEV bool next_piece(const SpanParams &p, const Share &sh, Piece &c) {
  if (c.t + c.n < c.tiles) return false;
  c.x += c.n + c.over;
  if (c.x >= sh.x1) return false;
  c.t = 0;
  if (++c.rt >= c.rt_n) {
    c.rt = 0;
    if (++c.h >= p.Hkv) {
      c.h = 0;
      const int form = p.list[c.li].thin;
      ++c.i;
      while (true) {
        if (c.i >= p.list[c.li].n || p.list[c.li].thin != form) {
          if (c.li == 1) return false;  // not reached while units are left
          c.li = 1;
          c.i = 0;
          continue;
        }
        load_seq(p, c);
        if (c.tiles > 0 && c.rt_n > 0) break;
        ++c.i;
      }
    }
  }
  c.n = min(c.tiles, sh.x1 - c.x);
  return true;
}

// Offset of token t (t = b * S + s).
MIA_DEV int64_t tok_off(const SpanParams &p, int t, int64_t sb, int64_t ss) {
  const int b = (int)fdiv((uint32_t)t, p.s_div);
  return (int64_t)b * sb + (int64_t)(t - b * p.S) * ss;
}

// Where a segment's keys lie (wave-uniform): its table row and the first byte
// of its head in K and V, the first scale of its head.
struct Keys {
  const int32_t *bt;  // NULL: dense, block = sequence
  int64_t bt_j;
  const uint8_t *k, *v;
  const float *ks, *vs;
  uint32_t k_blk, v_blk;    // block strides in 16-byte units
  uint32_t k_t, v_t;        // token strides in bytes (below 2^27)
  uint32_t ks_blk, vs_blk;  // scale strides in elements
  uint32_t ks_t, vs_t;
  int seq, len, nb, bs;
  FastDiv bs_div;

  template <bool SC>
  MIA_DEV void set(const SpanParams &p, const Piece &c) {
    const SpanList &l = p.list[c.li];
    bt = l.bt ? l.bt + (int64_t)c.i * l.bt_s : nullptr;
    bt_j = l.bt_j;
    k = p.k_cache + (int64_t)c.h * p.kc_h;
    v = p.v_cache + (int64_t)c.h * p.vc_h;
    k_blk = p.kc_blk16, v_blk = p.vc_blk16;
    k_t = (uint32_t)p.kc_t, v_t = (uint32_t)p.vc_t;
    if constexpr (SC) {
      ks = p.k_sc + (int64_t)c.h * p.ks_h;
      vs = p.v_sc + (int64_t)c.h * p.vs_h;
      ks_blk = p.ks_blk, vs_blk = p.vs_blk;
      ks_t = p.ks_t, vs_t = p.vs_t;
    }
    seq = c.i, len = c.len, nb = p.nb, bs = p.bs;
    bs_div = p.bs_div;
  }
  // The 16-key group of key k0 (k0 % 16 == 0), clamped into the span: its
  // first key and, loaded ahead of its use, its table entry.
  MIA_DEV int first(int k0) const { return min(k0, (len - 1) & ~15); }
  MIA_DEV int entry(int k0) const {
    return bt ? scalar_load(bt, (int64_t)fdiv((uint32_t)first(k0), bs_div) * bt_j) : seq;
  }
};

// A 16-key group: its first key, block, and first key inside the block.
struct Group {
  int k16;
  uint32_t blk, off;
  const uint8_t *k, *v;  // its first rows
  MIA_DEV void set(const Keys &s, int k0, int entry) {
    k16 = s.first(k0);
    blk = s.bt ? min(max(entry, 0), s.nb - 1) : s.seq;
    off = s.bt ? k16 - (int)fdiv((uint32_t)k16, s.bs_div) * s.bs : k16;
    k = s.k + (((uint64_t)blk * s.k_blk) << 4) + (uint64_t)off * s.k_t;
    v = s.v + (((uint64_t)blk * s.v_blk) << 4) + (uint64_t)off * s.v_t;
  }
  MIA_DEV const float *ks(const Keys &s) const {
    return s.ks + (uint64_t)blk * s.ks_blk + (uint64_t)off * s.ks_t;
  }
  MIA_DEV const float *vs(const Keys &s) const {
    return s.vs + (uint64_t)blk * s.vs_blk + (uint64_t)off * s.vs_t;
  }
};

// log2(e) x softmax scale x per-head scale of K: its magnitude; a negative
// factor goes to q (sign bits), so that the largest product is the largest
// score.
MIA_DEV float score_factor(const SpanParams &p, int h, uint32_t &neg) {
  float c1 = p.scale_log2;
  if (p.k_deq) c1 *= p.k_deq[h];
  neg = c1 < 0.f ? 0x80008000u : 0u;
  const float c2 = fabsf(c1);
  return c2 == 0.f ? 1e-37f : c2;  // masked scores (-inf) stay masked
}

// First partial row of piece c in share sh.w, and the header of a cut segment.
MIA_DEV int64_t piece_slot(const SpanParams &p, const Share &sh, const Piece &c, bool writer) {
  const SpanList &ls = p.list[c.li];
  int64_t slot;
  if (p.join) {
    const int segs = c.rt_n * p.Hkv;
    slot = (int64_t)(c.li ? c.i * segs : 0) + c.h * c.rt_n + c.rt + sh.w;
  } else {
    slot = 2 * sh.w + (c.t == 0 ? 1 : 0);
    if (c.t == 0 && writer) {
      int *hd = p.hdr + kHdr * sh.w;
      hd[1] = c.tok0;
      hd[2] = c.rows;
      hd[3] = c.rt;
      hd[4] = c.h;
      hd[0] = cut_of(sh.cut, c.x + c.tiles - 1) - sh.w + 1;
    }
  }
  return ls.part0 + slot * ls.part_rows;
}

// ---------------------------------------------------------------------------
// tall form
// ---------------------------------------------------------------------------
template <int D, int CT, bool SC>
struct TallLds {
  static constexpr int TILEB = kTallKeys * D * 2;
  uint8_t kv[2][2][TILEB];                       // [stage][K, V]
  float sc[2][2][SC ? kTallKeys : 4];            // [stage][K, V]
};

// DU <= D: the products stop there (a head dim of at most DU; channels past
// the head dim are zero).
template <int D, int CT, bool SC, int DU>
MIA_DEV void tall_body(const Share &sh, TallLds<D, CT, SC> &lds) {
  constexpr bool DMA = CT == kBf16;    // else through registers, widened
  constexpr int EB = CT == kBf16 ? 2 : 1;
  constexpr int CE = 16 / EB;          // elements per 16-byte load
  constexpr int LPR = D / CE;          // lanes per key row
  constexpr int RPW = 64 / LPR;        // key rows per wave and load
  constexpr int NP = 16 / RPW;         // loads per thread and tile (K, V each)
  static_assert(kTallKeys == 16 * kWaves, "a wave loads one 16-key group of a tile");
  constexpr int ROWB = D * 2;
  constexpr int TILEB = kTallKeys * ROWB;
  constexpr int KSTEPS = DU / 16;
  constexpr int DBLK = DU / 32;

  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int rl = lane & 31;
  lds_u8_t *const base = (lds_u8_t *)&lds.kv[0][0][0];
  lds_f32_t *const scb = (lds_f32_t *)&lds.sc[0][0][0];

  // ---- loads of a tile: wave w takes the 16 keys 16 w .. (one block: one
  // table entry), thread -> row j * RPW + lr of them, chunk lc
  const int lr = lane / LPR;
  const int lc = lane % LPR;
  const int d_used = fresh().d;
  const bool ch_ok = lc * CE < d_used;
  constexpr int NR = DMA ? 1 : NP;
  u32x4_t kr[NR], vr[NR];
  float sr[NR];
  Keys ks_;
  int ent = 0;  // the wave's table entry of a tile, loaded one tile ahead
  auto load_entry = [&](int t) { ent = ks_.entry(t * kTallKeys + wave * 16); };
  // the chunk a lane loads: for copies the one that the swizzle puts in its
  // slot, else its own (past the head dim: the first, stored nowhere)
  auto k_chunk = [&](int j) { return DMA ? lc ^ k_swz<D>(j * RPW + lr) : ch_ok ? lc : 0; };
  auto v_chunk = [&](int j) { return DMA ? lc ^ v_swz<D>(j * RPW + lr) : ch_ok ? lc : 0; };
  uint32_t ko[NP], vo[NP];  // a lane's bytes from its group's first row
  auto set_offsets = [&](int last) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const uint32_t rr = min(j * RPW + lr, last);
      ko[j] = rr * ks_.k_t + k_chunk(j) * 16;
      vo[j] = rr * ks_.v_t + v_chunk(j) * 16;
    }
  };
  auto set_keys = [&](const Piece &c) {
    ks_.set<SC>(fresh(), c);
    load_entry(c.t);
    set_offsets(15);
  };
  // Tile t of the segment of ks_ (its entry is loaded): copied into stage st,
  // or loaded into registers; the entry of the tile behind it.
  auto load_tile = [&](int t, int st) {
    const int k0 = t * kTallKeys + wave * 16;
    Group g;
    g.set(ks_, k0, ent);
    // rows past the span read its last key (in bounds) and are masked or
    // cleared later; the tail is a segment's last tile
    if (k0 + 16 > ks_.len) set_offsets(ks_.len - 1 - g.k16);
    if constexpr (DMA) {
      const uint32_t dst = (uint32_t)(uintptr_t)base + (st * 2) * TILEB + wave * 16 * ROWB;
      if (d_used == D) {
        copy16<NP>(g.k, ko, dst);
        copy16<NP>(g.v, vo, dst + TILEB);
      } else {
        // (one load per row group: its lanes past d differ from the others')
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if (k_chunk(j) * CE < d_used) copy1(g.k, ko[j], dst + j * 1024);
          if (v_chunk(j) * CE < d_used) copy1(g.v, vo[j], dst + TILEB + j * 1024);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        // (no condition on a load: the merge of its two results would wait)
        kr[j] = *reinterpret_cast<const u32x4_t *>(g.k + ko[j]);
        vr[j] = *reinterpret_cast<const u32x4_t *>(g.v + vo[j]);
        if constexpr (SC) {
          // even lanes of a row its K scale, odd ones its V scale
          const uint32_t rr = min(k0 + j * RPW + lr, ks_.len - 1) - g.k16;
          const float *sp = lc & 1 ? g.vs(ks_) : g.ks(ks_);
          sr[j] = sp[(uint64_t)rr * (lc & 1 ? ks_.vs_t : ks_.ks_t)];
        }
      }
    }
    if ((t + 1) * kTallKeys < ks_.len) load_entry(t + 1);
  };
  // 8-bit caches: the loaded tile widened into stage buf
  auto store_tile = [&](int t, int len, int buf) {
    const int kt = t * kTallKeys;
    lds_u8_t *const kb = base + (buf * 2) * TILEB;
    lds_u8_t *const vb = base + (buf * 2 + 1) * TILEB;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int row = wave * 16 + j * RPW + lr;
      // values past the span are cleared: 0 * NaN would reach the sums
      const bool in = kt + row < len;
      const u32x4_t v = in ? vr[j] : u32x4_t{0u, 0u, 0u, 0u};
      if (ch_ok)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        *(lds_u32x4_t *)(kb + row * ROWB + (((2 * lc + x) ^ k_swz<D>(row)) << 4)) =
            widen8<CT>(kr[j][2 * x], kr[j][2 * x + 1]);
        *(lds_u32x4_t *)(vb + row * ROWB + (((2 * lc + x) ^ v_swz<D>(row)) << 4)) =
            widen8<CT>(v[2 * x], v[2 * x + 1]);
        // converted a chunk at a time: all of them at once spill
        if constexpr (CT == kI8) __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (SC) {
        if (lc < 2) scb[(buf * 2 + lc) * kTallKeys + row] = in ? sr[j] : 0.f;
      }
    }
  };

  // ---- state of the current piece
  bf16x8_t qf[KSTEPS];
  f32x16_t acc[DBLK];
  float m_run = -INFINITY, l_run = 0.f;
  float c2 = 0.f;
  bool live = false;  // the wave has rows
  u32x4_t qw[KSTEPS];
  // the loads of the rows of a piece, issued ahead of its first tile's
  auto load_q = [&](const Piece &c) {
    const SpanParams &p = fresh();
    const int r = c.rt * kRows + wave * 32 + rl;
    live = c.rt * kRows + wave * 32 < c.rows;
    const bool ok = r < c.rows;
    const int pos = (int)fdiv((uint32_t)(ok ? r : 0), p.g_div);
    const int hq = c.h * p.G + (ok ? r - pos * p.G : 0);
    const uint16_t *qp = p.q + tok_off(p, c.tok0 + pos, p.qs_b, p.qs_s) + (int64_t)hq * p.qs_h;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      qw[ks] = u32x4_t{0u, 0u, 0u, 0u};
      const int d0 = ks * 16 + half * 8;
      if (ok && d0 < d_used) qw[ks] = *reinterpret_cast<const u32x4_t *>(qp + d0);
    }
  };
  auto begin_piece = [&](const Piece &c) {
    uint32_t neg;
    c2 = score_factor(fresh(), c.h, neg);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
      qf[ks] = __builtin_bit_cast(bf16x8_t, qw[ks] ^ u32x4_t{neg, neg, neg, neg});
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    m_run = -INFINITY;
    l_run = 0.f;
  };

  // transposed reads of V: within a 16-lane group, result lane k gets element
  // k % 4 of the 8 bytes read by lane 4j + k/4
  const int tr_k = lane & 15;
  const int tr_col = ((lane >> 4) & 1) * 16 + 4 * (tr_k & 3);
  const int tr_row = half * 4 + (tr_k >> 2);

  auto compute = [&](int t, int len, int buf) {
    const lds_u8_t *kb = base + (buf * 2) * TILEB;
    const lds_u8_t *vb = base + (buf * 2 + 1) * TILEB;
    const lds_f32_t *ksb = scb + (buf * 2) * kTallKeys;
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
    const int left = len - t * kTallKeys - half * 4;
    if ((t + 1) * kTallKeys > len) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = b * 32 + (e >> 2) * 8 + (e & 3) < left ? s[b][e] : -INFINITY;
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
    // moves the maximum of the rows with `bump` to mx
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

  // ---- end of a piece: final rows, or a partial
  auto end_piece = [&](const Piece &c) {
    const SpanParams &p = fresh();
    const float l = sum32(l_run);
    const int rloc = wave * 32 + rl;
    const int r = c.rt * kRows + rloc;
    if (!p.join && c.whole()) {
      if (r >= c.rows) return;
      const int pos = (int)fdiv((uint32_t)r, p.g_div);
      uint16_t *op = p.out + tok_off(p, c.tok0 + pos, p.os_b, p.os_s) +
                     (int64_t)(c.h * p.G + r - pos * p.G) * p.os_h;
      float inv = l == 0.f ? 0.f : 1.f / l;
      if (p.v_deq) inv *= p.v_deq[c.h];
#pragma unroll
      for (int i = 0; i < DBLK; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d0 = i * 32 + g * 8 + half * 4;
          if (d0 < p.d)
            *reinterpret_cast<u32x2_t *>(op + d0) =
                u32x2_t{pack2_bf16(acc[i][g * 4] * inv, acc[i][g * 4 + 1] * inv),
                        pack2_bf16(acc[i][g * 4 + 2] * inv, acc[i][g * 4 + 3] * inv)};
        }
      return;
    }
    const int64_t pr = piece_slot(p, sh, c, tid == 0) + rloc;
    if (r >= c.rows || rloc >= p.list[c.li].part_rows) return;
    float *po = p.part_o + pr * D;
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t *>(po + i * 32 + g * 8 + half * 4) =
            f32x4_t{acc[i][g * 4], acc[i][g * 4 + 1], acc[i][g * 4 + 2], acc[i][g * 4 + 3]};
    if (half == 0) p.part_ml[pr] = make_float2(m_run, l);
  };

  // ---- the stream
  Piece cur, nxt;
  if (!first_piece(fresh(), sh, cur)) return;
  if (d_used < D) {  // channels past d: zero in both stages, never written again
    for (int o = tid * 16; o < 4 * TILEB; o += kThreads * 16)
      *(lds_u32x4_t *)(base + o) = u32x4_t{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  load_q(cur);
  set_keys(cur);
  int t = cur.t, end = cur.t + cur.n, buf = 0;
  // The tile behind t, of the next piece behind the last of this one: go: there
  // is one, anew: it starts piece nxt.
  int tn = 0;
  bool go = false, anew = false;
  auto step = [&]() {
    tn = t + 1;
    go = true;
    anew = false;
    if (tn < end) return;
    nxt = cur;
    go = anew = next_piece(fresh(), sh, nxt);
    tn = 0;
    if (go) set_keys(nxt);
  };
  if constexpr (DMA) {
    load_tile(t, 0);
    begin_piece(cur);
    bool at_live = live;
    while (true) {
      // own copies of this tile have landed; the barrier makes every thread's
      // visible and the other stage free
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      step();
      if (anew) load_q(nxt);  // (sets live for the next piece)
      if (go) load_tile(tn, buf ^ 1);
      const int left = cur.len - t * kTallKeys;
      if (left < kTallKeys) {
        // values past the span are cleared: 0 * NaN would reach the sums
        lds_u8_t *const vb = base + (buf * 2 + 1) * TILEB;
        for (int o = left * ROWB + tid * 16; o < TILEB; o += kThreads * 16)
          *(lds_u32x4_t *)(vb + o) = u32x4_t{0u, 0u, 0u, 0u};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if (at_live) compute(t, cur.len, buf);
      if (!go || anew) {
        end_piece(cur);
        if (!go) return;
        cur = nxt;
        end = cur.n;
        begin_piece(cur);
        at_live = live;
      }
      t = tn;
      buf ^= 1;
    }
  } else {
    load_tile(t, 0);
    begin_piece(cur);
    store_tile(t, cur.len, 0);
    step();
    if (go) load_tile(tn, 0);
    __syncthreads();
    while (true) {
      if (live) compute(t, cur.len, buf);
      if (!go || anew) {
        end_piece(cur);
        if (!go) return;
        cur = nxt;
        end = cur.n;
        load_q(cur);  // (ahead of the products its registers would spill others)
        begin_piece(cur);
      }
      store_tile(tn, cur.len, buf ^ 1);
      t = tn;
      step();
      if (go) load_tile(tn, 0);
      __syncthreads();
      buf ^= 1;
    }
  }
}

// ---------------------------------------------------------------------------
// thin form
// ---------------------------------------------------------------------------
template <int D, bool SC>
struct ThinLds {
  uint8_t v[kWaves][kThinKeys * D * 2];
  float sc[kWaves][SC ? 2 * kThinKeys : 4];
};

// NC groups of 16 columns (rows of the segment).
template <int D, int CT, bool SC, int DU, int NC>
MIA_DEV void thin_body(const Share &sh, ThinLds<D, SC> &lds) {
  constexpr int EB = CT == kBf16 ? 2 : 1;
  // (8-bit k-steps come in pairs: all of D)
  constexpr int KSTEPS = (CT == kBf16 ? DU : D) / 32;
  constexpr int VE = 16 / EB;          // V elements per 16-byte load
  constexpr int DS = D / VE;           // lanes per V row
  constexpr int TL = 64 / DS;          // V rows per load
  constexpr int NV = kThinKeys / TL;   // V loads per tile
  static_assert(TL <= 16, "a V load's rows lie in one 16-key group");
  // K: bf16 k-step ks of lane group kg holds channels 32 ks + 8 kg; 8-bit
  // k-steps 2u and 2u + 1 channels 64 u + 16 kg and + 8 (one 16-byte load)
  constexpr int NK = CT == kBf16 ? KSTEPS : KSTEPS / 2;  // K loads per 16 keys
  constexpr int ROWB = D * 2;
  constexpr int VNCH = D / 8;
  constexpr int DB16 = DU / 16;

  const int wave = readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 15;
  const int kg = lane >> 4;
  lds_u8_t *const vw = (lds_u8_t *)&lds.v[wave][0];
  lds_f32_t *const sw = (lds_f32_t *)&lds.sc[wave][0];

  const int d_used = fresh().d;
  auto k_chan = [](int j, int g) { return CT == kBf16 ? j * 32 + g * 8 : j * 64 + g * 16; };
  const int vds = lane % DS, vtl = lane / DS;

  u32x4_t kr[2][NK], vr[NV];
  float sr = 0.f;
  // bytes of a lane's chunks in a row; past the head dim the first chunk: K is
  // cleared at its use, what V gives there is stored nowhere
  uint32_t kch[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j) kch[j] = k_chan(j, kg) < d_used ? k_chan(j, kg) * EB : 0;
  const uint32_t vch = vds * VE < d_used ? vds * 16 : 0;
  const bool narrow = d_used < D;
  Keys ks_;
  Group g[2];
  int ent[2];  // table entries of a tile, loaded one tile ahead
  auto load_entries = [&](int t) {
    ent[0] = ks_.entry(t * kThinKeys);
    ent[1] = ks_.entry(t * kThinKeys + 16);
  };
  auto set_keys = [&](const Piece &c) {
    ks_.set<SC>(fresh(), c);
    load_entries(c.t);
  };
  // the groups of tile t of the segment of ks_ (its entries are loaded), and
  // the entries of the tile behind it
  auto locate = [&](int t) {
    g[0].set(ks_, t * kThinKeys, ent[0]);
    g[1].set(ks_, t * kThinKeys + 16, ent[1]);
    if ((t + 1) * kThinKeys < ks_.len) load_entries(t + 1);
  };
  // rows past the span read its last key (in bounds) and are masked or
  // cleared later
  auto load_k = [&](int t) {
    const bool full = (t + 1) * kThinKeys <= ks_.len;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      int rr = col;
      if (!full) rr = min(t * kThinKeys + b * 16 + col, ks_.len - 1) - g[b].k16;
      // (no condition on a load: the merge of its two results would wait)
#pragma unroll
      for (int j = 0; j < NK; ++j)
        kr[b][j] = *reinterpret_cast<const u32x4_t *>(g[b].k + (rr * ks_.k_t + kch[j]));
    }
  };
  auto load_v = [&](int t) {
    const bool full = (t + 1) * kThinKeys <= ks_.len;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Group &x = g[j * TL / 16];
      int rr = j * TL % 16 + vtl;
      if (!full) rr = min(t * kThinKeys + j * TL + vtl, ks_.len - 1) - x.k16;
      vr[j] = *reinterpret_cast<const u32x4_t *>(x.v + (rr * ks_.v_t + vch));
    }
  };
  // lane l: scale of key l (K), of key l - 32 (V)
  auto load_s = [&](int t) {
    if constexpr (SC) {
      const int k = lane & 31;
      const bool hi = k >= 16;
      const uint32_t rr = min(t * kThinKeys + k, ks_.len - 1) - (hi ? g[1].k16 : g[0].k16);
      const float *ks = hi ? g[1].ks(ks_) : g[0].ks(ks_);
      const float *vs = hi ? g[1].vs(ks_) : g[0].vs(ks_);
      const float *sp = lane < 32 ? ks : vs;
      sr = sp[(uint64_t)rr * (lane < 32 ? ks_.ks_t : ks_.vs_t)];
    }
  };

  // ---- state of the current piece
  bf16x8_t qf[NC][KSTEPS];
  f32x4_t acc[NC][DB16];
  float m_run[NC], l_run[NC];
  float c2 = 0.f;
  u32x4_t qw[NC][KSTEPS];
  // the loads of the rows of a piece, issued ahead of its first tile's
  auto load_q = [&](const Piece &c) {
    const SpanParams &p = fresh();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int r = n * 16 + col;
      const bool ok = r < c.rows;
      const int pos = (int)fdiv((uint32_t)(ok ? r : 0), p.g_div);
      const int hq = c.h * p.G + (ok ? r - pos * p.G : 0);
      const uint16_t *qp = p.q + tok_off(p, c.tok0 + pos, p.qs_b, p.qs_s) + (int64_t)hq * p.qs_h;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int d0 = CT == kBf16 ? k_chan(ks, kg) : k_chan(ks >> 1, kg) + (ks & 1) * 8;
        qw[n][ks] = u32x4_t{0u, 0u, 0u, 0u};
        if (ok && d0 < d_used) qw[n][ks] = *reinterpret_cast<const u32x4_t *>(qp + d0);
      }
    }
  };
  auto begin_piece = [&](const Piece &c) {
    uint32_t neg;
    c2 = score_factor(fresh(), c.h, neg);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
        qf[n][ks] = __builtin_bit_cast(bf16x8_t, qw[n][ks] ^ u32x4_t{neg, neg, neg, neg});
#pragma unroll
      for (int i = 0; i < DB16; ++i) acc[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      m_run[n] = -INFINITY;
      l_run[n] = 0.f;
    }
  };

  // V^T operand of 16 channels: k index j of lane group kg is key 4 kg + j
  // (j < 4), 16 + 4 kg + j - 4 (else), the keys whose scores the lane holds;
  // source lane s of a 16-lane group addresses key 4 kg + s/4, channels 4 (s%4)
  const int tr_s = lane & 15;
  const int tr_row = 4 * kg + (tr_s >> 2);
  const int tr_x = tr_row & (VNCH - 1);

  // S^T of the tile; frees the K registers
  f32x4_t s[NC][2];
  auto scores = [&]() {
    if (narrow) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < NK; ++j)
          if (k_chan(j, kg) >= d_used) kr[b][j] = u32x4_t{0u, 0u, 0u, 0u};
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
  auto store_v = [&](int left) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int t = j * TL + vtl;
      // values past the span are cleared: 0 * NaN would reach the sums
      const u32x4_t v = t < left ? vr[j] : u32x4_t{0u, 0u, 0u, 0u};
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
  u32x4_t pk[NC];
  auto softmax = [&](int left0) {
    f32x4_t ks4[2], vs4[2];
    if constexpr (SC) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        ks4[b] = *(const lds_f32x4_t *)(sw + b * 16 + kg * 4);
        vs4[b] = *(const lds_f32x4_t *)(sw + 32 + b * 16 + kg * 4);
      }
    }
    const int left = left0 - kg * 4;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[n][b][i];
          if constexpr (SC) x *= ks4[b][i];
          x = b * 16 + i < left ? x : -INFINITY;
          s[n][b][i] = x;
          mx = fmaxf(mx, x);
        }
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
        // rounded to bf16 for the MFMA; the sum keeps the unrounded ones
        pk[n][2 * b] = pack2_bf16(pr[0], pr[1]);
        pk[n][2 * b + 1] = pack2_bf16(pr[2], pr[3]);
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
      for (int n = 0; n < NC; ++n)
        acc[n][blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, pk[n]), acc[n][blk], 0,
            0, 0);
    }
  };
  auto end_piece = [&](const Piece &c) {
    const SpanParams &p = fresh();
    const bool whole = !p.join && c.whole();
    const int64_t pr0 = whole ? 0 : piece_slot(p, sh, c, lane == 0);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float l = sum32(sum16(l_run[n]));
      const int r = n * 16 + col;
      if (r >= c.rows) continue;
      if (whole) {
        const int pos = (int)fdiv((uint32_t)r, p.g_div);
        uint16_t *op = p.out + tok_off(p, c.tok0 + pos, p.os_b, p.os_s) +
                       (int64_t)(c.h * p.G + r - pos * p.G) * p.os_h;
        float inv = l == 0.f ? 0.f : 1.f / l;
        if (p.v_deq) inv *= p.v_deq[c.h];
#pragma unroll
        for (int i = 0; i < DB16; ++i) {
          const int d0 = i * 16 + kg * 4;
          if (d0 < p.d)
            *reinterpret_cast<u32x2_t *>(op + d0) =
                u32x2_t{pack2_bf16(acc[n][i][0] * inv, acc[n][i][1] * inv),
                        pack2_bf16(acc[n][i][2] * inv, acc[n][i][3] * inv)};
        }
      } else if (r < p.list[c.li].part_rows) {
        float *po = p.part_o + (pr0 + r) * D;
#pragma unroll
        for (int i = 0; i < DB16; ++i)
          *reinterpret_cast<f32x4_t *>(po + i * 16 + kg * 4) = acc[n][i];
        if (kg == 0) p.part_ml[pr0 + r] = make_float2(m_run[n], l);
      }
    }
  };

  // ---- the stream: K (V) of the next tile is issued once this tile's
  // product (copy to LDS) has freed the registers
  Piece cur, nxt;
  if (!first_piece(fresh(), sh, cur)) return;
  load_q(cur);
  set_keys(cur);
  int t = cur.t, end = cur.t + cur.n;
  locate(t);
  load_k(t);
  load_s(t);
  load_v(t);
  begin_piece(cur);
  while (true) {
    // the tile behind t, of the next piece behind the last of this one
    int tn = t + 1;
    bool go = true, anew = false;
    if (tn >= end) {
      nxt = cur;
      go = anew = next_piece(fresh(), sh, nxt);
      tn = 0;
      if (go) {
        if (NC == 1) load_q(nxt);
        set_keys(nxt);
      }
    }
    if (go) locate(tn);
    const int left = cur.len - t * kThinKeys;
    scores();
    if constexpr (SC) sw[lane] = (lane & 31) < left ? sr : 0.f;
    if (go) {
      load_k(tn);
      load_s(tn);
    }
    softmax(left);
    store_v(left);
    if (go) load_v(tn);
    values();
    if (!go || anew) {
      end_piece(cur);
      if (!go) return;
      cur = nxt;
      end = cur.n;
      if (NC > 1) load_q(cur);  // (ahead of the products it would spill)
      begin_piece(cur);
    }
    t = tn;
  }
}

template <int D, int CT, bool SC, int DU, int NC>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void span_kernel(SpanParams p) {
  static_assert((D == 64 && DU == 64) || (D == 128 && (DU == 96 || DU == 128)), "tile widths");
  static_assert(CT != kBf16 || !SC, "bf16 caches have no per-key scales");
  __shared__ union __attribute__((aligned(1024))) {
    TallLds<D, CT, SC> tall;
    ThinLds<D, SC> thin;
  } lds;
  __shared__ PlanLds plan_lds;
  Share sh;
  const int form = plan(fresh(), plan_lds, sh);
  if (form == 0) tall_body<D, CT, SC, DU>(sh, lds.tall);
  else if (form == 1) thin_body<D, CT, SC, DU, NC>(sh, lds.thin);
}

// A row is joined by GR groups of D / 4 lanes, four channels a lane.
template <int D, int GR>
struct JoinLds {
  f32x4_t o[256 / (D / 4)][D / 4];
  float2 ml[256 / (D / 4)];
};

// The row's n pieces (partial row prow(j)): group g adds g, g + GR, ... to its
// (m, l, o), three loads in flight (drafted int8 rows 11.8 us, with four 12.5;
// two: 8 fp8 tokens over 1601-6404 keys 5.8 us against 5.5).
template <int D, int GR, typename F>
MIA_DEV void sum_pieces(const SpanParams &p, int n, F prow, float &m, float &l, f32x4_t &o) {
  constexpr int LPR = D / 4, U = 3;
  const int g = threadIdx.x / LPR % GR, c = threadIdx.x % LPR;
  for (int j = g; j < n; j += U * GR) {
    float2 ml[U];
    f32x4_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = prow(min(j + u * GR, n - 1));
      ml[u] = p.part_ml[r];
      v[u] = *reinterpret_cast<const f32x4_t *>(p.part_o + r * D + (c * 4 < p.d ? c * 4 : 0));
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * GR < n) add_piece(m, l, o, ml[u].x, ml[u].y, v[u]);
  }
}

// The groups of a row added through LDS (every thread of the workgroup calls
// this); group 0 has the result.
template <int D, int GR>
MIA_DEV void sum_groups(JoinLds<D, GR> &lds, float &m, float &l, f32x4_t &o) {
  constexpr int LPR = D / 4;
  const int gi = threadIdx.x / LPR, c = threadIdx.x % LPR;
  lds.o[gi][c] = o;
  if (c == 0) lds.ml[gi] = make_float2(m, l);
  __syncthreads();
  if (gi % GR) return;
#pragma unroll
  for (int k = 1; k < GR; ++k)
    add_piece(m, l, o, lds.ml[gi + k].x, lds.ml[gi + k].y, lds.o[gi + k][c]);
}

// Joins the pieces of cut segments (cross attention): workgroup (w, y) takes
// rows of the segment that starts, cut, in share w.
template <int D, int GR>
__global__ __launch_bounds__(256) void span_merge_kernel(SpanParams p) {
  __shared__ JoinLds<D, GR> lds;
  const int w = blockIdx.x;
  const int *hd = p.hdr + kHdr * w;
  const int n = hd[0];
  if (n == 0) return;
  constexpr int LPR = D / 4;
  const int c = threadIdx.x % LPR;
  const SpanList &l = p.list[1];
  const int rloc = blockIdx.y * (256 / LPR / GR) + threadIdx.x / LPR / GR;
  const int r = hd[3] * kRows + rloc;
  const bool ok = r < hd[2] && rloc < l.part_rows;
  auto prow = [&](int j) {
    return l.part0 + (int64_t)(j == 0 ? 2 * w + 1 : 2 * (w + j)) * l.part_rows + rloc;
  };
  float m = -INFINITY, ls = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  sum_pieces<D, GR>(p, ok ? n : 0, prow, m, ls, o);
  if constexpr (GR > 1) sum_groups<D, GR>(lds, m, ls, o);
  if (!ok || threadIdx.x / LPR % GR) return;
  float inv = ls == 0.f ? 0.f : 1.f / ls;
  const int h = hd[4];
  if (p.v_deq) inv *= p.v_deq[h];
  const int pos = (int)fdiv((uint32_t)r, p.g_div);
  if (c * 4 >= p.d) return;
  uint16_t *op = p.out + tok_off(p, hd[1] + pos, p.os_b, p.os_s) +
                 (int64_t)(h * p.G + r - pos * p.G) * p.os_h;
  *reinterpret_cast<u32x2_t *>(op + c * 4) =
      u32x2_t{pack2_bf16(o[0] * inv, o[1] * inv), pack2_bf16(o[2] * inv, o[3] * inv)};
}

// Shared prefix: joins the pieces of a row's prefix and own span, adds the
// new tokens that not every row of its sequence sees (the last S - 1 keys,
// row s sees s of them) and the sink.  D / 4 lanes per row.
constexpr int kJoinGroups = 8;

template <int D, int CT, bool SC, int GR>
__global__ __launch_bounds__(256) void span_join_kernel(SpanParams p, FastDiv hq_div) {
  constexpr int LPR = D / 4;
  __shared__ JoinLds<D, GR> lds;
  const int c = threadIdx.x % LPR;
  const int n_rows = p.num_tokens * (int)hq_div.d;
  const int my_row = blockIdx.x * (256 / LPR / GR) + threadIdx.x / LPR / GR;
  const int row = min(my_row, n_rows - 1);
  const int t = (int)fdiv((uint32_t)row, hq_div);
  const int hq = row - t * (int)hq_div.d;
  const int h = (int)fdiv((uint32_t)hq, p.g_div);
  const int g = hq - h * p.G;
  const int b = (int)fdiv((uint32_t)t, p.s_div);
  const int s = t - b * p.S;
  // first partial row and pieces of the row in list li, sequence i, its row r
  auto pieces = [&](int li, int i, int r, int rows, int64_t &first) {
    const SpanList &l = p.list[li];
    const int tiles = key_tiles(l, list_len(l, i));
    const int rt_n = row_tiles(l, rows), rt = l.thin ? 0 : r / kRows;
    const int in = h * rt_n + rt;  // segment of the sequence
    const Cut cut = {p.hdr[2 * l.thin], p.hdr[2 * l.thin + 1]};
    const int over = p.over[l.thin];
    const int x = p.hdr[kHdr + (li ? p.list[0].n + i : i)] + in * (tiles + over) + over;
    first = 0;
    if (tiles == 0) return 0;
    const int w = cut_of(cut, x);
    first = l.part0 + ((int64_t)i * rt_n * p.Hkv + in + w) * l.part_rows + (r - rt * kRows);
    return cut_of(cut, x + tiles - 1) - w + 1;
  };
  const SpanList &l0 = p.list[0], &l1 = p.list[1];
  int64_t f0, f1;
  const int n0 = pieces(0, 0, t * p.G + g, p.num_tokens * p.G, f0);
  const int n1 = pieces(1, b, s * p.G + g, p.S * p.G, f1);
  auto prow = [&](int j) {
    return j < n0 ? f0 + (int64_t)j * l0.part_rows : f1 + (int64_t)(j - n0) * l1.part_rows;
  };
  const int gr = threadIdx.x / LPR % GR;
  // the keys between the span that all rows see and row s's own last key:
  // group g takes common + g, ..., the first of them loaded ahead of the pieces
  struct Late {
    u32x2_t k, v;
    float ks, vs;
  };
  const bool c_ok = c * 4 < p.d;
  auto load_late = [&](int k) {
    const int bj = (int)fdiv((uint32_t)k, p.bs_div);
    const uint32_t blk =
        min(max(scalar_load(l1.bt, (int64_t)b * l1.bt_s + (int64_t)bj * l1.bt_j), 0), p.nb - 1);
    const uint32_t off = k - bj * p.bs;
    const uint8_t *ka =
        p.k_cache + (((uint64_t)blk * p.kc_blk16) << 4) + (int64_t)h * p.kc_h + off * p.kc_t;
    const uint8_t *va =
        p.v_cache + (((uint64_t)blk * p.vc_blk16) << 4) + (int64_t)h * p.vc_h + off * p.vc_t;
    Late x = {u32x2_t{0u, 0u}, u32x2_t{0u, 0u}, 1.f, 1.f};
    if (c_ok) {
      if constexpr (CT == kBf16) {
        x.k = *reinterpret_cast<const u32x2_t *>(ka + c * 8);
        x.v = *reinterpret_cast<const u32x2_t *>(va + c * 8);
      } else {
        x.k[0] = *reinterpret_cast<const uint32_t *>(ka + c * 4);
        x.v[0] = *reinterpret_cast<const uint32_t *>(va + c * 4);
      }
    }
    if constexpr (SC) {
      x.ks = p.k_sc[(uint64_t)blk * p.ks_blk + h * p.ks_h + (uint64_t)off * p.ks_t];
      x.vs = p.v_sc[(uint64_t)blk * p.vs_blk + h * p.vs_h + (uint64_t)off * p.vs_t];
    }
    return x;
  };
  auto four = [&](u32x2_t w, float (&x)[4]) {
    if constexpr (CT == kBf16) {
      x[0] = bf16lo(w[0]), x[1] = bf16hi(w[0]), x[2] = bf16lo(w[1]), x[3] = bf16hi(w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t byte = (w[0] >> (8 * i)) & 0xffu;
        x[i] = CT == kI8 ? (float)(int8_t)byte : e4m3fn_bits_to_f32(byte);
      }
    }
  };
  int late0 = 0, late1 = 0;
  u32x2_t qw = {0u, 0u};
  Late late;
  if (s > 0) {
    late0 = list_len(l1, b) + gr;
    late1 = min(max(scalar_load(l1.len, b), 0) - l1.len_sub + s, l1.len_cap);
    if (late0 < late1) {
      late = load_late(late0);
      if (c_ok)
        qw = *reinterpret_cast<const u32x2_t *>(p.q + (int64_t)b * p.qs_b + (int64_t)s * p.qs_s +
                                                (int64_t)hq * p.qs_h + c * 4);
    }
  }
  float m = -INFINITY, ls = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  if (p.sink && gr == 0) {
    m = p.sink[hq] * kLog2e;
    ls = 1.f;
  }
  sum_pieces<D, GR>(p, n0 + n1, prow, m, ls, o);
  if (late0 < late1) {
    float c1 = p.scale_log2;
    if (p.k_deq) c1 *= p.k_deq[h];
    const float qv[4] = {bf16lo(qw[0]), bf16hi(qw[0]), bf16lo(qw[1]), bf16hi(qw[1])};
    for (int k = late0; k < late1; k += GR) {
      if (k > late0) late = load_late(k);
      float x[4], v[4];
      four(late.k, x);
      four(late.v, v);
      float dot = qv[0] * x[0] + qv[1] * x[1] + qv[2] * x[2] + qv[3] * x[3];
#pragma unroll
      for (int q = 1; q < LPR; q <<= 1) dot += __shfl_xor(dot, q, 64);
      add_piece(m, ls, o, dot * late.ks * c1, 1.f,
                f32x4_t{v[0] * late.vs, v[1] * late.vs, v[2] * late.vs, v[3] * late.vs});
    }
  }
  sum_groups<D, GR>(lds, m, ls, o);
  if (gr != 0 || my_row >= n_rows) return;
  float inv = ls == 0.f ? 0.f : 1.f / ls;
  if (p.v_deq) inv *= p.v_deq[h];
  if (c * 4 >= p.d) return;
  uint16_t *op = p.out + (int64_t)b * p.os_b + (int64_t)s * p.os_s + (int64_t)hq * p.os_h;
  *reinterpret_cast<u32x2_t *>(op + c * 4) =
      u32x2_t{pack2_bf16(o[0] * inv, o[1] * inv), pack2_bf16(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

struct Layout {
  int grid;
  size_t hdr, ml, o, total;  // byte offsets and size
};

// Launch size and workspace of a call; fills the lists' forms and partials.
Layout span_layout(SpanParams &p, int D) {
  Layout w;
  w.grid = (D == 64 ? 3 : 2) * cu_count();
  int64_t rows = 0, hdr = kHdr;
  for (int li = 0; li < 2; ++li) {
    SpanList &l = p.list[li];
    if (l.n == 0) continue;
    const int64_t seq_rows = (int64_t)l.tok_max * p.G;
    l.thin = seq_rows <= 32;
    const int64_t units = (int64_t)w.grid * (l.thin ? kWaves : 1);
    l.part_rows = (int)std::min<int64_t>(kRows, seq_rows);
    l.part0 = rows;
    if (p.join) {
      const int64_t segs = (seq_rows + kRows - 1) / kRows * p.Hkv * l.n;
      rows += (segs + units) * l.part_rows;
      hdr += l.n;
    } else {
      rows += 2 * units * l.part_rows;
      hdr += units * kHdr;
    }
  }
  // Measured, side by side: a thin tile takes a wave 2.3 us and a tall one a
  // workgroup 1.7 us at d = 64 (3.8 and 2.6 us at d = 128): with four
  // waves to a workgroup 0.34 and 0.37.  Calls differ little by it; thin costs of
  // 0.30 / 0.35 / 0.40 / 0.45: 64 rows behind 8192 keys (d = 128) 53.8 / 53.5 /
  // 53.1 / 53.2 us; 128 rows behind 4133 (d = 64) 44.9 / 44.2 / 44.1 / 44.7; 64
  // drafted int8 rows behind 32768 127.3 / 119.9 / 119.7 / 122.7.  A segment's
  // start costs about two tiles (tall, three: ragged prompts of d = 80 61.4 us
  // against 59.8; thin at d = 128, one: 57.1 against 55.8), one for thin ones at
  // d = 64 (45.0 against 47.0).  Shares of six units and more leave CUs idle
  // on short calls (15.6 -> 18.3).
  p.cost[0] = 1.0f, p.cost[1] = 0.40f;
  p.over[0] = 2, p.over[1] = D == 64 ? 1 : 2;
  p.least[0] = 4, p.least[1] = D == 64 ? 3 : 4;
  w.hdr = 0;
  w.ml = (size_t)up(hdr * 4, 256);
  w.o = w.ml + (size_t)up(rows * 8, 256);
  w.total = w.o + (size_t)rows * D * 4;
  return w;
}

void bind_workspace(SpanParams &p, const Layout &w, void *ws) {
  p.hdr = (int *)((uint8_t *)ws + w.hdr);
  p.part_ml = (float2 *)((uint8_t *)ws + w.ml);
  p.part_o = (float *)((uint8_t *)ws + w.o);
}

template <typename A>
void set_cache(SpanParams &p, const A &a) {
  const int eb = a.cache_dtype == MIA_DTYPE_BF16 ? 2 : 1;
  p.k_cache = (const uint8_t *)a.k_cache;
  p.v_cache = (const uint8_t *)a.v_cache;
  p.kc_blk16 = (uint32_t)(a.k_cache_stride[0] * eb / 16);
  p.vc_blk16 = (uint32_t)(a.v_cache_stride[0] * eb / 16);
  p.kc_h = a.k_cache_stride[1] * eb, p.kc_t = a.k_cache_stride[2] * eb;
  p.vc_h = a.v_cache_stride[1] * eb, p.vc_t = a.v_cache_stride[2] * eb;
  p.k_sc = a.k_scales, p.v_sc = a.v_scales;
  p.ks_blk = (uint32_t)a.k_scale_stride[0], p.ks_t = (uint32_t)a.k_scale_stride[2];
  p.vs_blk = (uint32_t)a.v_scale_stride[0], p.vs_t = (uint32_t)a.v_scale_stride[2];
  p.ks_h = a.k_scale_stride[1], p.vs_h = a.v_scale_stride[1];
  p.k_deq = a.k_dequant, p.v_deq = a.v_dequant;
  p.nb = a.num_blocks, p.bs = a.block_size;
  p.bs_div = make_fastdiv(a.block_size);
  p.Hkv = a.num_kv_heads, p.G = a.num_q_heads / a.num_kv_heads, p.d = a.head_dim;
  p.g_div = make_fastdiv(p.G);
  p.scale_log2 = a.softmax_scale * kLog2e;
  p.q = (const uint16_t *)a.q, p.out = (uint16_t *)a.out;
}

SpanParams cross_params(const mia_cross_args &a) {
  SpanParams p = {};
  set_cache(p, a);
  p.num_tokens = a.num_tokens, p.S = 1;
  p.zero_rest = a.zero_rest;
  p.s_div = make_fastdiv(1);
  p.qs_b = a.q_stride[0], p.qs_s = 0, p.qs_h = a.q_stride[1];
  p.os_b = a.out_stride[0], p.os_s = 0, p.os_h = a.out_stride[1];
  SpanList &l = p.list[1];
  l.n = a.num_seqs;
  l.cu = a.cu_seqlens_q;
  l.tok_per = 1;
  l.tok_max = a.cu_seqlens_q ? a.max_seqlen_q : 1;
  l.len = a.key_lens;
  l.len_cap = a.block_table ? a.blocks_per_seq * a.block_size : a.block_size;
  l.bt = a.block_table, l.bt_s = a.bt_stride[0], l.bt_j = a.bt_stride[1];
  return p;
}

SpanParams prefix_params(const mia_shared_prefix_args &a) {
  SpanParams p = {};
  set_cache(p, a);
  p.num_tokens = a.batch * a.s_active, p.S = a.s_active;
  p.s_div = make_fastdiv(a.s_active);
  p.qs_b = a.q_stride[0], p.qs_s = a.q_stride[1], p.qs_h = a.q_stride[2];
  p.os_b = a.out_stride[0], p.os_s = a.out_stride[1], p.os_h = a.out_stride[2];
  p.sink = a.sink;
  p.join = 1;
  SpanList &l0 = p.list[0], &l1 = p.list[1];
  l0.n = 1;
  l0.tok_per = l0.tok_max = p.num_tokens;
  l0.len = a.prefix_len;
  l0.len_cap = a.prefix_blocks * a.block_size;
  l0.bt = a.prefix_table, l0.bt_j = a.prefix_stride;
  l1.n = a.batch;
  l1.tok_per = l1.tok_max = a.s_active;
  l1.len = a.seq_lens;
  l1.len_sub = a.s_active - 1;
  l1.len_cap = a.blocks_per_seq * a.block_size;
  l1.bt = a.block_table, l1.bt_s = a.bt_stride[0], l1.bt_j = a.bt_stride[1];
  return p;
}

template <int D, int CT, bool SC>
void launch_span(const SpanParams &p, int grid, hipStream_t s) {
  const int cols = std::max(p.list[0].thin && p.list[0].n ? p.list[0].part_rows : 0,
                            p.list[1].thin ? p.list[1].part_rows : 0);
  // head dims of 65 to 96 leave a quarter of the 128-wide products out
  constexpr int DN = D == 128 ? 96 : D;
  if (D == 128 && p.d <= DN) {
    if (cols <= 16) span_kernel<D, CT, SC, DN, 1><<<grid, kThreads, 0, s>>>(p);
    else span_kernel<D, CT, SC, DN, 2><<<grid, kThreads, 0, s>>>(p);
  } else {
    if (cols <= 16) span_kernel<D, CT, SC, D, 1><<<grid, kThreads, 0, s>>>(p);
    else span_kernel<D, CT, SC, D, 2><<<grid, kThreads, 0, s>>>(p);
  }
  if (p.join) {
    // Lane groups per row: more of them sum more of a row's pieces at once, as
    // long as the launch has fewer waves than one resident round (8 per SIMD).
    // By 2 / 4 / 8 groups, us: 4 rows of 32 heads (d = 64) 5.8 / 5.4 / 5.2; 64
    // rows of 32 (d = 128, a round exactly by 8) 7.7 / 7.4 / 8.7; 64 int8 rows
    // of 48 (d = 128) 14.0 / 12.3 / 16.0; 128 rows of 64 (d = 64, a round
    // exactly by 4) 7.6 / 9.0 / 13.8.
    const int hq = p.Hkv * p.G;
    const int rows = p.num_tokens * hq;
    const int64_t waves = (int64_t)rows * (D / 4) / 64, resident = 32 * cu_count();
    auto join = [&](auto kernel, int groups) {
      const int rpb = 256 / (D / 4) / groups;
      kernel<<<(rows + rpb - 1) / rpb, 256, 0, s>>>(p, make_fastdiv(hq));
    };
    if (waves * 8 < resident) join(span_join_kernel<D, CT, SC, 8>, 8);
    else if (waves * 4 < resident) join(span_join_kernel<D, CT, SC, 4>, 4);
    else join(span_join_kernel<D, CT, SC, 2>, 2);
  }
}

template <int D>
void launch_width(const SpanParams &p, int cache_dtype, int grid, hipStream_t s) {
  const bool sc = p.k_sc != nullptr;
  if (cache_dtype == MIA_DTYPE_BF16) launch_span<D, kBf16, false>(p, grid, s);
  else if (cache_dtype == MIA_DTYPE_I8) launch_span<D, kI8, true>(p, grid, s);
  else if (sc) launch_span<D, kFp8, true>(p, grid, s);
  else launch_span<D, kFp8, false>(p, grid, s);
  if (!p.join) {
    constexpr int RPB = 256 / (D / 4);
    const SpanList &l = p.list[1];
    if (l.thin)
      span_merge_kernel<D, kJoinGroups>
          <<<dim3(grid * kWaves, (l.part_rows * kJoinGroups + RPB - 1) / RPB), 256, 0, s>>>(p);
    else
      span_merge_kernel<D, 1><<<dim3(grid, (l.part_rows + RPB - 1) / RPB), 256, 0, s>>>(p);
  }
}

int launch(SpanParams &p, int cache_dtype, void *ws, hipStream_t s, const char *what) {
  const int D = p.d <= 64 ? 64 : 128;
  const Layout w = span_layout(p, D);
  bind_workspace(p, w, ws);
  if (D == 64) launch_width<64>(p, cache_dtype, w.grid, s);
  else launch_width<128>(p, cache_dtype, w.grid, s);
  return check_hip(hipGetLastError(), what);
}

}  // namespace

size_t cross_workspace(const mia_cross_args &a) {
  SpanParams p = cross_params(a);
  return span_layout(p, p.d <= 64 ? 64 : 128).total;
}

size_t shared_prefix_workspace(const mia_shared_prefix_args &a) {
  SpanParams p = prefix_params(a);
  return span_layout(p, p.d <= 64 ? 64 : 128).total;
}

int launch_cross(const mia_cross_args &a, hipStream_t s) {
  SpanParams p = cross_params(a);
  return launch(p, a.cache_dtype, a.workspace, s, "cross_attention");
}

int launch_shared_prefix(const mia_shared_prefix_args &a, hipStream_t s) {
  SpanParams p = prefix_params(a);
  return launch(p, a.cache_dtype, a.workspace, s, "shared_prefix_attention");
}

}  // namespace mia
