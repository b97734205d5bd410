// span_attention.hip — attention of query rows over spans of keys of another
// length, bf16 MFMA on gfx950: cross attention (ragged queries over ragged
// encoder keys) and decode attention of a batch that shares a long prefix
// (one span for all rows, and each row's own span).
//
// Mathematics.  Every row of a (sequence, kv head) sees every key of its
// span: out = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m), s_k = scale q.k_k,
// accumulated over 64-key tiles with a running maximum m and sum l in fp32.
// Spans of the same row are joined by their (m, l, o).  Codes of a quantised
// cache are exact in bf16, so they go to the MFMA as they are: the scale of a
// key multiplies its score, the scale of its value the probability.
//
// Rows.  The query rows of one kv head are packed GQA-first: row r = pos * G
// + g is query token `pos` and q head h * G + g.  A segment is (sequence, kv
// head, tile of 128 rows); its keys are walked in 64-key tiles.
//
// Work split.  The tiles of all segments are laid end to end and cut into
// equal shares, one per workgroup (two workgroups per CU), whatever the
// lengths: each workgroup computes its share from the lengths on the device
// (a block scan), so a captured call follows its tensors.  A share begins and
// ends inside a segment; pieces of cut segments go to the workspace as fp32
// (o, m, l) and a second kernel joins them.
#include <algorithm>

#include "mia_device.h"
#include "mia_internal.h"

namespace mia {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

constexpr int kThreads = 256;
constexpr int kRows = 128;  // query rows per segment (4 waves x 32)
constexpr int kKT = 64;     // keys per tile

enum CacheKind { kBf16 = 0, kFp8 = 1, kI8 = 2 };

// One list of sequences and their key spans.
struct SpanList {
  int n;              // sequences
  const int32_t *cu;  // [n + 1] first query tokens, or NULL: tok_per each
  int tok_per;
  int tok_max;        // query tokens of a sequence at most
  const int32_t *len; // [n] keys
  int len_sub;        // subtracted from len
  int len_cap;        // keys the table (or the dense rows) can hold
  const int32_t *bt;  // block table, or NULL: block = sequence
  int64_t bt_s, bt_j;
  int cost;           // cost of a tile in the work split
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
  int64_t kc_blk, kc_h, kc_t, vc_blk, vc_h, vc_t;  // bytes
  const float *k_sc, *v_sc;  // per-key scales or NULL
  int64_t ks_blk, ks_h, ks_t, vs_blk, vs_h, vs_t;  // elements
  const float *k_deq, *v_deq;  // per-head scales or NULL
  const float *sink;
  int nb, bs;
  FastDiv bs_div;
  float scale_log2;
  SpanList list[2];
  int join;  // every piece goes to the workspace (rows have several spans)
  int *hdr;
  float *part_o;   // [partial row][D]
  float *part_ml;  // [partial row][2]
};

MIA_DEV int list_len(const SpanList &l, int i) {
  return max(0, min(l.len[i] - l.len_sub, l.len_cap));
}
// first query token and token count of sequence i
MIA_DEV int2 list_tokens(const SpanList &l, int i, int num_tokens) {
  int a, b;
  if (l.cu) {
    a = min(max(l.cu[i], 0), num_tokens);
    b = min(max(l.cu[i + 1], a), num_tokens);
  } else {
    a = min(i * l.tok_per, num_tokens);
    b = min(a + l.tok_per, num_tokens);
  }
  return make_int2(a, min(b - a, l.tok_max));
}
MIA_DEV int row_tiles(int rows) { return (rows + kRows - 1) / kRows; }

// Cost of sequence u of the joined lists.
MIA_DEV int64_t seq_cost(const SpanParams &p, int u) {
  const int li = u < p.list[0].n ? 0 : 1;
  const SpanList &l = p.list[li];
  const int i = li ? u - p.list[0].n : u;
  const int tiles = (list_len(l, i) + kKT - 1) / kKT;
  if (tiles == 0) return 0;
  const int rt = row_tiles(list_tokens(l, i, p.num_tokens).y * p.G);
  return (int64_t)tiles * rt * p.Hkv * l.cost;
}

// Workgroup whose share [floor(w N / W), floor((w + 1) N / W)) holds cost
// coordinate x: the largest w with floor(w N / W) <= x.
MIA_DEV int wg_of(int64_t x, int64_t n, int w) { return (int)(((x + 1) * w - 1) / n); }

// Where a workgroup's share starts, found by the plan.
struct Share {
  int64_t n;        // total cost
  int w_eff, w;     // workgroups with work, this one's number
  int64_t x0, x1;   // its cost range
  int u;            // first sequence with a tile at or past x0
  int64_t base;     // cost before that sequence
};

MIA_DEV int64_t read64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)readfirstlane((int)(x >> 32)) << 32) |
                   (uint32_t)readfirstlane((int)x));
}

// Block scan of the sequences' costs (each thread sums a contiguous run) and
// this workgroup's share.  scan: int64 [kThreads + 1] and found: int64 [4] in
// LDS.  With `hdr` the partials of every segment of the joined lists are
// listed there: hdr[2 g] = first partial, hdr[2 g + 1] = how many.
MIA_DEV bool plan_share(const SpanParams &p, int64_t *scan, int64_t *found, Share &sh) {
  const int tid = threadIdx.x;
  const int n_seq = p.list[0].n + p.list[1].n;
  const int per = (n_seq + kThreads - 1) / kThreads;
  const int u0 = min(tid * per, n_seq), u1 = min(u0 + per, n_seq);
  int64_t sum = 0;
  for (int u = u0; u < u1; ++u) sum += seq_cost(p, u);
  // exclusive scan over the threads
  scan[tid] = sum;
  __syncthreads();
  for (int o = 1; o < kThreads; o <<= 1) {
    const int64_t v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  const int64_t n = read64(scan[kThreads - 1]);
  const int64_t base = scan[tid] - sum;
  sh.n = n;
  // shares of at least two of the dearest tiles, so that every workgroup
  // between a segment's first and last has a piece of it
  const int64_t least = 2 * max(p.list[0].cost, p.list[1].cost);
  const int grid = gridDim.x;
  int w_eff = n == 0 ? 0 : (int)min((int64_t)grid, max((int64_t)1, n / least));
  // workgroups go round-robin over the 8 XCDs: neighbouring shares (the row
  // tiles of one head over the same keys) stay on one XCD's L2
  int w = blockIdx.x;
  if (w_eff >= 8) {
    w_eff &= ~7;
    w = (int)(blockIdx.x % 8) * (w_eff / 8) + blockIdx.x / 8;
    if ((int)(blockIdx.x / 8) >= w_eff / 8) w = w_eff;
  }
  sh.w_eff = w_eff;
  sh.w = w;
  if (p.join) {
    // every segment's partials (also those without any), by the workgroup of
    // its sequence
    int64_t x = base;
    for (int u = u0; u < u1; ++u) {
      const int li = u < p.list[0].n ? 0 : 1;
      const SpanList &l = p.list[li];
      const int i = li ? u - p.list[0].n : u;
      const int tiles = (list_len(l, i) + kKT - 1) / kKT;
      const int rt = row_tiles(list_tokens(l, i, p.num_tokens).y * p.G);
      const int segs = rt * p.Hkv;
      const int g0 = li ? row_tiles(p.num_tokens * p.G) * p.Hkv * p.list[0].n + i * segs : 0;
      const int g_in = li ? i * segs : 0;  // segment number inside its list
      if (u % grid == (int)blockIdx.x) {
        for (int s = 0; s < segs; ++s) {
          const int64_t xs = x + (int64_t)s * tiles * l.cost;
          int first = 0, cnt = 0;
          if (tiles > 0) {
            first = wg_of(xs, n, w_eff);
            cnt = wg_of(xs + (int64_t)(tiles - 1) * l.cost, n, w_eff) - first + 1;
          }
          p.hdr[2 * (g0 + s)] = g_in + s + first;
          p.hdr[2 * (g0 + s) + 1] = cnt;
        }
      }
      x += (int64_t)tiles * segs * l.cost;
    }
  } else if (tid == 0 && w < grid) {
    // the cut segment that starts in this share, if any, fills it in later
    if (w < w_eff) p.hdr[8 * w] = 0;
    else p.hdr[8 * blockIdx.x] = 0;
  }
  if (w >= w_eff) return false;
  sh.x0 = w * n / w_eff;
  sh.x1 = (int64_t)(w + 1) * n / w_eff;
  if (base <= sh.x0 && sh.x0 < base + sum) {
    int64_t x = base;
    for (int u = u0; u < u1; ++u) {
      const int64_t c = seq_cost(p, u);
      if (sh.x0 < x + c) {
        found[0] = u;
        found[1] = x;
        break;
      }
      x += c;
    }
  }
  __syncthreads();
  sh.u = readfirstlane((int)found[0]);
  sh.base = read64(found[1]);
  return true;
}

// A position in the stream of tiles: segment and tile (all wave-uniform).
struct Pos {
  int li, i;        // list, sequence
  int tok0, rows;   // first query token, rows (tokens x G)
  int len, tiles;   // keys, tiles
  int rt_n, rt, h;  // row tiles, this one, kv head
  int t;            // tile
  int64_t x;        // cost coordinate of the tile
  bool ok;          // inside the share
};

MIA_DEV void load_seq(const SpanParams &p, Pos &c) {
  const SpanList &l = p.list[c.li];
  const int2 tk = list_tokens(l, c.i, p.num_tokens);
  c.tok0 = readfirstlane(tk.x);
  c.rows = readfirstlane(tk.y * p.G);
  c.len = readfirstlane(list_len(l, c.i));
  c.tiles = (c.len + kKT - 1) / kKT;
  c.rt_n = row_tiles(c.rows);
}

// The first sequence at or after (li, i) with a tile and a row; clears ok
// past the last.
MIA_DEV void skip_empty(const SpanParams &p, Pos &c) {
  while (true) {
    if (c.i >= p.list[c.li].n) {
      if (c.li == 1) {
        c.ok = false;
        return;
      }
      c.li = 1;
      c.i = 0;
      continue;
    }
    load_seq(p, c);
    if (c.tiles > 0 && c.rt_n > 0) return;
    ++c.i;
  }
}

MIA_DEV Pos first_pos(const SpanParams &p, const Share &sh) {
  Pos c;
  c.ok = true;
  c.li = sh.u < p.list[0].n ? 0 : 1;
  c.i = c.li ? sh.u - p.list[0].n : sh.u;
  load_seq(p, c);
  const int cost = p.list[c.li].cost;
  const int64_t k = (sh.x0 - sh.base + cost - 1) / cost;  // tile of the sequence
  const int seg = (int)(k / c.tiles);
  c.t = (int)(k - (int64_t)seg * c.tiles);
  c.x = sh.base + k * cost;
  c.h = seg / c.rt_n;
  c.rt = seg - c.h * c.rt_n;
  if (c.h >= p.Hkv) {  // x0 lies behind the start of the sequence's last tile
    ++c.i;
    c.h = c.rt = c.t = 0;
    skip_empty(p, c);
  }
  if (c.x >= sh.x1) c.ok = false;
  return c;
}

MIA_DEV void advance(const SpanParams &p, const Share &sh, Pos &c) {
  c.x += p.list[c.li].cost;
  if (c.x >= sh.x1) {
    c.ok = false;
    return;
  }
  if (++c.t < c.tiles) return;
  c.t = 0;
  if (++c.rt < c.rt_n) return;
  c.rt = 0;
  if (++c.h < p.Hkv) return;
  c.h = 0;
  ++c.i;
  skip_empty(p, c);
}

MIA_DEV bool same_segment(const Pos &a, const Pos &b) {
  return a.li == b.li && a.i == b.i && a.h == b.h && a.rt == b.rt;
}

template <int D>
MIA_DEV constexpr int k_swz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
MIA_DEV constexpr int v_swz(int row) { return D == 128 ? (row & 3) << 2 : (row & 2) << 1; }

// 16 bytes of codes -> two 16-byte chunks of bf16 (exact).
template <int CT>
MIA_DEV void widen(u32x4_t w, u32x4_t (&out)[2]) {
  if constexpr (CT == kFp8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[i >> 1][(i & 1) * 2] = __builtin_bit_cast(
          uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, false));
      out[i >> 1][(i & 1) * 2 + 1] = __builtin_bit_cast(
          uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, true));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // bytes + 128 as unsigned, converted one by one
      const uint32_t u = w[i] ^ 0x80808080u;
      const float f0 = (float)(u & 0xffu) - 128.f, f1 = (float)((u >> 8) & 0xffu) - 128.f;
      const float f2 = (float)((u >> 16) & 0xffu) - 128.f, f3 = (float)(u >> 24) - 128.f;
      out[i >> 1][(i & 1) * 2] = pack2_bf16(f0, f1);
      out[i >> 1][(i & 1) * 2 + 1] = pack2_bf16(f2, f3);
    }
  }
}

MIA_DEV float row_max2(float x) {  // over the lanes l and l ^ 32 of a row
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
MIA_DEV float row_sum2(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// Address of token t's row of head h (t = b * S + s).
MIA_DEV int64_t tok_off(const SpanParams &p, int t, int64_t sb, int64_t ss) {
  const int b = (int)fdiv((uint32_t)t, p.s_div);
  return (int64_t)b * sb + (int64_t)(t - b * p.S) * ss;
}

// Rows of sequences without any key (cross attention): zeros.
MIA_DEV void zero_empty(const SpanParams &p) {
  const SpanList &l = p.list[1];
  for (int i = blockIdx.x; i < l.n; i += gridDim.x) {
    if (list_len(l, i) > 0) continue;
    const int2 tk = list_tokens(l, i, p.num_tokens);
    const int c8 = p.d / 8, hq = p.Hkv * p.G;
    for (int64_t k = threadIdx.x; k < (int64_t)tk.y * hq * c8; k += kThreads) {
      const int c = (int)(k % c8);
      const int h = (int)(k / c8 % hq);
      const int t = tk.x + (int)(k / ((int64_t)c8 * hq));
      uint16_t *op = p.out + tok_off(p, t, p.os_b, p.os_s) + (int64_t)h * p.os_h + c * 8;
      *reinterpret_cast<u32x2_t *>(op) = u32x2_t{0u, 0u};
      *reinterpret_cast<u32x2_t *>(op + 4) = u32x2_t{0u, 0u};
    }
  }
}

template <int D, int CT, bool SC>
__global__ __launch_bounds__(kThreads, 2) void span_kernel(SpanParams p) {
  static_assert(D == 64 || D == 128, "tile widths");
  static_assert(CT != kBf16 || !SC, "bf16 caches have no per-key scales");
  constexpr int EB = CT == kBf16 ? 2 : 1;
  constexpr int CE = 16 / EB;          // elements per 16-byte load
  constexpr int LPR = D / CE;          // lanes per key row
  constexpr int RPW = 64 / LPR;        // key rows per wave and load
  constexpr int RP = 4 * RPW;          // key rows per load of the workgroup
  constexpr int NP = kKT / RP;         // loads per thread and tile (K, V each)
  static_assert(RPW <= 16, "a wave's rows of a load lie in one 16-key group");
  constexpr int ROWB = D * 2;
  constexpr int TILEB = kKT * ROWB;
  constexpr int KSTEPS = D / 16;
  constexpr int DBLK = D / 32;

  __shared__ __attribute__((aligned(1024))) uint8_t kv_lds[2][2][TILEB];
  __shared__ __attribute__((aligned(16))) float sc_lds[2][2][SC ? kKT : 4];
  __shared__ int64_t found[2];

  if (!p.join) zero_empty(p);
  Share sh;
  if (!plan_share(p, reinterpret_cast<int64_t *>(&kv_lds[0][0][0]), found, sh)) return;
  __syncthreads();  // the scan's memory becomes tiles

  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int rl = lane & 31;
  lds_u8_t *const base = (lds_u8_t *)&kv_lds[0][0][0];

  // ---- loads of a tile: thread -> key row j * RP + lrow, chunk lc
  const int lrow = wave * RPW + lane / LPR;
  const int lc = lane % LPR;
  const int g16 = (wave * RPW) & ~15;  // 16-key group of load 0
  const bool ch_ok = lc * CE < p.d;
  u32x4_t kr[NP], vr[NP];
  float sr[NP];
  auto load_tile = [&](const Pos &c) {
    const SpanList &l = p.list[c.li];
    const int kt = c.t * kKT;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      // the group's block is wave-uniform; rows past the span read its last
      // key (in bounds) and are masked or cleared later
      const int k16 = min(kt + j * RP + g16, (c.len - 1) & ~15);
      int blk, off;
      if (l.bt) {
        const int bj = (int)fdiv((uint32_t)k16, p.bs_div);
        blk = l.bt[(int64_t)c.i * l.bt_s + (int64_t)bj * l.bt_j];
        blk = readfirstlane(min(max(blk, 0), p.nb - 1));
        off = k16 - bj * p.bs;
      } else {
        blk = c.i;
        off = k16;
      }
      const int rr = min(kt + j * RP + lrow, c.len - 1) - k16;
      const uint8_t *kb = p.k_cache + (int64_t)blk * p.kc_blk + (int64_t)c.h * p.kc_h +
                          (int64_t)off * p.kc_t;
      const uint8_t *vb = p.v_cache + (int64_t)blk * p.vc_blk + (int64_t)c.h * p.vc_h +
                          (int64_t)off * p.vc_t;
      kr[j] = u32x4_t{0u, 0u, 0u, 0u};
      vr[j] = u32x4_t{0u, 0u, 0u, 0u};
      if (ch_ok) {
        kr[j] = *reinterpret_cast<const u32x4_t *>(kb + rr * (int)p.kc_t + lc * 16);
        vr[j] = *reinterpret_cast<const u32x4_t *>(vb + rr * (int)p.vc_t + lc * 16);
      }
      if constexpr (SC) {
        const float *ks = p.k_sc + (int64_t)blk * p.ks_blk + (int64_t)c.h * p.ks_h +
                          (int64_t)off * p.ks_t;
        const float *vs = p.v_sc + (int64_t)blk * p.vs_blk + (int64_t)c.h * p.vs_h +
                          (int64_t)off * p.vs_t;
        sr[j] = 0.f;
        if (lc < 2) sr[j] = lc ? vs[rr * p.vs_t] : ks[rr * p.ks_t];
      }
    }
  };
  auto store_tile = [&](const Pos &c, int buf) {
    const int kt = c.t * kKT;
    lds_u8_t *const kb = base + (buf * 2) * TILEB;
    lds_u8_t *const vb = base + (buf * 2 + 1) * TILEB;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int row = j * RP + lrow;
      // values past the span are cleared: 0 * NaN would reach the sums
      const bool in = kt + row < c.len;
      const u32x4_t v = in ? vr[j] : u32x4_t{0u, 0u, 0u, 0u};
      if constexpr (CT == kBf16) {
        *(__attribute__((address_space(3))) u32x4_t *)(kb + row * ROWB +
                                                       ((lc ^ k_swz<D>(row)) << 4)) = kr[j];
        *(__attribute__((address_space(3))) u32x4_t *)(vb + row * ROWB +
                                                       ((lc ^ v_swz<D>(row)) << 4)) = v;
      } else {
        u32x4_t w[2];
        widen<CT>(kr[j], w);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *(__attribute__((address_space(3))) u32x4_t *)(
              kb + row * ROWB + (((2 * lc + x) ^ k_swz<D>(row)) << 4)) = w[x];
        widen<CT>(v, w);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *(__attribute__((address_space(3))) u32x4_t *)(
              vb + row * ROWB + (((2 * lc + x) ^ v_swz<D>(row)) << 4)) = w[x];
      }
      if constexpr (SC) {
        if (lc < 2) sc_lds[buf][lc][row] = in ? sr[j] : 0.f;
      }
    }
  };

  // ---- state of the current piece
  bf16x8_t qf[KSTEPS];
  f32x16_t acc[DBLK];
  float m_run = -INFINITY, l_run = 0.f;
  float c2 = 0.f;  // log2(e) x softmax scale x per-head scale of K
  auto begin_piece = [&](const Pos &c) {
    const int r = c.rt * kRows + wave * 32 + rl;
    const bool ok = r < c.rows;
    const int pos = (int)fdiv((uint32_t)(ok ? r : 0), p.g_div);
    const int hq = c.h * p.G + (ok ? r - pos * p.G : 0);
    const uint16_t *qp = p.q + tok_off(p, c.tok0 + pos, p.qs_b, p.qs_s) + (int64_t)hq * p.qs_h;
    float c1 = p.scale_log2;
    if (p.k_deq) c1 *= p.k_deq[c.h];
    // a negative factor goes to q, so that the largest product is the
    // largest score
    const uint32_t neg = c1 < 0.f ? 0x80008000u : 0u;
    c2 = fabsf(c1);
    if (c2 == 0.f) c2 = 1e-37f;  // masked scores (-inf) stay masked
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      u32x4_t w = {0u, 0u, 0u, 0u};
      const int d0 = ks * 16 + half * 8;
      if (ok && d0 < p.d) {
        w = *reinterpret_cast<const u32x4_t *>(qp + d0);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] ^= neg;
      }
      qf[ks] = __builtin_bit_cast(bf16x8_t, w);
    }
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    m_run = -INFINITY;
    l_run = 0.f;
  };

  const int tr_k = lane & 15;
  const int tr_col = ((lane >> 4) & 1) * 16 + 4 * (tr_k & 3);
  const int tr_row = half * 4 + (tr_k >> 2);

  auto compute = [&](const Pos &c, int buf) {
    const lds_u8_t *kb = base + (buf * 2) * TILEB;
    const lds_u8_t *vb = base + (buf * 2 + 1) * TILEB;
    // S^T = K . Q^T: lane = row rl, value e of block b: key b*32 + (e/4)*8 +
    // half*4 + e%4
    f32x16_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int row = b * 32 + rl;
        const u32x4_t kf = *(const __attribute__((address_space(3))) u32x4_t *)(
            kb + row * ROWB + (((ks * 2 + half) ^ k_swz<D>(row)) << 4));
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf), qf[ks],
                                                       s[b], 0, 0, 0);
      }
    }
    if constexpr (SC) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_t ks4 =
              *reinterpret_cast<const f32x4_t *>(&sc_lds[buf][0][b * 32 + g * 8 + half * 4]);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[b][g * 4 + i] *= ks4[i];
        }
    }
    const int left = c.len - c.t * kKT - half * 4;
    if (c.t == c.tiles - 1) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = b * 32 + (e >> 2) * 8 + (e & 3) < left ? s[b][e] : -INFINITY;
    }
    // online softmax; the maximum moves only when a score passes it by more
    // than 8 (log2 units): probabilities stay below 2^8, the accumulators are
    // rescaled on few tiles
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[b][e]);
    mx = row_max2(mx) * c2;
    const bool bump = mx > m_run + 8.f || (m_run == -INFINITY && mx > -INFINITY);
    if (__builtin_amdgcn_ballot_w64(bump)) {
      const float m_new = bump ? mx : m_run;
      const float alpha = m_run == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < DBLK; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= alpha;
    }
    const float nm = m_run == -INFINITY ? 0.f : -m_run;
    uint32_t pk[2][8];
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
          const f32x4_t vs4 =
              *reinterpret_cast<const f32x4_t *>(&sc_lds[buf][1][b * 32 + g * 8 + half * 4]);
#pragma unroll
          for (int i = 0; i < 4; ++i) pr[i] *= vs4[i];
        }
        // probabilities rounded to bf16 for the MFMA (half a step, 2^-9);
        // their sum keeps the unrounded ones
        pk[b][g * 2] = pack2_bf16(pr[0], pr[1]);
        pk[b][g * 2 + 1] = pack2_bf16(pr[2], pr[3]);
      }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    // O^T += V^T . P^T
#pragma unroll
    for (int k2 = 0; k2 < 4; ++k2) {
      const int b = k2 >> 1, kh = k2 & 1;
      const u32x4_t bw = {pk[b][kh * 4], pk[b][kh * 4 + 1], pk[b][kh * 4 + 2], pk[b][kh * 4 + 3]};
      const bf16x8_t bop = __builtin_bit_cast(bf16x8_t, bw);
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        u32x2_t t2[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int row = k2 * 16 + rr * 8 + tr_row;
          const int dd = db * 32 + tr_col;
          const int off = row * ROWB + (((dd >> 3) ^ v_swz<D>(row)) << 4) + ((dd & 7) << 1);
          t2[rr] = __builtin_bit_cast(
              u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vb + off)));
        }
        const u32x4_t vw = {t2[0][0], t2[0][1], t2[1][0], t2[1][1]};
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vw), bop,
                                                          acc[db], 0, 0, 0);
      }
    }
  };

  // ---- end of a piece: final rows, or a partial.  t0: its first tile, c:
  // its last
  auto end_piece = [&](const Pos &c, int t0) {
    const float l = row_sum2(l_run);
    const int rloc = wave * 32 + rl;
    const int r = c.rt * kRows + rloc;
    const bool whole = t0 == 0 && c.t == c.tiles - 1;
    const SpanList &ls = p.list[c.li];
    if (!p.join && whole) {
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
          if (d0 < p.d) {
            const u32x2_t w = {pack2_bf16(acc[i][g * 4] * inv, acc[i][g * 4 + 1] * inv),
                               pack2_bf16(acc[i][g * 4 + 2] * inv, acc[i][g * 4 + 3] * inv)};
            *reinterpret_cast<u32x2_t *>(op + d0) = w;
          }
        }
      return;
    }
    int64_t slot;
    if (p.join) {
      const int segs = c.rt_n * p.Hkv;
      slot = (int64_t)(c.li ? c.i * segs : 0) + c.h * c.rt_n + c.rt + sh.w;
    } else {
      slot = 2 * sh.w + (t0 == 0 ? 1 : 0);
      if (t0 == 0 && tid == 0) {
        const int cost = ls.cost;
        int *hd = p.hdr + 8 * sh.w;
        const int64_t x_last = c.x + (int64_t)(c.tiles - 1 - c.t) * cost;
        hd[1] = c.tok0;
        hd[2] = c.rows;
        hd[3] = c.rt;
        hd[4] = c.h;
        hd[0] = wg_of(x_last, sh.n, sh.w_eff) - sh.w + 1;
      }
    }
    if (r >= c.rows || rloc >= ls.part_rows) return;
    const int64_t pr = ls.part0 + slot * ls.part_rows + rloc;
    float *po = p.part_o + pr * D;
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t *>(po + i * 32 + g * 8 + half * 4) =
            f32x4_t{acc[i][g * 4], acc[i][g * 4 + 1], acc[i][g * 4 + 2], acc[i][g * 4 + 3]};
    if (half == 0) {
      p.part_ml[2 * pr] = m_run;
      p.part_ml[2 * pr + 1] = l;
    }
  };

  // ---- the stream: tile n is computed while tile n + 1 is in LDS's other
  // buffer or in flight
  Pos cur = first_pos(p, sh);
  if (!cur.ok) return;
  load_tile(cur);
  begin_piece(cur);
  store_tile(cur, 0);
  Pos nxt = cur;
  advance(p, sh, nxt);
  if (nxt.ok) load_tile(nxt);
  __syncthreads();
  int buf = 0, t0 = cur.t;
  while (true) {
    compute(cur, buf);
    if (!nxt.ok) {
      end_piece(cur, t0);
      return;
    }
    if (!same_segment(cur, nxt)) {
      end_piece(cur, t0);
      begin_piece(nxt);
      t0 = nxt.t;
    }
    store_tile(nxt, buf ^ 1);
    cur = nxt;
    advance(p, sh, nxt);
    if (nxt.ok) load_tile(nxt);
    __syncthreads();
    buf ^= 1;
  }
}

// Joins the pieces of cut segments (cross attention): workgroup (w, y) takes
// rows of the segment that starts, cut, in share w.
template <int D>
__global__ __launch_bounds__(256) void span_merge_kernel(SpanParams p) {
  const int w = blockIdx.x;
  const int *hd = p.hdr + 8 * w;
  const int n = hd[0];
  if (n == 0) return;
  constexpr int LPR = D / 4;
  constexpr int RPB = 256 / LPR;
  const int c = threadIdx.x % LPR;
  const SpanList &l = p.list[1];
  const int rloc = blockIdx.y * RPB + threadIdx.x / LPR;
  const int r = hd[3] * kRows + rloc;
  if (r >= hd[2] || rloc >= l.part_rows) return;
  auto prow = [&](int j) {
    return l.part0 + (int64_t)(j == 0 ? 2 * w + 1 : 2 * (w + j)) * l.part_rows + rloc;
  };
  float m = -INFINITY;
  for (int j = 0; j < n; ++j) m = fmaxf(m, p.part_ml[2 * prow(j)]);
  const float mm = m == -INFINITY ? 0.f : m;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float ls = 0.f;
  for (int j = 0; j < n; ++j) {
    const int64_t pr = prow(j);
    const float wgt = __builtin_amdgcn_exp2f(p.part_ml[2 * pr] - mm);
    ls += wgt * p.part_ml[2 * pr + 1];
    const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p.part_o + pr * D + c * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += wgt * v[i];
  }
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
template <int D, int CT, bool SC>
__global__ __launch_bounds__(256) void span_join_kernel(SpanParams p) {
  constexpr int LPR = D / 4;
  const int c = threadIdx.x % LPR;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int Hq = p.Hkv * p.G;
  if (row >= (int64_t)p.num_tokens * Hq) return;  // whole groups of LPR lanes leave
  const int t = (int)(row / Hq);
  const int hq = (int)(row - (int64_t)t * Hq);
  const int h = (int)fdiv((uint32_t)hq, p.g_div);
  const int g = hq - h * p.G;
  const int b = (int)fdiv((uint32_t)t, p.s_div);
  const int s = t - b * p.S;
  const SpanList &l0 = p.list[0], &l1 = p.list[1];
  const int rt0 = row_tiles(p.num_tokens * p.G), rt1 = row_tiles(p.S * p.G);
  const int r0 = t * p.G + g, r1 = s * p.G + g;
  const int seg0 = h * rt0 + r0 / kRows;
  const int seg1 = rt0 * p.Hkv * l0.n + (b * p.Hkv + h) * rt1 + r1 / kRows;
  int n0 = 0;
  int64_t f0 = 0;
  if (l0.n) {
    f0 = l0.part0 + (int64_t)p.hdr[2 * seg0] * l0.part_rows + r0 % kRows;
    n0 = p.hdr[2 * seg0 + 1];
  }
  const int64_t f1 = l1.part0 + (int64_t)p.hdr[2 * seg1] * l1.part_rows + r1 % kRows;
  const int n1 = p.hdr[2 * seg1 + 1];
  auto prow = [&](int j) {
    return j < n0 ? f0 + (int64_t)j * l0.part_rows : f1 + (int64_t)(j - n0) * l1.part_rows;
  };
  const int n = n0 + n1;
  float m = -INFINITY;
  for (int j = c; j < n; j += LPR) m = fmaxf(m, p.part_ml[2 * prow(j)]);
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if (p.sink) m = fmaxf(m, p.sink[hq] * kLog2e);
  float mm = m == -INFINITY ? 0.f : m;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float ls = p.sink ? __builtin_amdgcn_exp2f(p.sink[hq] * kLog2e - mm) : 0.f;
  for (int j = 0; j < n; ++j) {
    const int64_t pr = prow(j);
    const float wgt = __builtin_amdgcn_exp2f(p.part_ml[2 * pr] - mm);
    ls += wgt * p.part_ml[2 * pr + 1];
    const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p.part_o + pr * D + c * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += wgt * v[i];
  }
  // the keys between the span that all rows see and row s's own last key
  if (s > 0) {
    const int common = list_len(l1, b);
    const int end = min(l1.len[b] - l1.len_sub + s, l1.len_cap);
    if (common < end) {
      float qv[4] = {0.f, 0.f, 0.f, 0.f};
      const bool c_ok = c * 4 < p.d;
      if (c_ok) {
        const uint16_t *qp = p.q + (int64_t)b * p.qs_b + (int64_t)s * p.qs_s + (int64_t)hq * p.qs_h;
        const u32x2_t w = *reinterpret_cast<const u32x2_t *>(qp + c * 4);
        qv[0] = bf16lo(w[0]), qv[1] = bf16hi(w[0]), qv[2] = bf16lo(w[1]), qv[3] = bf16hi(w[1]);
      }
      float c1 = p.scale_log2;
      if (p.k_deq) c1 *= p.k_deq[h];
      auto load4 = [&](const uint8_t *a, float (&x)[4]) {
        if constexpr (CT == kBf16) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t *>(a + c * 8);
          x[0] = bf16lo(w[0]), x[1] = bf16hi(w[0]), x[2] = bf16lo(w[1]), x[3] = bf16hi(w[1]);
        } else {
          const uint32_t w = *reinterpret_cast<const uint32_t *>(a + c * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t byte = (w >> (8 * i)) & 0xffu;
            x[i] = CT == kI8 ? (float)(int8_t)byte : e4m3fn_bits_to_f32(byte);
          }
        }
      };
      for (int k = common; k < end; ++k) {
        const int bj = (int)fdiv((uint32_t)k, p.bs_div);
        const int blk = min(max(l1.bt[(int64_t)b * l1.bt_s + (int64_t)bj * l1.bt_j], 0), p.nb - 1);
        const int off = k - bj * p.bs;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
        if (c_ok) {
          load4(p.k_cache + (int64_t)blk * p.kc_blk + (int64_t)h * p.kc_h + (int64_t)off * p.kc_t, x);
          load4(p.v_cache + (int64_t)blk * p.vc_blk + (int64_t)h * p.vc_h + (int64_t)off * p.vc_t, v);
        }
        float dot = qv[0] * x[0] + qv[1] * x[1] + qv[2] * x[2] + qv[3] * x[3];
#pragma unroll
        for (int q = 1; q < LPR; q <<= 1) dot += __shfl_xor(dot, q, 64);
        float vs = 1.f;
        if constexpr (SC) {
          dot *= p.k_sc[(int64_t)blk * p.ks_blk + (int64_t)h * p.ks_h + (int64_t)off * p.ks_t];
          vs = p.v_sc[(int64_t)blk * p.vs_blk + (int64_t)h * p.vs_h + (int64_t)off * p.vs_t];
        }
        const float sc = dot * c1;
        const float m2 = fmaxf(m, sc);
        const float mm2 = m2 == -INFINITY ? 0.f : m2;
        const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm2);
        const float e = __builtin_amdgcn_exp2f(sc - mm2);
        m = m2;
        ls = ls * a + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * a + e * (v[i] * vs);
      }
    }
  }
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
int cu_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

struct Layout {
  int grid;
  size_t hdr, ml, o, total;  // byte offsets and size
  int64_t part_rows;
};

// Sizes of a call's workspace; fills the lists' partial regions.
Layout span_layout(SpanParams &p, int D) {
  Layout w;
  w.grid = 2 * cu_count();
  int64_t rows = 0, hdr = 0;
  if (p.join) {
    for (int li = 0; li < 2; ++li) {
      SpanList &l = p.list[li];
      const int64_t seq_rows = (li ? (int64_t)p.S : (int64_t)p.num_tokens) * p.G;
      const int64_t segs = (seq_rows + kRows - 1) / kRows * p.Hkv * l.n;
      l.part_rows = (int)std::min<int64_t>(kRows, seq_rows);
      l.part0 = rows;
      rows += (segs + w.grid) * l.part_rows;
      hdr += segs * 2;
    }
  } else {
    SpanList &l = p.list[1];
    l.part_rows = (int)std::min<int64_t>(kRows, (int64_t)l.tok_max * p.G);
    l.part0 = 0;
    rows = (int64_t)2 * w.grid * l.part_rows;
    hdr = (int64_t)8 * w.grid;
  }
  w.part_rows = rows;
  w.hdr = 0;
  w.ml = (size_t)up(hdr * 4, 256);
  w.o = w.ml + (size_t)up(rows * 8, 256);
  w.total = w.o + (size_t)rows * D * 4;
  return w;
}

void bind_workspace(SpanParams &p, const Layout &w, void *ws) {
  p.hdr = (int *)((uint8_t *)ws + w.hdr);
  p.part_ml = (float *)((uint8_t *)ws + w.ml);
  p.part_o = (float *)((uint8_t *)ws + w.o);
}

template <typename A>
void set_cache(SpanParams &p, const A &a) {
  const int eb = a.cache_dtype == MIA_DTYPE_BF16 ? 2 : 1;
  p.k_cache = (const uint8_t *)a.k_cache;
  p.v_cache = (const uint8_t *)a.v_cache;
  p.kc_blk = a.k_cache_stride[0] * eb, p.kc_h = a.k_cache_stride[1] * eb,
  p.kc_t = a.k_cache_stride[2] * eb;
  p.vc_blk = a.v_cache_stride[0] * eb, p.vc_h = a.v_cache_stride[1] * eb,
  p.vc_t = a.v_cache_stride[2] * eb;
  p.k_sc = a.k_scales, p.v_sc = a.v_scales;
  p.ks_blk = a.k_scale_stride[0], p.ks_h = a.k_scale_stride[1], p.ks_t = a.k_scale_stride[2];
  p.vs_blk = a.v_scale_stride[0], p.vs_h = a.v_scale_stride[1], p.vs_t = a.v_scale_stride[2];
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
  l.cost = 1;
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
  l0.cost = 1;
  l1.n = a.batch;
  l1.tok_per = l1.tok_max = a.s_active;
  l1.len = a.seq_lens;
  l1.len_sub = a.s_active - 1;
  l1.len_cap = a.blocks_per_seq * a.block_size;
  l1.bt = a.block_table, l1.bt_s = a.bt_stride[0], l1.bt_j = a.bt_stride[1];
  l1.cost = 1;
  return p;
}

template <int D, int CT, bool SC>
void launch_span(const SpanParams &p, int grid, hipStream_t s) {
  span_kernel<D, CT, SC><<<grid, kThreads, 0, s>>>(p);
  if (p.join) {
    const int64_t rows = (int64_t)p.num_tokens * p.Hkv * p.G;
    constexpr int RPB = 256 / (D / 4);
    span_join_kernel<D, CT, SC><<<(unsigned)((rows + RPB - 1) / RPB), 256, 0, s>>>(p);
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
    span_merge_kernel<D><<<dim3(grid, (l.part_rows + RPB - 1) / RPB), 256, 0, s>>>(p);
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
