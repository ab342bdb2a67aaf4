// Attention under masks (part of flash_fwd.hip, which includes this file once, after its helpers).
//
//   p_i  = q_start[b] + i                                     position of query row i among the keys
//   s_ij = scale q_i . k_j ;  s = cap tanh(s / cap) ;  s += bias[h, clamp(j - p_i, -R, R) + R]
//   row i sees the keys j < len_b of the document of p_i that are (causal) at most p_i or in the prefix
//   out_i = sum_j softmax_j(s_ij) v_j,  zeros for a row that sees nothing
//
// Every one of these masks leaves a row an interval [lo, hi) of keys, so a workgroup reads only the tiles
// from its rows' first key to their last, and tiles inside every row's interval need no mask at all.
//
// Rows: the P query heads that share a k/v head are rows beside each other (row r is query r / P, head r %
// P), so grouped heads read their keys once and a single token fills P rows of a tile.
//
// As in the unmasked kernel S^T = K Q^T is computed with the keys on the MFMA's row axis: a lane holds one
// query row (lane % 32), its interval, its running max and sum, and P^T goes from the accumulator to O^T +=
// V^T P^T without a shuffle.  Scores are kept in units of log2(e): the largest finite bias stays finite.
//
// A masked key's weight is an exact 0, and 0 times a NaN or an infinity in its v row must not reach the
// output: tiles that need a mask are looked over, and where such a value is found their products are formed
// one by one for the keys that a row sees (exact_pv).

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<bf16> {
  typedef bf16x8 x8;
  typedef bf16x4 x4;
  typedef bf16x2 x2;
  static constexpr uint32_t kExpBits = 0x7f80;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // c + the sum of both values
  static __device__ __forceinline__ float add2(x2 v, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(v, x2{(bf16)1.0f, (bf16)1.0f}, c, false);
  }
};
template <> struct Elem<_Float16> {
  typedef f16x8 x8;
  typedef f16x4 x4;
  typedef f16x2 x2;
  static constexpr uint32_t kExpBits = 0x7c00;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(x2 v, float c) {
    return __builtin_amdgcn_fdot2(v, x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
  }
};

// ---------------------------------------------------------------------------
// tiles of keys in LDS: rows of HD channels in 16-byte chunks, chunk c of row r at position c ^ swizzle(r)
// ---------------------------------------------------------------------------

// k: the 16 rows that a phase of an operand read takes one chunk of lie on 16 distinct bank groups of 16
// bytes (of 256 bytes: one row of 128 channels, two of 64)
template <int HD> __device__ __forceinline__ int mk_swz(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
// v: the 4 rows x 4 chunks of a transposed read do
template <int HD> __device__ __forceinline__ int mv_swz(int row) { return HD == 128 ? (row & 3) << 2 : (row & 2) << 1; }

// Copies of a tile of KEYS rows in 1 KB blocks, wave w of NW issuing blocks w, w + NW, ...
template <int HD, int KEYS, int NW, bool V>
struct MaskedCopy {
  static constexpr int kRows = 512 / HD, kCpr = HD / 8;     // rows of a block, chunks of a row
  static constexpr int kPer = KEYS / kRows / NW;            // copies of a wave
  const char* base;        // key 0 of the (sample, head)
  int64_t row_bytes;
  uint32_t off[kPer];

  static __device__ __forceinline__ int row_of(int wave, int lane, int u) {
    return kRows * (wave + NW * u) + lane / kCpr;
  }
  static __device__ __forceinline__ int col_of(int row, int lane) {     // bytes
    return ((lane % kCpr) ^ (V ? mv_swz<HD>(row) : mk_swz<HD>(row))) * 16;
  }
  __device__ __forceinline__ void init(const void* p, int64_t stride, int wave, int lane) {
    base = static_cast<const char*>(p);
    row_bytes = stride * 2;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int row = row_of(wave, lane, u);
      off[u] = (uint32_t)(row * row_bytes) + col_of(row, lane);
    }
  }
  // Tile t into `dst`; rows past the tensor's last key repeat it.
  __device__ __forceinline__ void issue(int t, int keys, bf16* dst, int wave, int lane) const {
    const int k0 = t * KEYS;
    if (k0 + KEYS <= keys) {
      const char* tb = base + (int64_t)k0 * row_bytes;
#pragma unroll
      for (int u = 0; u < kPer; ++u) dma16_saddr(tb, off[u], lds_addr(dst + (wave + NW * u) * 512));
    } else {
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int row = row_of(wave, lane, u);
        const int key = min(k0 + row, keys - 1);
        dma16_vaddr(base + (int64_t)key * row_bytes + col_of(row, lane), lds_addr(dst + (wave + NW * u) * 512));
      }
    }
  }
};

// ---------------------------------------------------------------------------
// rows and their intervals
// ---------------------------------------------------------------------------

struct MaskedRow {
  int p, lo, hi;      // position; keys seen: [lo, hi), empty rows [0, 0)
};

__device__ __forceinline__ MaskedRow masked_row(const MaskedArgs& a, int b, int i) {
  MaskedRow r;
  const int start = a.q_start != nullptr ? a.q_start[b] : a.Lk - a.Lq;
  r.p = max(min(start, kMaxPosition), -kMaxPosition) + i;
  int len = a.Lk;
  if (a.seqlen_k != nullptr) len = min(max(a.seqlen_k[b], 0), a.Lk);
  int lo = 0, hi = len, prefix = 0;
  bool any = true;
  if (a.doc_starts != nullptr) {
    const int32_t* d = a.doc_starts + (int64_t)b * a.docs;
    int n = 0;                               // starts at or before p (they grow)
    for (int step = a.docs, at = 0; step > 0;) {
      const int half = step >> 1;
      if (d[at + half] <= r.p) {
        at += half + 1;
        step -= half + 1;
      } else {
        step = half;
      }
      n = at;
    }
    any = n > 0;
    if (any) {
      lo = max(d[n - 1], 0);
      if (n < a.docs) hi = min(hi, d[n]);
      if (a.prefix_lens != nullptr) prefix = a.prefix_lens[(int64_t)b * a.docs + n - 1];
    }
  } else if (a.prefix_lens != nullptr) {
    prefix = a.prefix_lens[b];
  }
  if (a.causal) {
    const int64_t shared = (int64_t)lo + prefix, past = (int64_t)r.p + 1;
    hi = (int)min((int64_t)hi, max(shared, past));
  }
  any = any && lo < hi;
  r.lo = any ? lo : 0;
  r.hi = any ? hi : 0;
  return r;
}

// min / max over the wave's 32 rows (lanes 32 apart hold the same)
__device__ __forceinline__ int rows_min(int v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v = min(v, __shfl_xor(v, m));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int rows_max(int v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v = max(v, __shfl_xor(v, m));
  return __builtin_amdgcn_readfirstlane(v);
}

// Which rows a block number stands for.
struct MaskedBlock {
  int b, h0, hk, rb;      // sample, first of the P query heads, their k/v head, block of rows
  __device__ __forceinline__ MaskedBlock(const MaskedArgs& a, int id, int blocks) {
    const int unit = id / blocks, per = a.Hq / a.pack;
    const int sample = unit / per, first = (unit - sample * per) * a.pack;
    rb = uniform(id - unit * blocks);
    b = uniform(sample);
    h0 = uniform(first);
    hk = uniform(first / (a.Hq / a.Hk));
  }
  // (divisions are vector arithmetic: their results go back to scalar registers, from which the tile
  // copies take their addresses)
  static __device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
};

// Part `part` of the tiles [t0, t0 + n): [first, end).
struct TileRange {
  int first, end;
  __device__ __forceinline__ TileRange(int t0, int n, int part, int parts) {
    const int each = n / parts, over = n - each * parts;
    first = MaskedBlock::uniform(t0 + each * part + min(part, over));
    end = MaskedBlock::uniform(t0 + each * (part + 1) + min(part + 1, over));
  }
};

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------

// The softmax's arithmetic on one lane's scores.  CAP: capped by a tanh.  BIAS: a table entry added.
// Without either the scores stay as the MFMA leaves them and the scale is folded into the exponent.
template <bool CAP, bool BIAS>
struct ScoreMap {
  float sl2;            // scale * log2(e)
  float cap2, k;        // cap * log2(e); 2 log2(e) scale / cap, or scale / cap with small_ok
  bool precise;

  __device__ __forceinline__ void init(const MaskedArgs& a) {
    sl2 = a.scale * kLog2e;
    cap2 = a.cap * kLog2e;
    precise = a.cap > kExactCap;
    k = CAP ? (precise ? a.scale / a.cap : 2.f * kLog2e * a.scale / a.cap) : 0.f;
  }
  // Scores in units of log2(e), without bias.
  // tanh(y) = 1 - 2 / (1 + e^2y): off by 2^-22 of the cap at most, which up to caps of 256 is less than the
  // rounding of the softmax weights; beyond, small y go by the series y - y^3/3 + 2 y^5/15.
  __device__ __forceinline__ void map(f32x16& s) const {
    if constexpr (CAP) {
      if (precise) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float y = s[r] * k, y2 = y * y;
          const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + fast_exp2(y * (2.f * kLog2e))), 1.f);
          const float near = fmaf(y * y2, fmaf(y2, 2.f / 15.f, -1.f / 3.f), y);
          s[r] = cap2 * (fabsf(y) < 0.1f ? near : far);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + fast_exp2(s[r] * k)), cap2);
      }
    } else if constexpr (BIAS) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= sl2;
    }
  }
  // exponent of a score against the reference point m
  __device__ __forceinline__ float weight(float s, float m) const {
    if constexpr (CAP || BIAS) return fast_exp2(s - m);
    else return fast_exp2(fmaf(s, sl2, -m));
  }
  // a max of scores in the units of m
  __device__ __forceinline__ float top(float s) const { return CAP || BIAS ? s : s * sl2; }
};

// A bias entry in units of log2(e).  What is finite stays finite: a table may hold the type's lowest value
// for "never", and rows of nothing else are uniform as they are without a bias.
__device__ __forceinline__ float bias_units(float v) {
  const float w = v * kLog2e;
  return fabsf(v) < INFINITY ? fmaxf(fminf(w, FLT_MAX), -FLT_MAX) : w;
}

// The distances that coming tiles need, of the P heads of a block, in LDS: entry (g, d - w0).
struct BiasWindow {
  int w0, end;        // distances held: [w0, end)
  int per;            // entries of a head
  __device__ __forceinline__ void init(int floats, int pack) {
    per = floats / pack;
    w0 = end = 0;
  }
  __device__ __forceinline__ bool holds(int first, int last) const { return first >= w0 && last < end; }
  // Entries from distance `first` on, `want` of them at most, by threads id of n.
  __device__ __forceinline__ void load(const MaskedArgs& a, int h0, int first, int64_t want, float* lds, int id, int n) {
    const int count = (int)min((int64_t)per, want);
    const int width = 2 * a.reach + 1;
    for (int g = 0; g < a.pack; ++g) {
      const float* row = a.bias + (int64_t)(h0 + g) * width + a.reach;
      for (int e = id; e < count; e += n) {
        const int d = max(min(first + e, a.reach), -a.reach);
        lds[g * per + e] = bias_units(row[d]);
      }
    }
    w0 = first;
    end = first + count;
  }
};

// ---------------------------------------------------------------------------
// products with v
// ---------------------------------------------------------------------------

// Whether a tile in LDS holds a NaN or an infinity (one answer for the wave).
template <typename T, int HD, int KEYS>
__device__ __forceinline__ bool tile_not_finite(const bf16* Vt, int lane) {
  constexpr uint32_t M = Elem<T>::kExpBits * 0x10001u;
  u16x2 top = {0, 0};
#pragma unroll
  for (int i = 0; i < KEYS * HD / 512; ++i) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(Vt + i * 512 + lane * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[j] & M));
  }
  return __builtin_amdgcn_ballot_w64(top[0] == Elem<T>::kExpBits || top[1] == Elem<T>::kExpBits) != 0;
}

// O^T += V^T P^T of 16 keys, product by product, of the keys from key0 on that this lane's row sees.
// `buf`: 1 KB of this wave's.
template <typename T, int HD>
__device__ __forceinline__ void exact_pv(f32x16 (&o)[HD / 32], typename Elem<T>::x8 pb, const bf16* Vt, int row0, int key0,
                                         const MaskedRow& m, T* buf, int lane) {
  typedef typename Elem<T>::x4 X4;
  const int n32 = lane & 31, hh = lane >> 5;
  // this lane's weights are of keys 4 hh .. +3 and 8 + 4 hh .. +3
  *reinterpret_cast<X4*>(buf + n32 * 16 + 4 * hh) = X4{pb[0], pb[1], pb[2], pb[3]};
  *reinterpret_cast<X4*>(buf + n32 * 16 + 8 + 4 * hh) = X4{pb[4], pb[5], pb[6], pb[7]};
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma nounroll
  for (int kk = 0; kk < 16; ++kk) {
    const float p = (float)buf[n32 * 16 + kk];
    const bool sees = key0 + kk >= m.lo && key0 + kk < m.hi;
    const T* row = reinterpret_cast<const T*>(Vt) + (row0 + kk) * HD;
    const int x = mv_swz<HD>(row0 + kk);
#pragma unroll
    for (int md = 0; md < HD / 32; ++md)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const X4 v = *reinterpret_cast<const X4*>(row + (((4 * md + g) ^ x) << 3) + 4 * hh);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[md][4 * g + e] = sees ? fmaf(p, (float)v[e], o[md][4 * g + e]) : o[md][4 * g + e];
      }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// What a lane reads of the tiles, and its Q fragments.
template <typename T, int HD>
struct MaskedOperands {
  typedef typename Elem<T>::x8 X8;
  X8 qf[HD / 16];       // query row lane % 32, channels 16 ks + 8 hh ..
  int k_rd[HD / 16];
  int v_rd[HD / 32];

  __device__ __forceinline__ void init(const void* q, int lane) {
    const int n32 = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      qf[ks] = *reinterpret_cast<const X8*>(static_cast<const T*>(q) + 16 * ks + 8 * hh);
      k_rd[ks] = n32 * HD + (((2 * ks + hh) ^ mk_swz<HD>(n32)) << 3);
    }
    const int row = 4 * hh + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int md = 0; md < HD / 32; ++md)
      v_rd[md] = row * HD + (((4 * md + chunk) ^ mv_swz<HD>(row)) << 3) + 4 * (lane & 1);
  }
  __device__ __forceinline__ X8 k_frag(const bf16* Kt, int ks, int row0) const {
    return *reinterpret_cast<const X8*>(Kt + row0 * HD + k_rd[ks]);
  }
  // V^T rows 32 md .., keys of MFMA step ksp in the accumulator's order
  __device__ __forceinline__ X8 v_frag(const bf16* Vt, int ksp, int md) const {
    const bf16* p = Vt + 16 * ksp * HD + v_rd[md];
    const i16x4 lo = lds_read_tr(p), hi = lds_read_tr(p + 8 * HD);
    return __builtin_bit_cast(X8, (short __attribute__((ext_vector_type(8)))){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1],
                                                                              hi[2], hi[3]});
  }
};

// The interval test of the 16 keys that a lane's accumulator holds, from key kt on: masked scores become -inf.
__device__ __forceinline__ void mask_scores(f32x16& s, int kt, int hh, const MaskedRow& m) {
  const uint32_t n = (uint32_t)(m.hi - m.lo);
  const int first = kt + 4 * hh - m.lo;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if ((uint32_t)(first + 8 * (r >> 2) + (r & 3)) >= n) s[r] = -INFINITY;
}

__device__ __forceinline__ float max16(const f32x16& s) {
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int r = 2; r < 16; ++r) mx = fmaxf(mx, s[r]);
  return mx;
}

// ---------------------------------------------------------------------------
// few rows: 32 rows a workgroup, its four waves on every fourth tile of 32 keys
// ---------------------------------------------------------------------------

constexpr int kStepWaves = 4, kStepKeys = 32;
constexpr int kStepWindow = 1200;       // bias entries of a wave

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(kStepWaves * 64, 1) void masked_step_kernel(const MaskedArgs a) {
  typedef typename Elem<T>::x8 X8;
  constexpr int kTile = kStepKeys * HD;       // elements
  __shared__ __attribute__((aligned(1024))) bf16 tiles[kStepWaves][2][2][kTile];     // [wave][slot][k, v]
  __shared__ __attribute__((aligned(16))) T exact_buf[kStepWaves][32 * 16];
  __shared__ float window[kStepWaves][BIAS ? kStepWindow : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int rows = a.Lq * a.pack, blocks = (rows + 31) / 32;
  const int slot_id = blockIdx.x / a.splits, part = blockIdx.x - slot_id * a.splits;
  const MaskedBlock blk(a, slot_id, blocks);
  // (rows past the last one repeat it; they are not stored)
  const int r = min(blk.rb * 32 + n32, rows - 1), i = r / a.pack, g = r - i * a.pack;
  const MaskedRow m = masked_row(a, blk.b, i);

  // this part's tiles
  const bool some = m.lo < m.hi;
  const int first = rows_min(some ? m.lo : 0x7fffffff), end = rows_max(m.hi);
  const int all_lo = rows_max(m.lo), all_hi = rows_min(m.hi);     // what every row sees: [all_lo, all_hi)
  const int t0 = first / kStepKeys;
  const TileRange range(t0, first < end ? (end - 1) / kStepKeys + 1 - t0 : 0, part, a.splits);
  const int tb = range.end;

  MaskedCopy<HD, kStepKeys, 1, false> kc;
  MaskedCopy<HD, kStepKeys, 1, true> vc;
  kc.init(static_cast<const T*>(a.k.ptr) + blk.b * a.k.sb + blk.hk * a.k.sh, a.k.st, 0, lane);
  vc.init(static_cast<const T*>(a.v.ptr) + blk.b * a.v.sb + blk.hk * a.v.sh, a.v.st, 0, lane);
  auto issue = [&](int t, int slot) {
    kc.issue(t, a.Lk, tiles[wave][slot][0], 0, lane);
    vc.issue(t, a.Lk, tiles[wave][slot][1], 0, lane);
  };
  int t = range.first + wave;
  if (t < tb) issue(t, 0);
  if (t + kStepWaves < tb) issue(t + kStepWaves, 1);

  MaskedOperands<T, HD> op;
  op.init(static_cast<const T*>(a.q.ptr) + blk.b * a.q.sb + (int64_t)i * a.q.st + (blk.h0 + g) * a.q.sh, lane);
  ScoreMap<CAP, BIAS> map;
  map.init(a);
  BiasWindow win;
  if (BIAS) win.init(kStepWindow, a.pack);
  const int p_max = rows_max(m.p), p_min = rows_min(m.p);

  f32x16 o[HD / 32];
#pragma unroll
  for (int md = 0; md < HD / 32; ++md) o[md] = f32x16{};
  float m_run = -FLT_MAX, l_run = 0.f;

  for (int slot = 0; t < tb; t += kStepWaves, slot ^= 1) {
    const int kt = t * kStepKeys;
    const bf16 *Kt = tiles[wave][slot][0], *Vt = tiles[wave][slot][1];
    if (BIAS && !win.holds(kt - p_max, kt + kStepKeys - 1 - p_min)) {
      win.load(a, blk.h0, kt - p_max, (int64_t)(tb - t) * kStepKeys + (p_max - p_min), window[wave], lane, 64);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // this tile has landed; the next one's copies stay in flight
    if (t + kStepWaves < tb)
      asm volatile("s_waitcnt vmcnt(%0)" :: "i"(2 * decltype(kc)::kPer) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) s = Elem<T>::mfma(op.k_frag(Kt, ks, 0), op.qf[ks], s);
    map.map(s);
    if constexpr (BIAS) {
      const float* w = window[wave] + g * win.per + (kt + 4 * hh - m.p - win.w0);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] += w[8 * (e >> 2) + (e & 3)];
    }
    const bool masked = kt < all_lo || kt + kStepKeys > all_hi;
    if (masked) mask_scores(s, kt, hh, m);

    const float m_new = fmaxf(m_run, map.top(pair_max(max16(s))));
    if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
      const float alpha = fast_exp2(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int md = 0; md < HD / 32; ++md) o[md] *= alpha;
      m_run = m_new;
    }
    X8 pb[2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      typename Elem<T>::x2 w = {(T)map.weight(s[e], m_run), (T)map.weight(s[e + 1], m_run)};
      pb[e >> 3][e & 7] = w[0];
      pb[e >> 3][(e & 7) + 1] = w[1];
      l_run = Elem<T>::add2(w, l_run);      // the sum of the rounded weights that the products use
    }
    if (masked && tile_not_finite<T, HD, kStepKeys>(Vt, lane)) {
#pragma unroll
      for (int ksp = 0; ksp < 2; ++ksp) exact_pv<T, HD>(o, pb[ksp], Vt, 16 * ksp, kt + 16 * ksp, m, exact_buf[wave], lane);
    } else {
#pragma unroll
      for (int ksp = 0; ksp < 2; ++ksp)
#pragma unroll
        for (int md = 0; md < HD / 32; ++md) o[md] = Elem<T>::mfma(op.v_frag(Vt, ksp, md), pb[ksp], o[md]);
    }
    // every read of this slot has returned before it is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + 2 * kStepWaves < tb) issue(t + 2 * kStepWaves, slot);
  }
  l_run = pair_sum(l_run);

  // The four waves' results through LDS: O [32][HD + 4], then each row's weights.
  constexpr int kRow = HD + 4;
  static_assert(kStepWaves * 32 * (kRow + 2) * 4 <= (int)sizeof(tiles), "the tiles hold the waves' results");
  __syncthreads();
  float* const all = reinterpret_cast<float*>(&tiles[0][0][0][0]);
  float* const mine = all + wave * (32 * kRow);
  float* const stat = all + kStepWaves * (32 * kRow);       // m [4][32], l [4][32]
#pragma unroll
  for (int md = 0; md < HD / 32; ++md)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(mine + n32 * kRow + 32 * md + 8 * q + 4 * hh) =
          f32x4{o[md][4 * q], o[md][4 * q + 1], o[md][4 * q + 2], o[md][4 * q + 3]};
  if (hh == 0) {
    stat[wave * 32 + n32] = m_run;
    stat[(kStepWaves + wave) * 32 + n32] = l_run;
  }
  __syncthreads();
  const int held = min(rows - blk.rb * 32, 32);             // rows of this block
  for (int x = threadIdx.x; x < held * (HD / 8); x += kStepWaves * 64) {
    const int row = x / (HD / 8), c = x - row * (HD / 8);
    float top = stat[row], l = 0.f;
#pragma unroll
    for (int w = 1; w < kStepWaves; ++w) top = fmaxf(top, stat[w * 32 + row]);
    float v[8] = {};
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) {
      const float f = fast_exp2(stat[w * 32 + row] - top);
      l += f * stat[(kStepWaves + w) * 32 + row];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(f, all[w * (32 * kRow) + row * kRow + 8 * c + e], v[e]);
    }
    if (a.splits > 1) {
      float* p = a.part + (int64_t)blockIdx.x * a.part_floats + row * HD + 8 * c;
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
      if (c == 0) {
        float* st = a.part + (int64_t)blockIdx.x * a.part_floats + a.part_rows * HD;
        st[row] = top;
        st[a.part_rows + row] = l;
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int rr = blk.rb * 32 + row, qi = rr / a.pack;
      X8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (T)(v[e] * inv);
      *reinterpret_cast<X8*>(static_cast<T*>(a.o) + blk.b * a.o_sb + (int64_t)qi * a.o_st +
                             (blk.h0 + rr - qi * a.pack) * a.o_sh + 8 * c) = y;
    }
  }
}

// Rows whose keys were split: O = sum_i w_i O_i / sum_i w_i l_i with w_i = exp2(m_i - max m).  A wave a row.
template <typename T, int HD>
__global__ __launch_bounds__(256) void masked_merge_kernel(const MaskedArgs a, int block_rows) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int rows = a.Lq * a.pack, blocks = (rows + block_rows - 1) / block_rows;
  const int64_t unit = id / rows;
  if (unit >= (int64_t)a.B * (a.Hq / a.pack)) return;
  const int r = (int)(id - unit * rows), rb = r / block_rows, row = r - rb * block_rows;
  const float* p0 = a.part + (unit * blocks + rb) * a.splits * a.part_floats;
  const float* st = p0 + a.part_rows * HD + row;
  float top = -FLT_MAX;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, st[s * a.part_floats]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  float v[HD / 64] = {}, l = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float* q = st + s * a.part_floats;
    const float f = fast_exp2(q[0] - top);
    l += f * q[a.part_rows];
#pragma unroll
    for (int e = 0; e < HD / 64; ++e)
      v[e] = fmaf(f, p0[s * a.part_floats + row * HD + (HD / 64) * lane + e], v[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int per = a.Hq / a.pack, b = (int)(unit / per), h0 = (int)(unit - (int64_t)b * per) * a.pack;
  const int qi = r / a.pack;
  T* o = static_cast<T*>(a.o) + b * a.o_sb + (int64_t)qi * a.o_st + (h0 + r - qi * a.pack) * a.o_sh + (HD / 64) * lane;
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) o[e] = (T)(v[e] * inv);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T, int HD, bool CAP, bool BIAS>
int launch_masked(MaskedArgs a, const MaskedPlan& p, hipStream_t s) {
  hipLaunchKernelGGL((masked_step_kernel<T, HD, CAP, BIAS>), dim3((unsigned)(p.blocks * p.splits)), dim3(kStepWaves * 64),
                     0, s, a);
  if (p.splits > 1)
    hipLaunchKernelGGL((masked_merge_kernel<T, HD>), dim3((unsigned)((p.out_rows + 3) / 4)), dim3(256), 0, s, a,
                       p.block_rows);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : set_error(4, "masked_attn launch: %s", hipGetErrorString(e));
}

template <typename T, int HD>
int launch_masked_map(const MaskedArgs& a, const MaskedPlan& p, hipStream_t s) {
  if (a.bias != nullptr)
    return a.cap > 0.f ? launch_masked<T, HD, true, true>(a, p, s) : launch_masked<T, HD, false, true>(a, p, s);
  return a.cap > 0.f ? launch_masked<T, HD, true, false>(a, p, s) : launch_masked<T, HD, false, false>(a, p, s);
}
