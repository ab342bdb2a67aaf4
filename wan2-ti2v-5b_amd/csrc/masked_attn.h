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
// output: tiles that need a mask are looked over, and where such a value is found it goes to the rows alone
// that see it (exact_pv).

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
  // Tile t, all of whose keys there are, into `dst`.
  __device__ __forceinline__ void issue_full(int t, bf16* dst, int wave) const {
    const char* tb = base + (int64_t)(t * KEYS) * row_bytes;
#pragma unroll
    for (int u = 0; u < kPer; ++u) dma16_saddr(tb, off[u], lds_addr(dst + (wave + NW * u) * 512));
  }
  // Tile t into `dst`; rows past the tensor's last key repeat it.
  __device__ __forceinline__ void issue(int t, int keys, bf16* dst, int wave, int lane) const {
    const int k0 = t * KEYS;
    if (k0 + KEYS <= keys) {
      issue_full(t, dst, wave);
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

__device__ __forceinline__ int first_position(const MaskedArgs& a, int b) {
  const int start = a.q_start != nullptr ? a.q_start[b] : a.Lk - a.Lq;
  return max(min(start, kMaxPosition), -kMaxPosition);
}

__device__ __forceinline__ MaskedRow masked_row(const MaskedArgs& a, int b, int i) {
  MaskedRow r;
  r.p = first_position(a, b) + i;
  int len = a.Lk;
  if (a.seqlen_k != nullptr) len = min(max(a.seqlen_k[b], 0), a.Lk);
  int lo = 0, hi = len, begin = 0, prefix = 0;      // begin: where the document does, be there a key or not
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
      begin = d[n - 1];
      lo = max(begin, 0);
      if (n < a.docs) hi = min(hi, d[n]);
      if (a.prefix_lens != nullptr) prefix = a.prefix_lens[(int64_t)b * a.docs + n - 1];
    }
  } else if (a.prefix_lens != nullptr) {
    prefix = a.prefix_lens[b];
  }
  if (a.causal) {
    const int64_t shared = (int64_t)begin + prefix, past = (int64_t)r.p + 1;
    hi = (int)min((int64_t)hi, max(shared, past));
  }
  any = any && lo < hi;
  r.lo = any ? lo : 0;
  r.hi = any ? hi : 0;
  return r;
}

// min / max over the wave's 32 rows (lanes 32 apart hold the same): within 16 lanes by rotations, then the two
// halves as scalars.
template <int N>
__device__ __forceinline__ int row_turn(int v) {       // the value N lanes on, in the lane's 16
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + N, 0xf, 0xf, false);
}
__device__ __forceinline__ int rows_min(int v) {
  v = min(v, row_turn<8>(v));
  v = min(v, row_turn<4>(v));
  v = min(v, row_turn<2>(v));
  v = min(v, row_turn<1>(v));
  return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
__device__ __forceinline__ int rows_max(int v) {
  v = max(v, row_turn<8>(v));
  v = max(v, row_turn<4>(v));
  v = max(v, row_turn<2>(v));
  v = max(v, row_turn<1>(v));
  return max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}

// The sample and heads of a unit.  The heads vary fastest: workgroup i runs on XCD i % 8, and every XCD has units of
// long and of short samples.
struct MaskedUnit {
  int b, h0, hk;          // sample, first of the P query heads, their k/v head
  __device__ __forceinline__ MaskedUnit(const MaskedArgs& a, int unit) {
    b = uniform(a.by_heads(unit));
    h0 = uniform((unit - b * a.head_groups) * a.pack);
    hk = uniform(a.by_group(h0));
  }
  // (the tile copies take their addresses from scalar registers)
  static __device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
};

// Part `part` of the tiles [t0, t0 + n): [first, end).
struct TileRange {
  int first, end;
  __device__ __forceinline__ TileRange(int t0, int n, int part, int parts) {
    if (parts == 1) {
      first = t0;
      end = t0 + n;
      return;
    }
    const int each = n / parts, over = n - each * parts;
    first = MaskedUnit::uniform(t0 + each * part + min(part, over));
    end = MaskedUnit::uniform(t0 + each * (part + 1) + min(part + 1, over));
  }
};

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------

// The softmax's arithmetic on one lane's scores.  CAP: capped by a tanh.  BIAS: a table entry added.
// map() leaves a value that times `factor` (plus the bias) is the score in units of log2(e): without CAP the MFMA's
// own, with it tanh(y), y = s scale / cap.  Where all of the wave's |y| are at most 1/4 that is the series
// y - y^3/3 + 2 y^5/15 - 17 y^7/315, off by 2^-23 at most, in five operations; its usual form 1 - 2 / (1 + e^2y) takes
// an exponential and a reciprocal, of a quarter of the rate, beside the softmax's own (us a tile of 256 rows, of 128 /
// 64 channels: 2.35 / 1.77 -> 2.25 / 1.70; uncapped 1.90 / 1.20).  That form is off by 2^-22, which up to caps of
// 256 is less than the rounding of the softmax weights; beyond, |y| up to 1/4 go by the series beside it too.  (So
// the scores of the rows beside it may move a capped row's by 2^-22 of the cap; nothing else of a row depends on
// another.)
// The factor is folded into the exponent; with BIAS value and entry are joined first.
template <bool CAP, bool BIAS>
struct ScoreMap {
  float factor;         // scale * log2(e); cap * log2(e)
  float c1, c3, c5, c7; // CAP: the series in s
  float k;              // 2 log2(e) scale / cap
  float small, exact;   // the |s| up to which all go by the series; the |y| up to which (for large caps) each does

  __device__ __forceinline__ void init(const MaskedArgs& a) {
    factor = (CAP ? a.cap : a.scale) * kLog2e;
    c1 = CAP ? a.scale / a.cap : 0.f;
    const float sq = c1 * c1;
    c3 = c1 * sq * (-1.f / 3.f);
    c5 = c1 * sq * sq * (2.f / 15.f);
    c7 = c1 * sq * sq * sq * (-17.f / 315.f);
    k = fminf(2.f * kLog2e * c1, FLT_MAX);
    small = CAP && c1 > 1e-5f && c1 < 1e4f ? 0.25f / c1 : -1.f;      // (where c7 neither overflows nor vanishes)
    exact = a.cap > kExactCap ? 0.25f : -1.f;
  }
  __device__ __forceinline__ float form(float s) const {
    return fmaf(2.f, __builtin_amdgcn_rcpf(-1.f - fast_exp2(s * k)), 1.f);
  }
  // What is left of the map after begin(): the series, or nothing.
  struct Rest {
    float c1, c3, c5, c7;
    __device__ __forceinline__ float operator()(float s) const {
      const float z = s * s;
      return s * fmaf(z, fmaf(z, fmaf(z, c7, c5), c3), c1);
    }
  };
  // The first half of the map, of N x 16 scores: where the series holds for all of the wave, nothing.
  template <int N>
  __device__ __forceinline__ Rest begin(f32x16* const (&s)[N]) const {
    Rest rest{c1, c3, c5, c7};
    if constexpr (CAP) {
      float top = fabsf((*s[0])[0]);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf((*s[n])[r]));
      if (__builtin_amdgcn_ballot_w64(!(top <= small)) != 0) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float v = (*s[n])[r], y = v * c1, z = y * y, far = form(v);
            const float near = y * fmaf(z, fmaf(z, fmaf(z, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
            (*s[n])[r] = fabsf(y) <= exact ? near : far;
          }
        rest = Rest{1.f, 0.f, 0.f, 0.f};
      }
    }
    return rest;
  }
  // N x 16 scores
  template <int N>
  __device__ __forceinline__ void map(f32x16* const (&s)[N]) const {
    if constexpr (CAP) {
      const Rest rest = begin<N>(s);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) (*s[n])[r] = rest((*s[n])[r]);
    }
  }
  // with BIAS: the mapped value and the table entry of its distance
  __device__ __forceinline__ float add(float s, float entry) const { return fmaf(s, factor, entry); }
  // the weight of a score against the reference point m
  __device__ __forceinline__ float weight(float s, float m) const {
    if constexpr (BIAS) return fast_exp2(s - m);
    else return fast_exp2(fmaf(s, factor, -m));
  }
  // a max of scores in the units of m
  __device__ __forceinline__ float top(float s) const { return BIAS ? s : s * factor; }
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
#pragma unroll 2        // (few registers: the kernels hold their accumulators here)
  for (int i = 0; i < KEYS * HD / 512; ++i) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(Vt + i * 512 + lane * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[j] & M));
  }
  return __builtin_amdgcn_ballot_w64(top[0] == Elem<T>::kExpBits || top[1] == Elem<T>::kExpBits) != 0;
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

// O^T += V^T P^T of a tile of 16 N keys from key kt on that holds NaNs or infinities, some of them perhaps of
// keys that a row does not see.  Their products are left out (v as 0); then each row gets the infinities of the
// keys that it sees: their number is the product of v's bad places (+inf 1, -inf 128, NaN both) with the keys
// that the row sees (1 or 0), which is exact.
template <typename T, int HD, int N>
__device__ __forceinline__ void exact_pv(const MaskedOperands<T, HD>& op, f32x16 (&o)[HD / 32],
                                         const typename Elem<T>::x8 (&pb)[N], const bf16* Vt, int kt, const MaskedRow& m,
                                         int hh) {
  typedef typename Elem<T>::x8 X8;
  typedef unsigned short U8 __attribute__((ext_vector_type(8)));
  constexpr unsigned short M = Elem<T>::kExpBits;
#pragma unroll
  for (int md = 0; md < HD / 32; ++md) {
    f32x16 count = {};
#pragma unroll
    for (int ksp = 0; ksp < N; ++ksp) {
      const U8 v = __builtin_bit_cast(U8, op.v_frag(Vt, ksp, md));
      U8 good;
      X8 bad, sees;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool is_bad = (v[e] & M) == M, nan = (v[e] & 0x7fff) != M;
        good[e] = is_bad ? 0 : v[e];
        bad[e] = (T)(!is_bad ? 0.f : nan ? 129.f : v[e] & 0x8000 ? 128.f : 1.f);
        const int key = kt + 16 * ksp + 4 * hh + (e & 3) + 8 * (e >> 2);
        sees[e] = (T)(key >= m.lo && key < m.hi ? 1.f : 0.f);
      }
      o[md] = Elem<T>::mfma(__builtin_bit_cast(X8, good), pb[ksp], o[md]);
      count = Elem<T>::mfma(bad, sees, count);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float down = floorf(count[r] * (1.f / 128.f));
      o[md][r] += count[r] - 128.f * down > 0.f ? INFINITY : 0.f;
      o[md][r] += down > 0.f ? -INFINITY : 0.f;
    }
  }
}

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
// 32 rows on tiles of 32 keys, by one wave alone
// ---------------------------------------------------------------------------

constexpr int kWaveKeys = 32;

// The rows of a wave: this lane's query and head, its interval, and what any and every row of the wave sees.
struct WaveRows {
  int i, g;
  MaskedRow m;
  int first, end, all_lo, all_hi;
  // rows row0 .. row0 + 31 of a unit; those past the last one repeat it (they are not stored)
  __device__ __forceinline__ WaveRows(const MaskedArgs& a, int b, int row0, int rows, int lane) {
    const int r = min(row0 + (lane & 31), rows - 1);
    i = a.by_pack(r);
    g = r - i * a.pack;
    m = masked_row(a, b, i);
    const bool some = m.lo < m.hi;
    first = rows_min(some ? m.lo : 0x7fffffff);
    end = rows_max(m.hi);
    all_lo = rows_max(m.lo);
    all_hi = rows_min(m.hi);
  }
};

// The tiles t, t + stride, ... < tb through SLOTS slots of k and v tiles at `tiles`, all of it this wave's
// own: copies of the next SLOTS - 1 tiles in flight, no barrier.  `window`: kept bias entries (`floats`).
// Leaves O unnormalised, its reference point and this lane's sum.
template <typename T, int HD, bool CAP, bool BIAS, int SLOTS>
__device__ __forceinline__ void attend_wave(const MaskedArgs& a, const MaskedUnit& u, const WaveRows& w, int t, int tb,
                                            int stride, bf16* tiles, float* window, int floats, int lane,
                                            f32x16 (&o)[HD / 32], float& m_run, float& l_run) {
  typedef typename Elem<T>::x8 X8;
  constexpr int kTile = kWaveKeys * HD;       // elements
  const int hh = lane >> 5;
  MaskedCopy<HD, kWaveKeys, 1, false> kc;
  MaskedCopy<HD, kWaveKeys, 1, true> vc;
  kc.init(static_cast<const T*>(a.k.ptr) + u.b * a.k.sb + u.hk * a.k.sh, a.k.st, 0, lane);
  vc.init(static_cast<const T*>(a.v.ptr) + u.b * a.v.sb + u.hk * a.v.sh, a.v.st, 0, lane);
  auto issue = [&](int t, int slot) {
    kc.issue(t, a.Lk, tiles + slot * (2 * kTile), 0, lane);
    vc.issue(t, a.Lk, tiles + slot * (2 * kTile) + kTile, 0, lane);
  };
  if (t < tb) issue(t, 0);

  MaskedOperands<T, HD> op;
  op.init(static_cast<const T*>(a.q.ptr) + u.b * a.q.sb + (int64_t)w.i * a.q.st + (u.h0 + w.g) * a.q.sh, lane);
  ScoreMap<CAP, BIAS> map;
  map.init(a);
  BiasWindow win;
  int p_max = 0, p_min = 0;
  if constexpr (BIAS) {
    win.init(floats, a.pack);
    p_max = rows_max(w.m.p);
    p_min = rows_min(w.m.p);
  }
#pragma unroll
  for (int md = 0; md < HD / 32; ++md) o[md] = f32x16{};
  m_run = -FLT_MAX;
  l_run = 0.f;

  // As in the block kernel, the query rows have to be there for the compiler too.  (A wait for all: the second tile goes
  // out behind it, 256 keys by one workgroup 6.6 -> 6.2 us.)
  wait_vm_all();
#pragma unroll
  for (int n = 1; n < SLOTS; ++n)
    if (t + n * stride < tb) issue(t + n * stride, n);
  for (int slot = 0; t < tb; t += stride, slot = SLOTS == 1 ? 0 : slot ^ 1) {
    const int kt = t * kWaveKeys;
    const bf16 *Kt = tiles + slot * (2 * kTile), *Vt = Kt + kTile;
    if constexpr (BIAS) {
      if (!win.holds(kt - p_max, kt + kWaveKeys - 1 - p_min)) {
        win.load(a, u.h0, kt - p_max, (int64_t)(tb - t) * kWaveKeys + (p_max - p_min), window, lane, 64);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
    // this tile has landed; the next one's copies stay in flight
    if (SLOTS > 1 && t + stride < tb)
      asm volatile("s_waitcnt vmcnt(%0)" :: "i"(2 * decltype(kc)::kPer) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) s = Elem<T>::mfma(op.k_frag(Kt, ks, 0), op.qf[ks], s);
    map.template map<1>({&s});
    if constexpr (BIAS) {
      const float* e0 = window + w.g * win.per + (kt + 4 * hh - w.m.p - win.w0);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = map.add(s[e], e0[8 * (e >> 2) + (e & 3)]);
    }
    const bool masked = kt < w.all_lo || kt + kWaveKeys > w.all_hi;
    if (masked) mask_scores(s, kt, hh, w.m);

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
      const typename Elem<T>::x2 p = {(T)map.weight(s[e], m_run), (T)map.weight(s[e + 1], m_run)};
      pb[e >> 3][e & 7] = p[0];
      pb[e >> 3][(e & 7) + 1] = p[1];
      l_run = Elem<T>::add2(p, l_run);      // the sum of the rounded weights that the products use
    }
    if (masked && tile_not_finite<T, HD, kWaveKeys>(Vt, lane)) {
      exact_pv<T, HD>(op, o, pb, Vt, kt, w.m, hh);
    } else {
#pragma unroll
      for (int ksp = 0; ksp < 2; ++ksp)
#pragma unroll
        for (int md = 0; md < HD / 32; ++md) o[md] = Elem<T>::mfma(op.v_frag(Vt, ksp, md), pb[ksp], o[md]);
    }
    // every read of this slot has returned before it is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + SLOTS * stride < tb) issue(t + SLOTS * stride, slot);
  }
}

// ---------------------------------------------------------------------------
// few rows: 32 rows a workgroup, its four waves on every fourth tile
// ---------------------------------------------------------------------------
//
// Bound by the bytes of k and v: one token each of 16 samples over 1080 to 8192 keys, 32 heads over 8 of 128
// channels, takes 85 us with the merge (5.0 TB/s; a large copy reaches 5.1); over 1000 keys of one sample 8.6 us in a
// replayed graph, most of it the two launches.  A wave keeps two tiles of its own in flight and meets no barrier
// before the end.

constexpr int kStepWaves = 4;
constexpr int kStepWindow = 1200;       // bias entries of a wave

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(kStepWaves * 64, 1) void masked_step_kernel(const MaskedArgs a) {
  typedef typename Elem<T>::x8 X8;
  constexpr int kTiles = 4 * kWaveKeys * HD;         // a wave's two slots of k and v, elements
  __shared__ __attribute__((aligned(1024))) bf16 tiles[kStepWaves][kTiles];
  __shared__ float window[kStepWaves][BIAS ? kStepWindow : 1];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const int rows = a.Lq * a.pack;
  const int block = a.by_splits(blockIdx.x), part = blockIdx.x - block * a.splits;
  const int unit = a.by_blocks(block), row0 = (block - unit * a.blocks) * 32;
  const MaskedUnit blk(a, unit);
  const WaveRows w(a, blk.b, row0, rows, lane);
  const int t0 = w.first / kWaveKeys;
  const TileRange range(t0, w.first < w.end ? (w.end - 1) / kWaveKeys + 1 - t0 : 0, part, a.splits);

  f32x16 o[HD / 32];
  float m_run, l_run;
  attend_wave<T, HD, CAP, BIAS, 2>(a, blk, w, range.first + wave, range.end, kStepWaves, tiles[wave], window[wave],
                                   kStepWindow, lane, o, m_run, l_run);
  l_run = pair_sum(l_run);

  // The four waves' results through LDS: O [32][HD + 4], then each row's weights.
  constexpr int kRow = HD + 4;
  static_assert(kStepWaves * 32 * (kRow + 2) * 4 <= (int)sizeof(tiles), "the tiles hold the waves' results");
  __syncthreads();
  float* const all = reinterpret_cast<float*>(&tiles[0][0]);
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
  const int held = min(rows - row0, 32);             // rows of this block
  for (int x = threadIdx.x; x < held * (HD / 8); x += kStepWaves * 64) {
    const int row = x / (HD / 8), c = x - row * (HD / 8);
    float top = stat[row], l = 0.f;
#pragma unroll
    for (int n = 1; n < kStepWaves; ++n) top = fmaxf(top, stat[n * 32 + row]);
    float v[8] = {};
#pragma unroll
    for (int n = 0; n < kStepWaves; ++n) {
      const float f = fast_exp2(stat[n * 32 + row] - top);
      l += f * stat[(kStepWaves + n) * 32 + row];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(f, all[n * (32 * kRow) + row * kRow + 8 * c + e], v[e]);
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
      const int rr = row0 + row, qi = a.by_pack(rr);
      X8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (T)(v[e] * inv);
      *reinterpret_cast<X8*>(static_cast<T*>(a.o) + blk.b * a.o_sb + (int64_t)qi * a.o_st +
                             (blk.h0 + rr - qi * a.pack) * a.o_sh + 8 * c) = y;
    }
  }
}

// ---------------------------------------------------------------------------
// many rows: 32 a wave, on tiles of 64 keys that a workgroup's waves share
// ---------------------------------------------------------------------------
//
// KG = 1: all NW waves have rows of their own, eight (256 rows, a workgroup a CU) for 128 channels, four for 64, of
// which two workgroups fit a CU, so that one's start and end overlap the other's tiles.  (us, 64 channels, eight /
// four: 512 text tokens with bias 19.4 / 15.4, 2049 tokens with prefixes 38.2 / 32.1, 24 heads of 4096 tokens
// 140 / 127, 2 x 7854 causal 441 / 452.  With 128 channels four have LDS for rings of two tiles: 24 heads of 4096
// tokens 216 / 202, 2 x 7854 causal 722 / 745.)
// KG = 2: eight waves, four of rows (128), the other four the same rows on every second tile; a block then takes
// half as many steps, which is what a launch with few, or unequally long, blocks ends sooner by, for twice the
// tile copies (us, KG 1 / 2: 2 x 1024 tokens causal, 16 over 4 heads of 128 channels 30.0 / 20.6, 24 heads of 1000
// tokens 29.5 / 21.4, of 64 channels 17.7 / 15.8; 2 x 7854 causal 722 / 787).

constexpr int kBlockKeys = kTileKeys;
template <int HD> constexpr int kBlockWaves = HD == 128 ? 8 : 4;
constexpr int kWaveWindow = 1016;       // bias entries of a workgroup, for each of its waves

// The order of the workgroups: units (and their parts) in groups of kUnitGroup, in a group the first blocks of all its
// units first.  Those are the rows that see the most keys (the last ones, which under a causal mask do, or the
// longest document's), so that the short blocks fill the end of the launch.  Workgroup i runs on XCD i % 8: the blocks
// of a unit share one L2 where the units of a group are a multiple of 8, and where they are fewer each unit's long and
// short blocks spread evenly over the XCDs.
struct BlockOrder {
  int up, at;
  __device__ __forceinline__ BlockOrder(const MaskedArgs& a, int id) {
    const int turned = (id - a.turn_first) >> 3;
    if (turned >= 0 && turned < a.turn_eights) id = a.turn_first + (a.turn_eights - 1 - turned) * 8 + (id & 7);
    const int group = a.by_blocks(id / kUnitGroup), in = id - group * (kUnitGroup * a.blocks);
    // (the last group may be smaller)
    const bool whole = (group + 1) * kUnitGroup <= a.ups;
    const int size = whole ? kUnitGroup : a.ups - group * kUnitGroup;
    at = whole ? in / kUnitGroup : a.by_last_ups(in);
    up = group * kUnitGroup + (in - at * size);
  }
};

// Inclusive scans over the wave's 64 lanes, `none` where there is nothing to the left.
template <typename F>
__device__ __forceinline__ int wave_scan(int v, int none, F op) {
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xf, 0xf, false));    // 1, 2, 4, 8 lanes on, in 16
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xa, 0xf, false));    // lane 15's, 47's to the next 16
  v = op(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xc, 0xf, false));    // lane 31's to the upper 32
  return v;
}

// The rows of block `at` of a sample's unit: of blocks of BM rows, the last ones first; with documents (not
// split) of blocks that begin where a document of 2 BM rows or more begins or ends.  A block over the border of
// two such reads the keys of both, half of its waves idle in each.  (7854 tokens in documents of 374, 1080, 2244
// and 4156, 24 heads of 128 channels: 366 -> 278 us.)  Runs of smaller documents stay together.  The longest
// run's blocks come first.  Rows before the first document are a run too, and a row is in one block whatever
// the starts hold.  Blocks past the last one have no rows.
struct RowBlock {
  int first, end;
  __device__ __forceinline__ RowBlock(const MaskedArgs& a, int b, int at, int BM, int lane) {
    const int rows = a.Lq * a.pack;
    if (!a.by_docs) {
      first = (a.blocks - 1 - at) * BM;
      end = min(first + BM, rows);
      return;
    }
    const int start = first_position(a, b);
    const int32_t* d = a.doc_starts + (int64_t)b * a.docs;
    int begun = 0;            // rows of the runs before these 64
    first = end = rows;
    for (int j0 = 0; j0 <= a.docs; j0 += 64) {
      // this lane's document (0: none yet, j: the j-th) ends in front of row `to`
      const int j = j0 + lane;
      int to = rows;
      if (j < a.docs) {
        const int64_t q = (int64_t)d[j] - start;
        to = (int)(min(max(q, (int64_t)0), (int64_t)a.Lq) * a.pack);
      }
      to = max(begun, wave_scan(to, 0, [](int x, int y) { return max(x, y); }));
      int from = __shfl_up(to, 1);
      if (lane == 0) from = begun;
      const bool large = to - from >= 2 * BM;
      const bool large_before = __shfl_up((int)large, 1) != 0;
      const uint64_t heads = __builtin_amdgcn_ballot_w64(lane == 0 || large || large_before);
      const bool head = heads >> lane & 1;
      const uint64_t later = lane == 63 ? 0 : heads >> (lane + 1);
      const int run_last = later != 0 ? lane + __builtin_ctzll(later) : 63;       // the run's last lane
      const int run_end = __shfl(to, run_last), size = run_end - from;
      const int count = head ? (size + BM - 1) / BM : 0;
      const int total = __builtin_amdgcn_readlane(wave_scan(count, 0, [](int x, int y) { return x + y; }), 63);
      if (at < total) {
        int before = 0;       // blocks of the longer runs
        for (uint64_t m = heads; m != 0; m &= m - 1) {
          const int other = __builtin_ctzll(m), s = __builtin_amdgcn_readlane(size, other);
          if (s > size || (s == size && other < lane)) before += __builtin_amdgcn_readlane(count, other);
        }
        const int mine = __builtin_ctzll(__builtin_amdgcn_ballot_w64(head && before <= at && at < before + count));
        const int k = at - __builtin_amdgcn_readlane(before, mine), n = __builtin_amdgcn_readlane(count, mine);
        first = __builtin_amdgcn_readlane(from, mine) + (n - 1 - k) * BM;
        end = min(first + BM, __builtin_amdgcn_readlane(run_end, mine));
        return;
      }
      at -= total;
      begun = __builtin_amdgcn_readlane(to, 63);
    }
  }
};

// The arithmetic of a wave's 32 rows on a tile of 64 keys (scores c0: keys 0 .. 31, c1: 32 .. 63).
template <typename T, int HD, bool CAP, bool BIAS>
struct BlockCore {
  typedef typename Elem<T>::x8 X8;
  typedef typename Elem<T>::x2 X2;
  // A lane's sum of a tile's weights that makes the wave take a new reference point: with less, every
  // weight fits the type, and a reference point below the running max cancels in O / l.
  static constexpr float kBound = sizeof(X8) == 16 && Elem<T>::kExpBits == 0x7c00 ? 32768.f : kSumBound;
  static constexpr int kSteps = HD / 16, kEach = 16 / kSteps;    // MFMA steps, scores of a half in each

  MaskedOperands<T, HD> op;
  ScoreMap<CAP, BIAS> map;
  f32x16 o[HD / 32];
  float m_run, l_run;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int md = 0; md < HD / 32; ++md) o[md] = f32x16{};
    m_run = -FLT_MAX;
    l_run = 0.f;
  }

  __device__ __forceinline__ void qk(const bf16* Kt, f32x16& s0, f32x16& s1) const {
    s0 = f32x16{};
    s1 = f32x16{};
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      s0 = Elem<T>::mfma(op.k_frag(Kt, ks, 0), op.qf[ks], s0);
      s1 = Elem<T>::mfma(op.k_frag(Kt, ks, 32), op.qf[ks], s1);
    }
  }

  __device__ __forceinline__ void weigh(const f32x16& c, int r, float m, X8 pb[2], float& acc) const {
    const X2 w = {(T)map.weight(c[r], m), (T)map.weight(c[r + 1], m)};
    pb[r >> 3][r & 7] = w[0];
    pb[r >> 3][(r & 7) + 1] = w[1];
    acc = Elem<T>::add2(w, acc);
  }

  // The weights of a tile and this lane's sum of them (of the rounded values that the products use), eight
  // exponentials in flight at most.
  __device__ __forceinline__ float exp_tile(const f32x16& c0, const f32x16& c1, X8 pb[4]) const {
    float acc[2] = {0.f, 0.f}, m = m_run;
    // (a value of its own for the compiler, which otherwise moves this and qk_exp's exponents out of the branch
    // between them, in front of the MFMAs that they are to run beside)
    asm volatile("" : "+v"(m));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        weigh(h == 0 ? c0 : c1, r, m, pb + 2 * h, acc[h]);
        if ((r & 7) == 6) __builtin_amdgcn_sched_barrier(0);
      }
    return acc[0] + acc[1];
  }

  // The same with the MFMAs of the next tile's scores in between, k fragments read one step ahead.  MAP: what is left
  // of the scores' map too (`bias`: this lane's entry of the tile's first key).
  template <bool MAP>
  __device__ __forceinline__ float qk_exp(const bf16* Kt, f32x16& n0, f32x16& n1, f32x16& c0, f32x16& c1, X8 pb[4],
                                          const typename ScoreMap<CAP, BIAS>::Rest& rest, const float* bias) const {
    float acc0 = 0.f, acc1 = 0.f;
    X8 a0 = op.k_frag(Kt, 0, 0), a1 = op.k_frag(Kt, 0, 32);
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) {
      X8 b0, b1;
      if (ks < kSteps - 1) {
        b0 = op.k_frag(Kt, ks + 1, 0);
        b1 = op.k_frag(Kt, ks + 1, 32);
      }
      n0 = Elem<T>::mfma(a0, op.qf[ks], ks == 0 ? f32x16{} : n0);
      n1 = Elem<T>::mfma(a1, op.qf[ks], ks == 0 ? f32x16{} : n1);
      if constexpr (MAP && (CAP || BIAS)) {
#pragma unroll
        for (int r = kEach * ks; r < kEach * (ks + 1); ++r) {
          if (CAP) {
            c0[r] = rest(c0[r]);
            c1[r] = rest(c1[r]);
          }
          if constexpr (BIAS) {
            c0[r] = map.add(c0[r], bias[8 * (r >> 2) + (r & 3)]);
            c1[r] = map.add(c1[r], bias[32 + 8 * (r >> 2) + (r & 3)]);
          }
        }
      }
#pragma unroll
      for (int r = kEach * ks; r < kEach * (ks + 1); r += 2) {
        weigh(c0, r, m_run, pb, acc0);
        weigh(c1, r, m_run, pb + 2, acc1);
      }
      if (ks < kSteps - 1) {
        a0 = b0;
        a1 = b1;
      }
    }
    return acc0 + acc1;
  }

  __device__ __forceinline__ float tile_top(const f32x16& c0, const f32x16& c1) const {
    return map.top(pair_max(fmaxf(max16(c0), max16(c1))));
  }

  // Takes a tile's sum of weights rs; a row whose sum passes the bound (or is inf or NaN) goes over to the tile's
  // exact max, rescales and weighs again, with the wave's other rows as they were, so that no row's reference
  // point depends on the rows beside it.
  __device__ __forceinline__ void finish(const f32x16& c0, const f32x16& c1, float rs, X8 pb[4]) {
    const bool over = !(rs <= kBound);
    if (__builtin_amdgcn_ballot_w64(over) != 0) {
      const float top = tile_top(c0, c1);
      const float m_new = pair_max(over ? 1.f : 0.f) > 0.f ? fmaxf(m_run, top) : m_run;
      const float alpha = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int md = 0; md < HD / 32; ++md) o[md] *= alpha;
      rs = exp_tile(c0, c1, pb);
    }
    l_run += rs;
  }

  // O^T += V^T P^T, v fragments read one MFMA ahead
  __device__ __forceinline__ void pv(const X8 pb[4], const bf16* Vt) {
    constexpr int MD = HD / 32;
    X8 cur = op.v_frag(Vt, 0, 0);
#pragma unroll
    for (int i = 0; i < 4 * MD; ++i) {
      X8 nxt;
      if (i < 4 * MD - 1) nxt = op.v_frag(Vt, (i + 1) / MD, (i + 1) % MD);
      o[i % MD] = Elem<T>::mfma(cur, pb[i / MD], o[i % MD]);
      if (i < 4 * MD - 1) cur = nxt;
    }
  }
};

template <typename T, int HD, bool CAP, bool BIAS, int NW, int KG>
__global__ __launch_bounds__(NW * 64, 2) void masked_block_kernel(const MaskedArgs a) {
  typedef typename Elem<T>::x8 X8;
  typedef typename Elem<T>::x4 X4;
  constexpr int kRowWaves = NW / KG, BM = kRowWaves * 32, BK = kBlockKeys, kTile = BK * HD;
  // Rings of four k and v tiles and a barrier every second tile.  With KG = 1, as in the unmasked kernel, an
  // even step issues the copies of the next pair of tiles and the odd one waits for them; with KG = 2 a step
  // is a pair of tiles.
  __shared__ __attribute__((aligned(1024))) bf16 k_lds[4][kTile];
  __shared__ __attribute__((aligned(1024))) bf16 v_lds[4][kTile];
  __shared__ float window[BIAS ? NW * kWaveWindow : 1];
  __shared__ int ends[2][NW];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, hh = lane >> 5;
  const BlockOrder order(a, blockIdx.x);
  const int unit = a.by_splits(order.up), part = order.up - unit * a.splits;
  const MaskedUnit blk(a, unit);
  const RowBlock block_rows(a, blk.b, order.at, BM, lane);
  const int row0 = MaskedUnit::uniform(block_rows.first), rows = MaskedUnit::uniform(block_rows.end);
  if (row0 >= rows) return;
  const int kg = wave / kRowWaves, wrow0 = row0 + (wave - kg * kRowWaves) * 32;
  const bool live = wrow0 < rows;      // (a wave without rows copies its share and meets the barriers)
  WaveRows w(a, blk.b, wrow0, rows, lane);
  if (!live) {
    w.first = 0x7fffffff;
    w.end = 0;
  }
  // What the first tile needs goes out before it is known which tiles these rows see: without documents, and
  // not split, they begin with tile 0 (if they see any).
  MaskedCopy<HD, BK, NW, false> kc;
  MaskedCopy<HD, BK, NW, true> vc;
  kc.init(static_cast<const T*>(a.k.ptr) + blk.b * a.k.sb + blk.hk * a.k.sh, a.k.st, wave, lane);
  vc.init(static_cast<const T*>(a.v.ptr) + blk.b * a.v.sb + blk.hk * a.v.sh, a.v.st, wave, lane);
  const bool early = a.doc_starts == nullptr && a.splits == 1 && a.Lk > 0;
  if (early) {
    kc.issue(0, a.Lk, k_lds[0], wave, lane);
    vc.issue(0, a.Lk, v_lds[0], wave, lane);
  }
  BlockCore<T, HD, CAP, BIAS> c;
  c.op.init(static_cast<const T*>(a.q.ptr) + blk.b * a.q.sb + (int64_t)w.i * a.q.st + (blk.h0 + w.g) * a.q.sh, lane);
  // the tiles that any row of the workgroup sees keys of, this part of them
  if (lane == 0) {
    ends[0][wave] = w.first;
    ends[1][wave] = w.end;
  }
  __syncthreads();
  int first = ends[0][0], end = ends[1][0];
#pragma unroll
  for (int n = 1; n < NW; ++n) {
    first = min(first, ends[0][n]);
    end = max(end, ends[1][n]);
  }
  const TileRange range(first / BK, first < end ? (end - 1) / BK + 1 - first / BK : 0, part, a.splits);
  const int nt = range.end - range.first;

  bool bad = false;       // a tile that needed a mask held a NaN or an infinity in v
  c.reset();
  c.map.init(a);
  if (nt > 0) {
    auto copy_k = [&](int u) {
      if (u < nt) kc.issue(range.first + u, a.Lk, k_lds[u & 3], wave, lane);
    };
    auto copy_v = [&](int u) {
      if (u < nt) vc.issue(range.first + u, a.Lk, v_lds[u & 3], wave, lane);
    };
    if (!early) {
      copy_k(0);
      copy_v(0);
    }
    copy_k(1);
    copy_v(1);
    copy_k(2);
    if (KG == 2) copy_k(3);

    BiasWindow win;
    int p_first = 0, p_last = 0;       // positions of the workgroup's rows
    if constexpr (BIAS) {
      win.init(NW * kWaveWindow, a.pack);
      const int at = MaskedUnit::uniform(w.m.p - w.i);
      p_first = at + a.by_pack(row0);
      p_last = at + a.by_pack(rows - 1);
    }
    auto load_window = [&](int u0) {
      win.load(a, blk.h0, (range.first + u0) * BK - p_last, (int64_t)(nt - u0 + KG - 1) * BK + (p_last - p_first), window,
               threadIdx.x, NW * 64);
    };
    if constexpr (BIAS) load_window(0);       // (while the tiles are on their way)
    // whether the wave's rows see any key of tile u
    auto seen = [&](int u) {
      const int kt = (range.first + u) * BK;
      return u < nt && kt < w.end && kt + BK > w.first;
    };
    bool fresh = true;
    const int base = range.first * BK, last = range.end - 1;
    // One step: tiles u0 (.. u0 + KG - 1), this wave's its u.  LEAN: every row sees all of tile u, some see
    // tile u + KG, and the tiles to be copied are whole, so that no such question is asked (past the last one
    // it is copied again).
    auto step = [&](auto lean, int u0, f32x16& c0, f32x16& c1, f32x16& n0, f32x16& n1) {
      constexpr bool LEAN = decltype(lean)::value;
      const int u = u0 + kg, kt = (range.first + u) * BK;
      if constexpr (BIAS && !LEAN) {
        const int k0 = (range.first + u0) * BK;
        if (!win.holds(k0 - p_last, k0 + KG * BK - 1 - p_first)) {
          __syncthreads();
          load_window(u0);
          __syncthreads();
        }
      }
      const bool here = LEAN || seen(u), next = LEAN || seen(u + KG);
      const bool masked = !LEAN && here && (kt < w.all_lo || kt + BK > w.all_hi);
      const bf16 *Kn = k_lds[(u + KG) & 3], *Vt = v_lds[u & 3];
      X8 pb[4];
      if (here) {
        const float* bias = nullptr;
        if constexpr (BIAS) bias = window + w.g * win.per + (kt + 4 * hh - w.m.p - win.w0);
        float rs;
        if constexpr (LEAN) {
          const auto rest = c.map.template begin<2>({&c0, &c1});
          rs = c.template qk_exp<true>(Kn, n0, n1, c0, c1, pb, rest, bias);
        } else {
          c.map.template map<2>({&c0, &c1});
          if constexpr (BIAS) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              c0[e] = c.map.add(c0[e], bias[8 * (e >> 2) + (e & 3)]);
              c1[e] = c.map.add(c1[e], bias[32 + 8 * (e >> 2) + (e & 3)]);
            }
          }
          if (masked) {
            mask_scores(c0, kt, hh, w.m);
            mask_scores(c1, kt + 32, hh, w.m);
          }
          if (fresh) {
            c.m_run = fmaxf(-FLT_MAX, c.tile_top(c0, c1));
            fresh = false;
          }
          rs = next ? c.template qk_exp<false>(Kn, n0, n1, c0, c1, pb, {}, nullptr) : c.exp_tile(c0, c1, pb);
        }
        c.finish(c0, c1, rs, pb);
      } else if (next) {
        c.qk(Kn, n0, n1);
      }
      if (KG == 2 || (u0 & 1) == 0) {
        if constexpr (LEAN) {
          kc.issue_full(min(range.first + u0 + 2 + KG, last), k_lds[(u0 + 2 + KG) & 3], wave);
          kc.issue_full(min(range.first + u0 + 3 + KG, last), k_lds[(u0 + 3 + KG) & 3], wave);
          vc.issue_full(min(range.first + u0 + 2, last), v_lds[(u0 + 2) & 3], wave);
          vc.issue_full(min(range.first + u0 + 3, last), v_lds[(u0 + 3) & 3], wave);
        } else {
          copy_k(u0 + 2 + KG);
          copy_k(u0 + 3 + KG);
          copy_v(u0 + 2);
          copy_v(u0 + 3);
        }
      }
      if (here) {
        if (masked) bad = bad || tile_not_finite<T, HD, BK>(Vt, lane);
        c.pv(pb, Vt);
      }
      if (KG == 2 || (u0 & 1)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
      }
    };
    // Two steps from u0 on are lean for this wave if lean_lo <= u0 < lean_hi (and it has begun).
    const int seen_end = min(nt, (w.end - 1 - base) / BK + 1);
    const int lean_lo = (w.all_lo - base + BK - 1) / BK - kg;
    const int lean_hi = min(min((w.all_hi - base) / BK - KG, seen_end - 2 * KG) - kg,
                            range.end * BK <= a.Lk ? nt : nt - 1 - (KG == 1 ? 4 : 7));

    // (the compiler's own wait: it must know here that the query rows are there, or it waits for them, and so for
    // every copy in flight, at their first use in each step)
    wait_vm_all();
    __syncthreads();
    f32x16 sa0, sa1, sb0, sb1;
    if (seen(kg)) {
      c.qk(k_lds[kg], sa0, sa1);
      // The first reference point, where every row sees the whole tile.  (With a bias it needs the mapped scores:
      // one that lies above all of a row's would leave it no weights.  The tanh grows with the score.)
      if (!BIAS && lean_lo <= 0 && base + (kg + 1) * BK <= w.all_hi) {
        const float top = pair_max(fmaxf(max16(sa0), max16(sa1)));
        c.m_run = c.map.top(CAP ? c.map.form(top) : top);
        fresh = !(c.m_run >= -FLT_MAX && c.m_run <= FLT_MAX);
        if (__builtin_amdgcn_ballot_w64(fresh) != 0) c.m_run = -FLT_MAX;
        fresh = __builtin_amdgcn_ballot_w64(fresh) != 0;
      }
    }
    __syncthreads();      // every wave is done with the first tiles of k before they are overwritten
    for (int u = 0; u < nt; u += 2 * KG) {
      while (u >= lean_lo && u < lean_hi && !fresh &&
             (!BIAS || win.holds(base + u * BK - p_last, base + (u + 2 * KG) * BK - 1 - p_first))) {
        step(std::true_type{}, u, sa0, sa1, sb0, sb1);
        step(std::true_type{}, u + KG, sb0, sb1, sa0, sa1);
        u += 2 * KG;
      }
      if (u < nt) step(std::false_type{}, u, sa0, sa1, sb0, sb1);
      if (u + KG < nt) step(std::false_type{}, u + KG, sb0, sb1, sa0, sa1);
    }
    if (KG == 2 && lane == 0) ends[0][wave] = bad;
    __syncthreads();      // ... and with the last tiles before the output is staged over them
    if (KG == 2) bad = ends[0][wave % kRowWaves] | ends[0][wave % kRowWaves + kRowWaves];
  } else {
    wait_vm_all();        // (tile 0 has landed before its place is used otherwise)
    __syncthreads();
  }
  if (KG == 1 && !live) return;
  // This wave's share of the rings, from here on.
  bf16* const share = wave < 4 ? k_lds[wave] : v_lds[wave - 4];
  // Such a value may have reached rows that do not see it: the wave's rows once more, by itself.  (Told apart in
  // the loop above, the second way to form O left it too few registers: 40 were spilled in every tile.)
  if (bad)
    attend_wave<T, HD, CAP, BIAS, 1>(a, blk, w, max(range.first * (BK / kWaveKeys), w.first / kWaveKeys) + kg,
                                     min(range.end * (BK / kWaveKeys), (w.end - 1) / kWaveKeys + 1), KG, share,
                                     window + wave * (kWaveWindow), kWaveWindow, lane, c.o,
                                     c.m_run, c.l_run);
  if constexpr (KG == 2) {
    // The second four waves leave what they have to the first: the rows lie in the same lanes.
    float* const other = reinterpret_cast<float*>(&v_lds[0][0]) + (wave % kRowWaves) * (kTile / 2) + lane * 4;
    float* const stat = reinterpret_cast<float*>(&k_lds[0][0]) + (wave % kRowWaves) * (kTile / 2) + lane;
    __syncthreads();      // (the share of a wave that went over its rows again is read no more)
    if (kg == 1) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
        *reinterpret_cast<f32x4*>(other + n * 256) = f32x4{c.o[n / 4][4 * (n & 3)], c.o[n / 4][4 * (n & 3) + 1],
                                                           c.o[n / 4][4 * (n & 3) + 2], c.o[n / 4][4 * (n & 3) + 3]};
      stat[0] = c.m_run;
      stat[64] = c.l_run;
    }
    __syncthreads();
    if (kg == 1 || !live) return;
    const float m1 = stat[0], top = fmaxf(c.m_run, m1);
    const float f0 = fast_exp2(c.m_run - top), f1 = fast_exp2(m1 - top);
    c.m_run = top;
    c.l_run = f0 * c.l_run + f1 * stat[64];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(other + n * 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) c.o[n / 4][4 * (n & 3) + e] = f0 * c.o[n / 4][4 * (n & 3) + e] + f1 * v[e];
    }
    // (all of it read before the rows are staged over it)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  const float l = pair_sum(c.l_run);
  const int held = min(rows - wrow0, 32);        // rows of this wave
  if (a.splits > 1) {
    const int block = unit * a.blocks + row0 / BM, at = wrow0 - row0 + n32;
    float* p = a.part + ((int64_t)block * a.splits + part) * a.part_floats;
    if (n32 < held) {
#pragma unroll
      for (int md = 0; md < HD / 32; ++md)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(p + at * HD + 32 * md + 8 * q + 4 * hh) =
              f32x4{c.o[md][4 * q], c.o[md][4 * q + 1], c.o[md][4 * q + 2], c.o[md][4 * q + 3]};
      if (hh == 0) {
        p[a.part_rows * HD + at] = c.m_run;
        p[a.part_rows * HD + a.part_rows + at] = l;
      }
    }
    return;
  }
  // The wave's rows leave through 4 KB of LDS, 64 channels at a time, as whole 128-byte segments: chunk c of
  // row r at position c ^ (r % 8).
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* stage = reinterpret_cast<T*>(share);
  T* obase = static_cast<T*>(a.o) + blk.b * a.o_sb + blk.h0 * a.o_sh;
#pragma unroll
  for (int half = 0; half < HD / 64; ++half) {
#pragma unroll
    for (int mm = 0; mm < 2; ++mm)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        X4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (T)(c.o[2 * half + mm][4 * q + e] * inv);
        *reinterpret_cast<X4*>(stage + n32 * 64 + (((4 * mm + q) ^ (n32 & 7)) << 3) + 4 * hh) = w;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = 8 * j + (lane >> 3), ch = lane & 7;
      const X8 v = *reinterpret_cast<const X8*>(stage + row * 64 + ((ch ^ (row & 7)) << 3));
      if (row < held) {
        const int rr = wrow0 + row, qi = a.by_pack(rr);
        __builtin_nontemporal_store(v, reinterpret_cast<X8*>(obase + (int64_t)qi * a.o_st + (rr - qi * a.pack) * a.o_sh +
                                                              64 * half + 8 * ch));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// Rows whose keys were split: O = sum_i w_i O_i / sum_i w_i l_i with w_i = exp2(m_i - max m).  A row has HD / 4
// lanes, four channels each.
template <typename T, int HD>
__global__ __launch_bounds__(256) void masked_merge_kernel(const MaskedArgs a, int out_rows, int block_shift) {
  typedef typename Elem<T>::x4 X4;
  constexpr int kLanes = HD / 4;
  const int lane = threadIdx.x % kLanes, id = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (id >= out_rows) return;
  const int unit = a.by_rows(id);
  const int r = id - unit * (a.Lq * a.pack), rb = r >> block_shift, row = r - (rb << block_shift);
  const float* p0 = a.part + ((int64_t)unit * a.blocks + rb) * a.splits * a.part_floats;
  const float* st = p0 + a.part_rows * HD + row;
  float top = -FLT_MAX;
  for (int s = lane; s < a.splits; s += kLanes) top = fmaxf(top, st[(int64_t)s * a.part_floats]);
#pragma unroll
  for (int x = kLanes / 2; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  f32x4 v = {};
  float l = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float* q = st + (int64_t)s * a.part_floats;
    const f32x4 o = *reinterpret_cast<const f32x4*>(p0 + (int64_t)s * a.part_floats + row * HD + 4 * lane);
    const float f = fast_exp2(q[0] - top);
    l += f * q[a.part_rows];
    v += f * o;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int b = a.by_heads(unit), h0 = (unit - b * a.head_groups) * a.pack, qi = a.by_pack(r);
  X4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(v[e] * inv);
  *reinterpret_cast<X4*>(static_cast<T*>(a.o) + b * a.o_sb + (int64_t)qi * a.o_st +
                         (h0 + r - qi * a.pack) * a.o_sh + 4 * lane) = y;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T, int HD, bool CAP, bool BIAS>
int launch_masked(MaskedArgs a, const MaskedPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.blocks * p.splits));
  if (p.block_rows == 32)
    hipLaunchKernelGGL((masked_step_kernel<T, HD, CAP, BIAS>), grid, dim3(kStepWaves * 64), 0, s, a);
  else if (p.key_groups == 2)
    hipLaunchKernelGGL((masked_block_kernel<T, HD, CAP, BIAS, 8, 2>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((masked_block_kernel<T, HD, CAP, BIAS, kBlockWaves<HD>, 1>), grid, dim3(kBlockWaves<HD> * 64), 0, s, a);
  if (p.splits > 1)
    hipLaunchKernelGGL((masked_merge_kernel<T, HD>), dim3((unsigned)((p.out_rows + 1024 / HD - 1) / (1024 / HD))),
                       dim3(256), 0, s, a,
                       (int)p.out_rows, p.block_rows == 32 ? 5 : p.block_rows == 128 ? 7 : 8);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : set_error(4, "masked_attn launch: %s", hipGetErrorString(e));
}

template <typename T, int HD>
int launch_masked_map(const MaskedArgs& a, const MaskedPlan& p, hipStream_t s) {
  if (a.bias != nullptr)
    return a.cap > 0.f ? launch_masked<T, HD, true, true>(a, p, s) : launch_masked<T, HD, false, true>(a, p, s);
  return a.cap > 0.f ? launch_masked<T, HD, true, false>(a, p, s) : launch_masked<T, HD, false, false>(a, p, s);
}
