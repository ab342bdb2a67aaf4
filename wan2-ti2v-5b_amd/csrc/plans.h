// How launches are laid out: sizes in, tiles, parts and grids out.  Host arithmetic only, so that
// it can be checked over any sizes without a device.
#pragma once

#include <cstddef>
#include <cstdint>

namespace wan {

// ---------------------------------------------------------------------------
// the attention (flash_fwd.hip)
// ---------------------------------------------------------------------------

constexpr int kAttnWaves = 8, kTileKeys = 64;   // waves per workgroup (32 query rows each), keys per tile
// A split part's result: per wave (32 query rows) 16 groups of 64 x 4 fp32 (group 4 md + g
// holds o[md][4g..4g+3] of every lane, so that one store writes 1 KB), then m and l per lane.
constexpr int kPartFloats = 64 * 64 + 128;

// How the 8-wave kernel's last round of workgroups (one per CU) is split.  When the blocks
// leave `rem` of them for a last round and that fills half of the CUs at most, each of
// those is run as n workgroups over a part of the keys and merged.  A tile less costs ~1.4 us
// less; a split costs ~5 us (the merge launch, the parts' own start) and 0.05 us per part
// (132 KB of fp32 written and read).  Self-attention, batch 2, 24 heads, us unsplit / split:
//   1500 tokens (rem 32, n 8)  107.6 / 92.6      2048 (rem 128, n 2)  139.4 / 132.8
//   4114 (rem 48, n 5)         482.1 / 437.3
// More than one round of parts loses: 4862 tokens (rem 144) 576 / 581 at n 3, 7854 (rem 208)
// 1382 / 1411 at n 2 -- while a last round is partly idle the busy CUs clock higher.
// The best n is not monotone in the keys (rem 32: 65 tiles in 6 parts, 64 in 8), and the scratch was
// sized for all keys of the tensor where the launch may be given fewer: n is what `scratch` holds.
struct SplitPlan {
  int from, blocks, splits;   // whole blocks, split blocks, parts of each
  size_t bytes;
};
constexpr int kMaxSplits = 8;
inline SplitPlan split_plan(int B, int H, int Lq, int keys, int cus, size_t scratch) {
  SplitPlan p{0, 0, 1, 0};
  const int64_t blocks = (int64_t)((Lq + kAttnWaves * 32 - 1) / (kAttnWaves * 32)) * B * H;
  const int rem = (int)(blocks % cus), nt = (keys + kTileKeys - 1) / kTileKeys;
  if (rem == 0 || blocks > 0x7fffffff) return p;
  const size_t part = (size_t)rem * kAttnWaves * kPartFloats * sizeof(float);   // bytes, one part of each block
  float best = 0.f;
  for (int n = 2; part * n <= scratch && n <= kMaxSplits && rem * n <= cus && n <= nt; ++n) {
    const float gain = 1.4f * (nt - (nt + n - 1) / n) - 5.f - 0.05f * (rem * n);
    if (gain > best) {
      best = gain;
      p.splits = n;
    }
  }
  if (p.splits < 2) return p;
  p.from = (int)(blocks - rem);
  p.blocks = rem;
  p.bytes = part * p.splits;
  return p;
}

// ---------------------------------------------------------------------------
// the attention under masks (masked_attn.h)
// ---------------------------------------------------------------------------

// Positions of the first query row within +- this, as many keys, and twice as many rows keep every position and
// distance in 32 bits.
constexpr int kMaxPosition = (1 << 29) - 1;
// Caps above this take the form of the tanh that is exact for small arguments too.
constexpr float kExactCap = 256.f;
// Query heads that are rows beside each other, at most: as many as a wave's share of the bias entries (1016)
// holds the distances of 32 keys and 3 positions for.
constexpr int kMaxPack = 28;

// How a call is run: `pack` query heads of one k/v head are rows of a unit, in `blocks` blocks of block_rows
// rows, each as `splits` workgroups over a part of its keys.  A part's result: part_rows rows of D fp32,
// their maxima and their sums.
struct MaskedPlan {
  int pack, block_rows, key_groups, splits, part_rows, part_floats;
  int64_t blocks, out_rows;
  size_t bytes;
  bool by_docs;       // blocks begin and end with the documents of two blocks or more (not split)
  int slots;          // workgroups that a CU holds
};
// Up to this many rows of a unit go by tiles of 32 rows, whose waves split the keys, more by blocks.
constexpr int kStepRows = 32;
constexpr int kMaskedMaxSplits = 64;
// The kernels of blocks: rows, key groups, workgroups that a CU holds, and what a step of theirs (a tile, with two
// key groups two) takes in us where as many run as a CU holds, and where one runs alone.
struct MaskedKernel {
  int D, rows, key_groups, slots;
  float step, alone, block;     // block: what one takes besides
};
constexpr MaskedKernel kMaskedKernels[] = {{128, 256, 1, 1, 1.9f, 1.9f, 3.f},
                                           {128, 128, 2, 1, 2.2f, 2.05f, 4.f},
                                           {64, 128, 1, 2, 1.1f, 0.75f, 3.f},
                                           {64, 128, 2, 1, 1.3f, 1.25f, 4.f}};
// What the last blocks take where not all run at once; and a split: the merge launch, and the parts' way through
// memory.
constexpr float kTailUs = 5.f, kMaskedMergeUs = 7.f, kMaskedPartUs = 4.f / 1e7f;
inline MaskedPlan masked_plan(int B, int Hq, int Hk, int Lq, int Lk, int D, bool causal, bool ragged, int docs,
                              int cus, size_t scratch) {
  MaskedPlan p{};
  const int group = Hq / Hk;
  p.pack = group < kMaxPack ? group : kMaxPack;
  while (group % p.pack != 0) --p.pack;
  const int64_t rows = (int64_t)Lq * p.pack, units = (int64_t)(Hq / p.pack) * B;
  p.out_rows = rows * units;
  int nt = (Lk + kTileKeys - 1) / kTileKeys;
  // blocks of `block_rows` rows, `n` parts: whether the scratch holds them
  auto layout = [&](int block_rows, int key_groups, int n) {
    p.block_rows = block_rows;
    p.key_groups = key_groups;
    p.slots = 1;
    p.blocks = (rows + block_rows - 1) / block_rows * units;
    p.part_rows = (int)(rows < block_rows ? rows : block_rows);
    p.part_floats = (p.part_rows * (D + 2) + 3) / 4 * 4;
    p.splits = n;
    p.bytes = n > 1 ? (size_t)p.blocks * p.part_floats * sizeof(float) * n : 0;
    return p.bytes <= scratch;
  };
  // A run of documents ends in a block of its own: there is one for each large document and between two of them,
  // and at every 64th of all (the kernel goes through 64 at a time).
  auto by_documents = [&] {
    if (docs <= 0 || p.splits > 1) return;
    const int64_t plain = (rows + p.block_rows - 1) / p.block_rows;
    const int64_t runs = plain + 2 + docs / 64;
    p.blocks = (plain + (runs < docs + 1 ? runs : docs + 1)) * units;
    p.by_docs = true;
  };
  if (rows <= kStepRows) {
    // One workgroup a CU, a tile of 32 keys a wave at least (with more than 16 parts two, for the merge), and none
    // split that reads 128 KB at most (us with 1 / 2 / 4 / 8 / 16 / 32 parts, one token of 32 over 8 heads of 128
    // channels: 256 keys 6.2 / 7.9 / 7.6 / 7.9 / 8.8, 500 keys 9.4 / 9.9 / 8.2 / 8.5 / 9.3, 1000 keys 14.8 / 12.3 / 9.7 /
    // 8.6 / 9.4, 4000 keys 45 / 28 / 18 / 12.3 / 10.4 / 10.9; of 8 heads of 64 channels: 500 keys 6.4 / 7.3 / 6.5 / 6.7).
    // With key lengths of their own three a CU, if they are left 20 tiles each, so that the long samples do not end
    // last (us with 1 / 2 / 4 / 6 / 8 parts, 16 samples of 8 k/v heads: 8192 keys 115 / 99 / 110 / 106 / 112, 2048 to
    // 8192 keys 105 / 78 / 74 / 69 / 71, 1000 keys 20 / 20 / 25 / 30 / 31).
    int64_t n = cus / units;
    const int fine = (nt + 1) / 2 < 16 ? (nt + 1) / 2 : 16, coarse = (nt + 3) / 4;
    if (n > (fine > coarse ? fine : coarse)) n = fine > coarse ? fine : coarse;
    if (nt * D <= 512) n = 1;
    if (ragged && n < 3 * (int64_t)cus / units) {
      const int64_t more = 3 * (int64_t)cus / units < nt / 20 ? 3 * (int64_t)cus / units : nt / 20;
      if (more > n) n = more;
    }
    if (n > kMaskedMaxSplits) n = kMaskedMaxSplits;
    if (n < 1) n = 1;
    while (!layout(32, 1, (int)n)) --n;
    return p;
  }
  // (documents are of unequal length: about twice the mean of them)
  if (docs > 0 && 2 * (nt / docs + 1) < nt) nt = 2 * (nt / docs + 1);
  // Of a block's tiles (nt at most) `mean` are seen.  Without a causal mask the blocks run in rounds; with one the
  // longest come first and the launch ends with the longest or when the sum of all is done.  Over 26 random sizes
  // the choice was 4% slower than the best of both kernels and 1 to 8 parts, 20% at worst.
  const float mean = causal ? nt - 0.5f * ((Lq < Lk ? Lq : Lk) / kTileKeys) : (float)nt;
  float best = 0.f;
  const MaskedKernel* chosen = nullptr;
  int chosen_n = 1;
  for (const MaskedKernel& k : kMaskedKernels) {
    if (k.D != D) continue;
    const int tiles = k.key_groups;       // of a step
    for (int n = 1; n <= kMaskedMaxSplits && (n == 1 || n * 4 * tiles <= nt); ++n) {
      if (!layout(k.rows, k.key_groups, n)) break;
      const float wgs = (float)p.blocks * n, slots = (float)cus * k.slots;
      // a block of all tiles (where the causal ones get shorter the rest runs at a higher clock)
      auto whole = [&](float step) { return (causal ? 0.8f : 1.f) * step * ((nt + n * tiles - 1) / (n * tiles)) + k.block; };
      float us;
      if (causal) {
        const float sum = wgs * (k.step * (mean / (n * tiles) + 0.5f) + k.block) / slots;
        const float longest = whole(wgs <= cus ? k.alone : k.step);
        us = (sum > longest ? sum : longest) + (wgs > slots ? kTailUs : 0.f);
      } else {
        const float full = (float)(int64_t)(wgs / slots), rest = wgs - full * slots;
        us = full * whole(k.step) + (rest > 0.f ? whole(rest <= cus ? k.alone : k.step) : 0.f);
      }
      if (n > 1) us += kMaskedMergeUs + p.bytes * kMaskedPartUs;
      if (chosen == nullptr || us < 0.97f * best) {
        best = us;
        chosen = &k;
        chosen_n = n;
      }
    }
  }
  layout(chosen->rows, chosen->key_groups, chosen_n);
  p.slots = chosen->slots;
  by_documents();
  return p;
}

// Causal blocks come with the longest first.  Where about all run at once, two on a CU, the second of each CU are turned
// round, so that the longest runs beside the shortest: as many eights of workgroups from the cus-th on (us, 64 channels:
// 24 heads of 1000 tokens 21.9 / 20.6, of 3000 43.0 / 42.6, 32 over 8 of 2048 31.4 / 30.2, 16 over 4 of 4096 47.9 /
// 48.2; with four times as many blocks as run at once 152.0 / 153.0).
inline int masked_turn(int64_t workgroups, int cus) {
  if (cus % 8 != 0 || workgroups <= cus || workgroups >= 3 * (int64_t)cus) return 0;
  return (int)((workgroups < 2 * (int64_t)cus ? workgroups - cus : cus) / 8);
}

// ---------------------------------------------------------------------------
// the token-row kernels (prep.hip, adaln.hip)
// ---------------------------------------------------------------------------

// Their blocks: the W waves of one token row, with a wave a row (W = 1) four rows.
constexpr int rows_per_block(int W) { return W == 1 ? 4 : 1; }
constexpr int row_threads(int W) { return 64 * W * rows_per_block(W); }

// The grid of `blocks` workgroups of `threads`.  A launch has fewer than 2^32 threads along x (22
// million rows of 3072 channels at three waves a row): what is over goes on along y, with up to a
// line's last workgroups too many.
struct RowGrid {
  uint32_t x, y;
};
inline RowGrid row_grid(int64_t blocks, int threads) {
  const int64_t line = 0xffffffffll / threads, y = (blocks + line - 1) / line;
  return {(uint32_t)((blocks + y - 1) / y), (uint32_t)y};
}

// ---------------------------------------------------------------------------
// the norms of q and k heads (head_norm.hip)
// ---------------------------------------------------------------------------

// A wave holds 64 / lanes heads at once.  2^slot_shift of them are one token's, of 2^token_shift tokens;
// a token's heads are `waves_per_token` waves with `chunks` such steps each.
struct HeadNormPlan {
  int waves_per_token, slot_shift, token_shift;
  int64_t waves;
};
inline HeadNormPlan head_norm_plan(int64_t tokens, int heads, int lanes, int chunks) {
  HeadNormPlan p{};
  int slots = 0;
  while ((64 / lanes) >> (slots + 1)) ++slots;
  while (p.slot_shift < slots && (1 << p.slot_shift) < heads) ++p.slot_shift;
  p.token_shift = slots - p.slot_shift;
  const int per_wave = chunks << p.slot_shift;
  p.waves_per_token = (heads + per_wave - 1) / per_wave;
  const int64_t groups = (tokens + (1 << p.token_shift) - 1) >> p.token_shift;
  p.waves = groups * p.waves_per_token;
  return p;
}
// Heads a lane works on: one where the launch then still has few waves, else as leaves the fewest lanes
// without a head, the larger of equals.
constexpr int64_t kFewWaves = 4096;
inline int head_norm_chunks(int64_t tokens, int heads, int lanes) {
  if (head_norm_plan(tokens, heads, lanes, 1).waves <= kFewWaves) return 1;
  int best = 1;
  int64_t least = -1;
  for (int n = 4; n >= 1; --n) {
    const int64_t lanes_used = head_norm_plan(tokens, heads, lanes, n).waves * n;
    if (least < 0 || lanes_used < least) {
      least = lanes_used;
      best = n;
    }
  }
  return best;
}

// ---------------------------------------------------------------------------
// the projection GEMM (gemm.hip)
// ---------------------------------------------------------------------------

// Columns of an output tile and k per stage.
constexpr int kGemmCols = 256, kGemmBK = 64;

// Tile heights: the x rows of a workgroup's tile, and what a full round of such tiles (one
// workgroup per CU) takes, in us: per 64 of k, and besides (fitted over M 40 to 15708).
constexpr struct { int rows; float k_us; bool power; } kTiles[] = {
    {320, 1.86f, true}, {256, 1.55f, true}, {192, 1.32f, true}, {128, 0.81f, false}};
constexpr float kRoundUs = 6.f;
// A round that fills only a share of the CUs runs at a higher clock (256 rows, N 9216: a second
// round of 0.11, 0.27, 0.55, 0.69 and 0.97 of the CUs takes 54, 58, 62, 67 and 83 us, a full one
// 78); tiles of 128 rows wait for their copies and gain nothing.
inline float round_share(float fill, bool power) { return power ? 0.66f + 0.25f * fill + 0.1f * fill * fill : 1.f; }
// The merge launch, and the write and read of a part's row of 256 fp32 (plain stores: past the
// L2s, non-temporally, the calls took 3-7 us longer).
constexpr float kMergeUs = 4.f, kMergeRowUs = 2 * 256 * 4 / 8e6f;
constexpr int kGemmMaxSplits = 16, kMinSplitTiles = 4;

// The rows of a tile of x are copied from 32-bit byte offsets of its first: whether the last row's
// last byte has one.  wan_qkv_proj_sumsq takes row strides below 2^23 elements, with which it has
// in tiles of up to 256 rows; 320 rows end at 6731920 elements.
inline bool tile_addressable(int M, int rows, int64_t ldx) {
  return (int64_t)((M < rows ? M : rows) - 1) * ldx * 2 + kGemmBK * 2 <= int64_t(1) << 32;
}

// How a product is run: tiles of `rows` rows, the first `from` of them whole, the `rest` as
// `splits` parts over k each.
struct GemmPlan {
  int rows, from, rest, splits;
  float us;
};

// The plan whose rounds take least, with up to `scratch` bytes for the parts, for x rows `ldx`
// elements apart.  Between two heights the number of rounds decides, and where a last (or only)
// round leaves half of the CUs or more idle, its tiles may be split over k: the parts' fp32 sums
// cost a merge launch and their way through memory.  us, tiles of 256 rows alone / as chosen here:
//   N 9216, K 3072:   M 80  56 / 23   M 256  58 / 28   M 896  60 / 46   M 2170  136 / 98 (320 rows)
//                     M 2280  136 / 120 (a tail of 68 tiles, three parts)   M 2940  143 (256 rows)
//                     M 4480  222 / 185 (320)   M 8228  375 / 360 (320)   M 15708  690 / 680
//   N 3072, K 14336 (the best height unsplit / as chosen):   M 80  182 / 36   M 748  178 / 82
//                     M 1500  173 / 132   M 2160  187 / 172 (320 rows, three parts)   M 8228  739 / 581
inline GemmPlan gemm_plan(int M, int N, int K, int64_t ldx, int cus, size_t scratch) {
  GemmPlan best{0, 0, 0, 1, 0.f};
  const int kt = K / kGemmBK;
  for (const auto& t : kTiles) {
    if (!tile_addressable(M, t.rows, ldx)) continue;
    const int64_t tiles = ((int64_t)M + t.rows - 1) / t.rows * (N / kGemmCols);
    const int64_t full = tiles / cus;
    const int rest = (int)(tiles % cus);
    for (int n = 1; n == 1 || (rest > 0 && n <= kGemmMaxSplits && rest * n <= cus && n * kMinSplitTiles <= kt); ++n) {
      if (n > 1 && (size_t)rest * n * t.rows * kGemmCols * sizeof(float) > scratch) break;
      float us = full * (kt * t.k_us + kRoundUs);
      if (rest > 0) us += ((kt + n - 1) / n * t.k_us + kRoundUs) * round_share((float)(rest * n) / cus, t.power);
      if (n > 1) us += kMergeUs + (float)rest * n * t.rows * kMergeRowUs;
      if (best.rows == 0 || us < best.us) best = {t.rows, n > 1 ? (int)(tiles - rest) : 0, n > 1 ? rest : 0, n, us};
    }
  }
  return best;
}

inline size_t gemm_plan_bytes(const GemmPlan& p) {
  return p.splits > 1 ? (size_t)p.rest * p.splits * p.rows * kGemmCols * sizeof(float) : 0;
}

}  // namespace wan
