// Attention over the paged cache for many rows (gfx950): chunks and whole prompts.
//
// One workgroup = 4 waves = 128 rows of one key head, 32 per wave; two workgroups per CU (registers and half of the LDS;
// one where values are wider than 128 columns), each with its own barriers: what one does between its products runs under
// the other's.  (4 x 1,024 rows x 8 heads over 8,024 keys: D 64, R 32 126 us, D 128, R 64 239; as one workgroup of 8 waves,
// two groups of 4 that took turns with the key blocks, 151 and 273.)
//
// Bound by the matrix cores where the chip is full, and by the heaviest tiles where it is not.  Measured: prompts of 4,096
// tokens x 8 heads, 2 of them, D 64, R 32: 80 us and 9 for the join, 540 TFLOP/s of what the formula has and 860 with the
// second part of Q_hat; the matrix cores are busy 38 % of the cycles, 1.55 of 2 waves per SIMD alive (causal tiles end at
// different times).  130 rows over 16,000 keys, 8 heads, D 64, R 64: 32 us and 4; 46 MB, in 512 parts of 16 blocks whose
// start and end cost as much as their keys.  20 rows (5 tokens x 4 query heads) of 16 sequences of up to 4,101 keys, 8 key
// heads, D 128, R 64, 200 MB: 48 us and 4.5, 4.2 TB/s.
//
// Blocks of K and V go to LDS as they lie in the pages (direct loads, no registers), into a ring of three to eight
// stages: while step t is in use and t + 1 has landed, the others are on their way.  Pages hold operands of 16x16
// MFMAs in units of 8 elements, and a unit is 8 consecutive k elements of one row: the 32x32x16 products here read the
// same units in another order.  S^T row x of the product is key 16 (x / 8 % 2) + 8 (x / 16) + x % 8 of the block, so that
// a lane's scores 8 s .. 8 s + 7 belong, in order, to the eight keys of the V unit of group 2 s + lane / 32, and P goes
// from product to product in registers.  Eight consecutive lanes always read consecutive units: no bank conflicts, and
// every read is one base register and an immediate.  8-bit codes are unpacked behind the LDS read.
//
// A step's score products run between the exponentials of the step before (a wave alone keeps both units busy), its
// P V products between the maxima of the scores just made.  The running maximum m moves only when a row's maximum
// exceeds it by more than 2^8 in p (or is the row's first): p <= 2^8 loses nothing, and O is rescaled rarely.
//
// Precision: as in paged_attn.hpp, but P is rounded once to 16 bits (8-bit pages: times the value's scale, to bf16; two parts where
// outputs are fp16): its second part would double the second product, a quarter of all products at R = D / 2.  Against
// 64 bits, relative to the output's norm, bf16 0.0021-0.0024 (an fp32 computation rounded once: 0.0016), fp16 0.00029
// (0.00021).  l sums what P was before.
#pragma once
#include <type_traits>

#include "paged_dev.hpp"

namespace pope {

template <bool Q8, int KS, int VT>
struct PagedRows {
  static constexpr int kRows = 128;
  static constexpr int kKB = KS * (Q8 ? 1024 : 2048), kVB = VT * (Q8 ? 512 : 1024);   // bytes of a staged block's K and V
  static constexpr int kBlock = kKB + kVB;
  static constexpr int kRegs = KS * 16 + VT * 8;                     // of Q_hat (two parts) and O
  static constexpr bool kPipe = kRegs + 40 <= 170;                   // scores of two steps at once
  static constexpr int BG = 2 * kBlock * 3 <= 79 * 1024 && VT <= 8 && kRegs + (kPipe ? 64 : 32) <= 150 ? 2 : 1;   // blocks per step
  static constexpr int kStage = BG * (kBlock + (Q8 ? 64 : 0));    // 8-bit: the blocks' exponents behind them
  static constexpr int kLds = (VT <= 8 ? 80 : 160) * 1024, kFit = (kLds - 128) / kStage, kSlots = kFit < 8 ? kFit : 8;
  static constexpr int QST = KS * 32 + 8;
  // rows of Q_hat made at a time
  static constexpr int kQRows = 128 * QST * 4 <= kStage ? 128 : 64 * QST * 4 <= kStage ? 64 : 32;
  static constexpr int kBytes = kSlots * kStage;
  // stages that load while Q_hat is made behind them
  static constexpr int kEarly = (kBytes - kQRows * QST * 4) / kStage < kSlots - 1 ? (kBytes - kQRows * QST * 4) / kStage : kSlots - 1;
  static_assert(kSlots >= 3 && kEarly >= 1 && kBytes + 128 <= kLds, "LDS");
};

template <typename T, bool Q8, int KS, int VT>
__global__ __launch_bounds__(256, VT <= 8 ? 2 : 1) void paged_rows_kernel(PagedAttnParams p) {
  using C = PagedRows<Q8, KS, VT>;
  typedef typename T::vec8 vec8;
  // The second product's type: P x 2^e (8-bit values' scales) leaves fp16's range where values are far from 1.  fp16 outputs
  // then take P as two bf16 parts.
  typedef std::conditional_t<Q8, BF16, T> V;
  typedef typename V::vec8 vvec8;
  constexpr int kParts = Q8 && T::kCode == 1 ? 2 : 1;
  constexpr int BG = C::BG, NDB = VT / 2, K16 = 2 * KS, kRows = C::kRows;
  __shared__ __attribute__((aligned(16))) char smem[C::kBytes];
  // Per (step % 8, block of the step): keys of values that are not finite.  Never cleared: add_seen looks at the value again.
  __shared__ uint32_t odd[32];
  const PagedCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), lr = lane & 31, hf = lane >> 5;

  const PagedPlan job = paged_plan(p, kRows);
  const int hk = (int)(blockIdx.x % (unsigned)c.Hk);
  const PagedTile& t = job.t;
  const PagedSeg& g = t.seg;
  const int rows_all = g.n * (int)p.G.d, r0 = t.local * kRows;
  if (r0 >= rows_all) return;
  const bool causal = p.causal != 0;
  const int blocks = paged_tile_blocks(g, t.local, kRows, p.G, causal);
  const int parts = paged_parts(blocks, p.splits, job.least, 1);
  const PagedRange range = paged_range(blocks, p.splits, job.least, 1, job.split);
  if (job.split > 0 && range.begin >= range.end) return;
  if (p.splits > 1 && job.split == 0 && tid == 0) p.parts[(int64_t)job.tile * c.Hk + hk] = parts;

  // ---- the lane's row, and the keys that all of the wave's (of the tile's) rows see -----------------------------
  const PagedRowMap map(r0, p.G);
  const int count = min(rows_all - r0, kRows), x = wave * 32 + lr;   // the lane's row of the tile
  const bool live = x < count;
  const int row_i = live ? map.token(x) : 0, row_h = live ? map.group(x) * c.Hk + hk : hk;
  const int lim = live ? paged_limit(g.first + row_i, g.len, causal) : 0;
  const int least_lim = wave * 32 < count ? paged_limit(g.first + map.token(wave * 32), g.len, causal) : 0;
  const int tile_lim = paged_limit(g.first + map.i0, g.len, causal);   // the first row sees the fewest keys

  // ---- staging -------------------------------------------------------------------------------------------------
  // A step's blocks are dealt to the waves, 4 / BG waves per block, so that a wave finds one page per step.  Page numbers
  // of 64 pages at a time, one per lane; `lost`: some page was outside the cache (then gone_of looks closer).
  const int steps = (range.end - range.begin + BG - 1) / BG;
  constexpr int kPer = C::kBlock / 1024, kShare = 4 / BG;   // a block's units of 64 x 16 bytes; waves per block
  constexpr int kWaveUnits = (kPer + kShare - 1) / kShare, kLeast = kPer / kShare;   // units a wave has at most / at least
  constexpr int kE = Q8 ? 1 : 2;
  const int my_block = wave / kShare, my_part = wave % kShare;
  const int cols = c.seqs.capacity >> (c.blk_shift + 5);
  int page_base = range.begin >> c.blk_shift, pids = 0;
  bool lost = false;
  auto window = [&] {
    const int id = g.b >= 0 ? c.table[(int64_t)g.b * c.table_sb + min(page_base + lane, cols - 1)] : -1;
    pids = (unsigned)id < (unsigned)c.pages ? id : -1;
    lost |= __any(pids < 0 && page_base + lane <= (range.end - 1) >> c.blk_shift);
    pids = max(pids, 0);   // loads of pages outside the cache read page 0 and are masked
  };
  if (steps > 0) window();
  const int64_t k_page = (int64_t)c.Hk * c.k_head * kE, v_page = (int64_t)c.Hk * c.v_head * kE;
  const char* k_at = static_cast<const char*>(c.k) + hk * c.k_head * kE + my_part * 1024;
  const char* v_at = static_cast<const char*>(c.v) + hk * c.v_head * kE + (my_part * 1024 - C::kKB);
  auto issue = [&](int step, int slot) {   // slot: byte offset of the stage
    const int first = range.begin + step * BG, blk = min(first + my_block, range.end - 1), pg = blk >> c.blk_shift, sub = blk - (pg << c.blk_shift);
    if ((first >> c.blk_shift) + BG - page_base > 64) {   // the same for all waves: `lost` has to be
      POPE_COLD_PATH();
      page_base = first >> c.blk_shift;
      window();
    }
    const int page = __builtin_amdgcn_readlane(pids, pg - page_base);
    const char* k_src = k_at + page * k_page + sub * C::kKB;
    const char* v_src = v_at + page * v_page + sub * C::kVB;
    const uint32_t dst = lds_addr(smem) + slot + my_block * C::kBlock + my_part * 1024;
#pragma unroll
    for (int i = 0; i < kWaveUnits; ++i) {   // unit my_part + i kShare
      const int x = i * kShare;
      if (x + kShare > kPer && x + my_part >= kPer) break;
      const bool key = x + kShare <= C::kKB / 1024 || (x < C::kKB / 1024 && x + my_part < C::kKB / 1024);
      load_lds16((key ? k_src : v_src) + x * 1024, lane * 16, dst + x * 1024);
    }
    if (Q8 && my_part == 0 && lane < 4)   // the block's 64 bytes of exponents
      load_lds16(c.scales + (((((int64_t)page * c.Hk + hk) << c.blk_shift) + sub) * 64 + lane * 16), lds_addr(smem) + slot + BG * C::kBlock + my_block * 64);
  };

  // ---- the loop --------------------------------------------------------------------------------------------------
  vec8 qh[K16], ql[K16];
  f32x16 acc[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  // m: the reference maximum, log2 units (0 until a row has seen a key); its negative is where S starts from
  float m = 0.f, l = 0.f;
  bool set = false;
  constexpr bool kKeep = C::kRegs + (C::kPipe ? 40 : 24) * BG <= 160;   // registers for 16 copies of it
  f32x16 negm;
#pragma unroll
  for (int i = 0; i < 16; ++i) negm[i] = 0.f;
  // operand bases within a block: K row lr of the product is key kkey
  const int kkey = 16 * ((lr >> 3) & 1) + 8 * (lr >> 4) + (lr & 7);
  const int kbase = Q8 ? ((kkey & 15) + 16 * hf) * 16 + (kkey >> 4) * 8 : (kkey >> 4) * 1024 + ((kkey & 15) + 16 * hf) * 16;
  const int vbase = C::kKB + (Q8 ? ((lr & 15) + 16 * hf) * 16 + (lr >> 4) * 8 : (lr >> 4) * 1024 + ((lr & 15) + 16 * hf) * 16);
  // the lane's key of score x, less 4 hf
  auto key_of = [](int x) { return 16 * ((x >> 2) & 1) + 8 * (x >> 3) + (x & 3); };
  // the group's blocks of a step; `slot`: byte offset of its stage
  auto stage_of = [&](int slot) -> const char* { return smem + slot; };
  auto scales_of = [&](int slot, int b) -> const uint8_t* { return reinterpret_cast<const uint8_t*>(smem + slot + BG * C::kBlock + b * 64); };
  auto first_block = [&](int st) { return range.begin + st * BG; };
  auto gone = [&](int blk) { return lost && (g.b < 0 || paged_page(c, g.b, min(blk, range.end - 1)) < 0); };
  // whether some block of the step has keys that some row of the wave (of the tile) does not see
  const int free_blocks = min(least_lim / kBlockKeys, range.end), tile_blocks = min(tile_lim / kBlockKeys, range.end);
  auto edge_of = [&](int st) { return first_block(st) + BG > free_blocks || lost; };
  using Raw = std::conditional_t<Q8, u32x2, u32x4>;   // an operand as it lies in LDS
  auto k_read = [&](const char* stage, int b, int k) -> Raw {
    return *reinterpret_cast<const Raw*>(stage + b * C::kBlock + kbase + ((k >> 1) * 2048 + (k & 1) * (Q8 ? 1024 : 512)) / (Q8 ? 2 : 1));
  };
  auto v_read = [&](const char* stage, int b, int d, int h) -> Raw {
    return *reinterpret_cast<const Raw*>(stage + b * C::kBlock + vbase + (d * 2048 + h * (Q8 ? 1024 : 512)) / (Q8 ? 2 : 1));
  };
  auto operand = [&](Raw w, float unit) -> vec8 {
    if constexpr (Q8) return as_vec8<vec8>(unpack_e4m3<T>(w, unit));
    else return as_vec8<vec8>(w);
  };
  auto v_operand = [&](Raw w) -> vvec8 {
    if constexpr (Q8) return as_vec8<vvec8>(unpack_e4m3<V>(w, 1.f));
    else return as_vec8<vvec8>(w);
  };
  auto power = [](uint32_t w, int i) { return __uint_as_float(((w >> (8 * i)) & 0xffu) << 23); };   // 2^(byte i - 127)
  // S of a step.  8-bit: bf16 holds code x 2^e, so the scale goes into the unpacking; fp16 does not, the scores take it.
  constexpr bool kUnpackScale = Q8 && T::kCode == 2, kLate = T::kCode == 1;
  // The loop's two bursts of products, in an explicit order (a fence behind each operand's products): operand reads run
  // kAhead operands in front, and every product is followed by its share of the vector work that the burst covers.  Left
  // to the compiler, each read stood right before its product and the vector work in front of or behind them all, and a
  // step of two workgroups took the sum of both, 3,700 cycles at D 64, R 32; it takes 2,860 so (the products alone: 2,048).
  constexpr int kAhead = Q8 || VT < 8 ? 6 : 4;
  // what the products do not carry: fp16 takes a row's scale, and a softmax scale above 1, behind them
  auto finish = [&](int slot, f32x16* s) {
    if constexpr (kLate) {
      if (Q8 || p.late != 1.f) {
#pragma unroll
        for (int b = 0; b < BG; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w = Q8 ? *reinterpret_cast<const uint32_t*>(scales_of(slot, b) + paged_scale_off(key_of(4 * q) + 4 * hf, 0)) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[b][4 * q + i] = s[b][4 * q + i] * ((Q8 ? power(w, i) : 1.f) * p.late) - m;
          }
      } else {
#pragma unroll
        for (int b = 0; b < BG; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[b][i] -= m;
      }
    }
  };
  auto scores = [&](int slot, f32x16* s, auto&& between) {
    const char* stage = stage_of(slot);
    float unit[BG];
    if constexpr (!kKeep) {
#pragma unroll
      for (int i = 0; i < 16; ++i) negm[i] = kLate ? 0.f : -m;
    }
#pragma unroll
    for (int b = 0; b < BG; ++b) unit[b] = kUnpackScale ? __uint_as_float((uint32_t)scales_of(slot, b)[paged_scale_off(kkey, 0)] << 23) : 1.f;
    constexpr int n = K16 * BG;
    Raw w[n];
#pragma unroll
    for (int i = 0; i < kAhead && i < n; ++i) w[i] = k_read(stage, i % BG, i / BG);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int b = i % BG, k = i / BG;
      const vec8 a = operand(w[i], unit[b]);
      s[b] = T::mfma32(a, qh[k], k ? s[b] : negm);
      if (i + kAhead < n) w[i + kAhead] = k_read(stage, (i + kAhead) % BG, (i + kAhead) / BG);
      between(2 * i, 2 * n);
      __builtin_amdgcn_sched_barrier(0);
      s[b] = T::mfma32(a, ql[k], s[b]);
      between(2 * i + 1, 2 * n);
      __builtin_amdgcn_sched_barrier(0);
    }
    finish(slot, s);
  };
  // the same in the second pass: finite elements of K times both parts of Q_hat, the others times its signs
  auto careful_scores = [&](int slot, f32x16* s) {
    const char* stage = stage_of(slot);
#pragma unroll
    for (int b = 0; b < BG; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = kLate ? 0.f : -m;
#pragma unroll
    for (int i = 0; i < K16 * BG; ++i) {
      const int b = i % BG, k = i / BG;
      u32x4 w, fin, rest;
      if constexpr (!Q8) w = k_read(stage, b, k);
      split_finite<T>(w, &fin, &rest);
      s[b] = T::mfma32(as_vec8<vec8>(fin), qh[k], s[b]);
      s[b] = T::mfma32(as_vec8<vec8>(fin), ql[k], s[b]);
      if (__any((rest[0] | rest[1] | rest[2] | rest[3]) != 0)) s[b] = T::mfma32(as_vec8<vec8>(rest), sign_operand<T>(qh[k]), s[b]);
    }
    finish(slot, s);
  };
  auto mask = [&](int st, f32x16* s) {
#pragma unroll
    for (int b = 0; b < BG; ++b) {
      const int blk = first_block(st) + b, left = blk >= range.end || gone(blk) ? 0 : lim - blk * kBlockKeys - 4 * hf;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = key_of(i) < left ? s[b][i] : -INFINITY;
    }
  };
  auto row_max = [&](const f32x16* s) {
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < BG; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    return half_swap_max(mx);
  };
  // m moves where a row's maximum (relative to m) is above 8, or to the row's first maximum
  auto rescale = [&](float mx, f32x16* s) {
    const bool need = mx > -INFINITY && (!set || mx > 8.f);
    if (__any(need)) {
      POPE_COLD_PATH();
      const float up = need ? mx : 0.f, alpha = need && set ? __builtin_amdgcn_exp2f(-mx) : 1.f;
      m += up;
      set |= need;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
#pragma unroll
      for (int b = 0; b < BG; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] -= up;
      if constexpr (kKeep && !kLate) {
#pragma unroll
        for (int i = 0; i < 16; ++i) negm[i] = -m;
      }
    }
  };
  // Unit u of BG x 8: two probabilities, their share of the sum, packed (8-bit: times the values' scales).
  auto prob = [&](int slot, f32x16* s, u32x4 (*pw)[2 * kParts], int u) {
    const int b = u / 8, q = u % 8;
    float x[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      x[k] = __builtin_amdgcn_exp2f(s[b][2 * q + k]);
      l += x[k];
    }
    if constexpr (Q8) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(scales_of(slot, b) + paged_scale_off(key_of(4 * (q / 2)) + 4 * hf, 1));
#pragma unroll
      for (int k = 0; k < 2; ++k) x[k] *= power(w, 2 * (q & 1) + k);
    }
    pw[b][q >> 2][q & 3] = V::pack2(x[0], x[1]);
    if constexpr (kParts == 2) {
      const uint32_t w = pw[b][q >> 2][q & 3];
      pw[b][2 + (q >> 2)][q & 3] = V::pack2(x[0] - V::to_float((uint16_t)w), x[1] - V::to_float((uint16_t)(w >> 16)));
    }
    if constexpr (C::kPipe) asm volatile("" : "+v"(pw[b][q >> 2][q & 3]), "+v"(l));   // stays between its fences
    s[b][2 * q] = x[0];
    s[b][2 * q + 1] = x[1];
  };
  auto probs = [&](int slot, f32x16* s, u32x4 (*pw)[2 * kParts]) {
#pragma unroll
    for (int u = 0; u < 8 * BG; ++u) prob(slot, s, pw, u);
  };
  auto products = [&](int slot, const u32x4 (*pw)[2 * kParts], auto&& between) {
    const char* stage = stage_of(slot);
    constexpr int n = BG * 2 * NDB, ahead = n < 4 ? n : 4;
    Raw w[n];
#pragma unroll
    for (int i = 0; i < ahead; ++i) w[i] = v_read(stage, i / (2 * NDB), i % NDB, i / NDB % 2);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int b = i / (2 * NDB), h = i / NDB % 2, d = i % NDB;
      const vvec8 a = v_operand(w[i]);
      acc[d] = V::mfma32(a, as_vec8<vvec8>(pw[b][h]), acc[d]);
      if constexpr (kParts == 2) acc[d] = V::mfma32(a, as_vec8<vvec8>(pw[b][2 + h]), acc[d]);
      if (i + ahead < n) w[i + ahead] = v_read(stage, (i + ahead) / (2 * NDB), (i + ahead) % NDB, (i + ahead) / NDB % 2);
      between(i, n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto nothing = [](int, int) {};
  // Blocks with keys that some row of the tile does not see: 0 x NaN must not count.  Slots from len on, and pages outside
  // the cache, hold whatever was there and become zeros in the stage; values that are not finite do too, and their keys are
  // noted, for `add_seen` to add them outside the product where they are seen.
  // The second pass (rows that infinite keys or values made NaN, paged_dev.hpp) does so in all blocks.
  auto tile_edge = [&](int st) { return range.begin + (st + 1) * BG > tile_blocks || lost; };
  auto sanitize = [&](int st, int slot) {
    char* stage = smem + slot;
    for (int u = tid; u < BG * (C::kVB / 16); u += 256) {
      const int b = u / (C::kVB / 16), x = u % (C::kVB / 16), blk = range.begin + st * BG + b;
      const int have = gone(blk) ? 0 : g.len - blk * kBlockKeys - 4 * ((x & 63) >> 4);
      uint32_t* w = reinterpret_cast<uint32_t*>(stage + b * C::kBlock + C::kKB + x * 16);
      // an element with all exponent bits set (8-bit: a NaN code) carries into its sign bit
      const u32x4 v4 = *reinterpret_cast<const u32x4*>(w);
      constexpr uint32_t kMag = Q8 ? 0x7f7f7f7fu : 0x7fff7fffu, kOne = Q8 ? 0x01010101u : T::kCode == 2 ? 0x00800080u : 0x04000400u;
      uint32_t carry = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) carry |= ((v4[i] & kMag) + kOne) & ~kMag;
      if (!carry && have >= 20) continue;   // all 8 keys, 16 (j / 4) + j % 4, are there
      uint32_t noted = 0;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        uint32_t v = w[i], keep = 0;
#pragma unroll
        for (int e = 0; e < (Q8 ? 4 : 2); ++e) {   // element j of a unit: key 16 (j / 4) + j % 4 (8-bit: two units of 8)
          const int j = Q8 ? (4 * i + e) & 7 : 2 * i + e, key = 16 * (j >> 2) + (j & 3);
          const uint32_t x1 = Q8 ? (v >> (8 * e)) & 0xffu : (v >> (16 * e)) & 0xffffu;
          const bool in = key < have, fin = Q8 ? (x1 & 0x7f) != 0x7f : !nonfinite16<T>(x1);
          keep |= in && fin ? (Q8 ? 0xffu << (8 * e) : 0xffffu << (16 * e)) : 0u;
          noted |= in && !fin ? 1u << (key + 4 * ((x & 63) >> 4)) : 0u;
        }
        w[i] = v & keep;
      }
      if (noted) atomicOr(&odd[(st & 7) * 4 + b], noted);
    }
  };
  auto add_seen = [&](int st, const f32x16* s) {
#pragma unroll
    for (int b = 0; b < BG; ++b) {
      uint32_t keys = __builtin_amdgcn_readfirstlane(odd[(st & 7) * 4 + b]);
      const int blk = first_block(st) + b;
      if (keys && blk < range.end) {
        POPE_COLD_PATH();
        const int page = paged_page(c, g.b, blk);
        if (page < 0) continue;
        const int64_t at = paged_block_off(c, page, hk, blk, c.v_head, VT * 512);
#pragma unroll 1
        for (; keys; keys &= keys - 1) {
          const int key = __builtin_ctz(keys), q = (key & 15) >> 2, x = 8 * (q >> 1) + 4 * (key >> 4) + (key & 3);
          float pk = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) pk = i == x ? s[b][i] : pk;
          pk = __shfl(pk, lr + 32 * (q & 1), 64);
          const bool seen = blk * kBlockKeys + key < lim;
#pragma unroll
          for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int64_t off = at + paged_v_off(Q8, key, 32 * d + 8 * (i >> 2) + 4 * hf + (i & 3));
              const uint32_t w = Q8 ? ((static_cast<const uint8_t*>(c.v)[off] & 0x7f) == 0x7f ? 0x7fffu : 0u) : static_cast<const uint16_t*>(c.v)[off];
              if (nonfinite16<T>(w) && seen) acc[d][i] = fmaf(pk, T::to_float((uint16_t)w), acc[d][i]);
            }
        }
      }
    }
  };

  if (tid < 32) odd[tid] = 0;
  constexpr int RB = C::kQRows, kTurns = (RB * VT * 2 + 255) / 256;   // rows at a time, chunks per thread
  PagedQueryIn in[kRows / RB][kTurns];
#pragma unroll
  for (int b = 0; b < kRows / RB; ++b)
#pragma unroll
    for (int k = 0; k < kTurns; ++k) in[b][k] = paged_query_load<T>(p, g, map, b * RB + (tid + 256 * k) % RB, count, hk, (tid + 256 * k) / RB * 8);
  __builtin_amdgcn_sched_barrier(0);
  auto next_slot = [](int slot) { return slot + C::kStage == C::kSlots * C::kStage ? 0 : slot + C::kStage; };
  int put = 0;   // stage of the next step to issue
#pragma unroll
  for (int st = 0; st < C::kEarly; ++st) {
    if (st < steps) issue(st, put);
    put += C::kStage;
  }
  // ---- Q_hat, through the stages behind, while the first ones load ---------------------------------------------
  {
    uint16_t* hi = reinterpret_cast<uint16_t*>(smem + C::kEarly * C::kStage);
    uint16_t* lo = hi + RB * C::QST;
#pragma unroll
    for (int x0 = 0; x0 < kRows; x0 += RB) {
      if (x0) __syncthreads();
#pragma unroll
      for (int k = 0; k < kTurns; ++k)
        paged_query_make<T>(p, in[x0 / RB][k], __any(x0 + (tid + 256 * k) % RB < count), (tid + 256 * k) % RB, (tid + 256 * k) / RB * 8, C::QST, hi, lo);
      paged_query_tail<RB>(p, tid, 256, KS * 32, C::QST, hi, lo);
      __syncthreads();
      if (wave * 32 >= x0 && wave * 32 < x0 + RB) {
        const int at = (x - x0) * C::QST + 8 * hf;
#pragma unroll
        for (int k = 0; k < K16; ++k) {
          qh[k] = as_vec8<vec8>(*reinterpret_cast<const u32x4*>(hi + at + 16 * k));
          ql[k] = as_vec8<vec8>(*reinterpret_cast<const u32x4*>(lo + at + 16 * k));
        }
      }
    }
  }
  if constexpr (C::kEarly < C::kSlots - 1) {
    __syncthreads();   // the last rows of Q_hat have been read
    for (int st = C::kEarly; st < C::kSlots - 1; ++st) {
      if (st < steps) issue(st, put);
      put += C::kStage;
    }
  }
  // Loads of steps up to `st` have landed; later ones, with at least kLeast loads of this wave each, may be in flight.
  auto landed = [&](int st) {
    constexpr int most = C::kSlots - 2 - (C::kPipe ? 1 : 0);
    if (steps - 1 - st >= most) wait_vmcnt<most * kLeast>();
    else wait_vmcnt<0>();   // the last steps were issued long ago
  };
  auto refill = [&](int st) {   // behind the barrier that ends the use of stage st - 1
    if (st + C::kSlots - 1 < steps) issue(st + C::kSlots - 1, put);
    put = next_slot(put);
  };
  const bool idle = wave * 32 >= count;
  f32x16 sa[BG], sb[C::kPipe ? BG : 1];
  u32x4 pw[BG][2 * kParts];
  int slot = 0;   // stage of the current step
  if (idle) {   // a wave without rows: the others' loads and barriers
    int at = 0;
    if constexpr (C::kPipe) {
      if (steps > 0) {
        wait_vmcnt<0>();
        __syncthreads();
        if (tile_edge(0)) sanitize(0, 0);
        for (int st = 0; st + 1 < steps; ++st) {
          landed(st + 1);
          __syncthreads();
          refill(st);
          at = next_slot(at);
          if (tile_edge(st + 1)) sanitize(st + 1, at);
        }
        __syncthreads();
      }
    } else {
      for (int st = 0; st < steps; ++st) {
        landed(st);
        __syncthreads();
        refill(st);
        if (tile_edge(st)) {
          sanitize(st, at);
          __syncthreads();
        }
        at = next_slot(at);
      }
    }
  } else {
    if constexpr (C::kPipe) {
      float mx = -INFINITY;
      if (steps > 0) {
        if (steps >= C::kSlots - 1) wait_vmcnt<(C::kSlots - 2) * kLeast>();
        else wait_vmcnt<0>();
        __syncthreads();
        if (tile_edge(0)) {
          POPE_COLD_PATH();
          sanitize(0, 0);
        }
        scores(0, sa, nothing);
        if (edge_of(0)) {
          POPE_COLD_PATH();
          mask(0, sa);
        }
        mx = row_max(sa);
      }
      auto step = [&](int st, f32x16* cur, f32x16* nxt) {
        const int ahead = next_slot(slot);
        rescale(mx, cur);
        landed(st + 1);
        __syncthreads();   // stage st + 1 is whole, and the values of stage st are clean; stage st - 1 is free
        refill(st);
        if (tile_edge(st + 1)) {
          POPE_COLD_PATH();
          sanitize(st + 1, ahead);   // its V is read behind the next barrier
        }
#pragma unroll
        for (int b = 0; b < BG; ++b) asm volatile("" : "+v"(cur[b]));   // nothing of it above the branches before
        scores(ahead, nxt, [&](int i, int n) {
#pragma unroll
          for (int u = i * 8 * BG / n; u < (i + 1) * 8 * BG / n; ++u) prob(slot, cur, pw, u);
        });
        if (edge_of(st + 1)) {
          POPE_COLD_PATH();
          mask(st + 1, nxt);
        }
        mx = -INFINITY;
        products(slot, pw, [&](int i, int n) {
#pragma unroll
          for (int x = i * 16 * BG / n; x < (i + 1) * 16 * BG / n; ++x) mx = fmaxf(mx, nxt[x / 16][x % 16]);
          asm volatile("" : "+v"(mx));
        });
        mx = half_swap_max(mx);
        if (tile_edge(st)) {
          POPE_COLD_PATH();
          add_seen(st, cur);
        }
        slot = ahead;
      };
      auto last = [&](int st, f32x16* cur) {
        __syncthreads();   // the values of stage st are clean
        rescale(mx, cur);
        probs(slot, cur, pw);
        products(slot, pw, nothing);
        if (tile_edge(st)) {
          POPE_COLD_PATH();
          add_seen(st, cur);
        }
      };
      int st = 0;
      for (; st + 2 < steps; st += 2) {
        step(st, sa, sb);
        step(st + 1, sb, sa);
      }
      if (st + 2 == steps) {
        step(st, sa, sb);
        last(st + 1, sb);
      } else if (st + 1 == steps) {
        last(st, sa);
      }
    } else {
      for (int st = 0; st < steps; ++st) {
        landed(st);
        __syncthreads();   // stage st is whole; stage st - 1 is free
        refill(st);
        const bool edge = tile_edge(st);
        if (edge) {
          POPE_COLD_PATH();
          sanitize(st, slot);
          __syncthreads();
        }
        scores(slot, sa, nothing);
        if (edge_of(st)) {
          POPE_COLD_PATH();
          mask(st, sa);
        }
        rescale(row_max(sa), sa);
        // the first half of the keys' probabilities, the second half's under the first half's products
#pragma unroll
        for (int u = 0; u < 4; ++u) prob(slot, sa, pw, u);
        products(slot, pw, [&](int i, int) {
#pragma unroll
          for (int u = 4 + 4 * i / NDB; u < 8 && u < 4 + 4 * (i + 1) / NDB; ++u) prob(slot, sa, pw, u);
        });
        if (edge) {
          POPE_COLD_PATH();
          add_seen(st, sa);
        }
        slot = next_slot(slot);
      }
    }
  }
  // ---- a second pass, for rows that infinite keys or values made NaN (paged_dev.hpp) ----------------------------
  if constexpr (!Q8) {
    float x = l;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) x += acc[d][i];
    if (__builtin_expect(__any(x != x), false)) {
      POPE_COLD_PATH();
      bool fin = true;
#pragma unroll
      for (int k = 0; k < K16; ++k) fin = fin && all_finite<T>(qh[k]);
      const uint64_t nan = __ballot(x != x && live), off = __ballot(!fin);   // of a row: in either of its lanes
      if ((uint32_t)(nan | nan >> 32) & ~(uint32_t)(off | off >> 32)) odd[3] = 1;   // no step has a fourth block
    }
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(odd[3]), 0)) {
      POPE_COLD_PATH();
      m = l = 0.f;
      set = false;
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
      page_base = range.begin >> c.blk_shift;
      window();
      put = 0;
#pragma unroll 1
      for (int st = 0; st < C::kSlots - 1; ++st) {
        if (st < steps) issue(st, put);
        put += C::kStage;
      }
      slot = 0;
#pragma unroll 1
      for (int st = 0; st < steps; ++st) {
        landed(st);
        __syncthreads();
        refill(st);
        sanitize(st, slot);
        __syncthreads();
        if (!idle) {
          careful_scores(slot, sa);
          mask(st, sa);
          rescale(row_max(sa), sa);
          probs(slot, sa, pw);
          products(slot, pw, nothing);
          add_seen(st, sa);
        }
        slot = next_slot(slot);
      }
    }
  }
  l += wave_shfl_xor(l, 32);

  // ---- output, or this split's part -----------------------------------------------------------------------------
  if (!live) return;
  if (!set) m = -INFINITY;
  const bool part = parts > 1;
  const float f = part ? 1.f : l == 0.f ? 0.f : 1.f / l;
  const int64_t row = part ? (((int64_t)job.tile * c.Hk + hk) * kRows + x) * p.splits + job.split : 0;
  uint16_t* dst = p.o + (int64_t)g.batch * p.o_s[0] + (int64_t)row_h * p.o_s[1] + (int64_t)(g.row0 + row_i) * p.o_s[2];
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = 32 * d + 8 * q + 4 * hf;
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = acc[d][4 * q + i] * f;
      if (!part) x = averages<T>(x);
      if (part) {
        *reinterpret_cast<f32x4*>(p.part_o + row * (VT * 16) + col) = x;
      } else if (p.o_vec) {
        if (col < c.D) *reinterpret_cast<u32x2*>(dst + col) = u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < c.D) dst[col + i] = T::bits(x[i]);
      }
    }
  if (hf == 0) {
    if (part) *reinterpret_cast<float2*>(p.part_ml + row * 2) = make_float2(m, l);
    else if (p.lse)
      p.lse[((int64_t)g.batch * p.Hq + row_h) * p.N + g.row0 + row_i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

}  // namespace pope
