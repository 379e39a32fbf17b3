// Dispatch rules that are arithmetic on sizes and alignments alone: plain C++, so that a test can hold
// them against what the kernels behind them assume, without a GPU.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace cti {

// Whether the ragged kernel may read a table of `rows` rows of `dim` elements of `elem_bytes`, `row_bytes`
// apart from `base` on, with buffer loads: rows of at least one 16-byte chunk, every chunk 4-byte aligned
// (the last one ends with the row, so the row's own length counts beside the base and the stride; it also
// keeps the table's end, where loads past a bag go, a whole number of words away), and no offset from the
// end on, by up to a row, wrapping around 32 bits.
inline bool ragged_buffer_loads(uint64_t base, int64_t rows, int64_t row_bytes, int64_t dim, int elem_bytes) {
  const int64_t len = dim * elem_bytes;
  const int64_t span = (rows - 1) * row_bytes + len;
  return len >= 16 && base % 4 == 0 && row_bytes % 4 == 0 && len % 4 == 0 && span + len < (int64_t{1} << 32);
}

// ---------------------------------------------------------------------------------------------
// LayerNorm-Linear: y [M, N] = a [M, K] w^T, K in steps of kLinearStep.
// ---------------------------------------------------------------------------------------------
constexpr int kLinearStep = 64;
constexpr int kLinearCus = 256;                 // one workgroup per CU
constexpr int kLinearBandParams = 28 * 1024;    // LDS of the band form for gamma and beta

enum LinearForm {
  kLinearGeneral,  // any K: 64 x 256 tiles
  kLinearTile128,  // K a multiple of 128, byte offsets below 2^31: 128 x 128 tiles, K split if they are few
  kLinearTile256,  // 128 x 256 tiles, from two per CU on
  kLinearBand,     // bands of 128 rows by 256, 384 or 512 columns, K split if they are few
};
struct LinearPlan {
  LinearForm form;
  int splits;  // of K: 1, or as many fp32 partial products as the workspace then has to hold
  int steps;   // per split (even)
};

constexpr int64_t linear_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Column fragments per wavefront of the band form: 8 wavefronts cover N = 256, 384 or 512 columns.
inline int linear_band_fragments(int32_t N) { return N <= 256 ? 2 : (N <= 384 ? 3 : 4); }
inline int64_t linear_band_tiles(int64_t M, int32_t N) {
  return linear_ceil(M, 128) * linear_ceil(N, 128 * linear_band_fragments(N));
}

// Splits K into at most `want` parts of even step counts, as many as `ws_bytes` of fp32 partials hold;
// 1 = no split. `steps` receives the steps per split.
inline int linear_split(int64_t want, int64_t M, int32_t N, int32_t K, int64_t ws_bytes, int* steps) {
  const int nk = K / kLinearStep;
  *steps = nk;
  if (want <= 1 || nk < 4) return 1;
  const int64_t fit = ws_bytes / (M * N * 4);
  if (want > fit) want = fit;
  if (want > nk / 2) want = nk / 2;
  if (want <= 1) return 1;
  const int per = static_cast<int>((linear_ceil(nk, want) + 1) / 2 * 2);
  *steps = per;
  return static_cast<int>(linear_ceil(nk, per));
}

// The form and the splits of K for a shape; param_bytes: an element of gamma and beta (0: the plain Linear).
//
// 128 x 256 tiles when there are at least two per CU, else 128 x 128, whole or split for one workgroup per CU
// (two measured slower: M = 1024, K = 3584, N = 512 took 28.0 against 18.7 us, the partials' HBM traffic
// outweighing the extra parallelism); or the band form, whole or split for at most one workgroup per CU:
// whichever has the lowest estimated time. The estimates: rounds of one workgroup per CU, each of a
// fixed and a per-step time (us; the band form's steps slow down by kFull as the chip fills, with x, the
// weight and the products each at a limit), the second launch of a split with its partial products, and the
// band form's stores of rows that are no multiple of 4 columns. Fitted to 2,000 shapes (K = 256 to 7168,
// M = 512 to 65,536, N = 64 to 1024); the choice is on average 1% off the better form's time. What decides,
// in measured us of the tiles | the band form whole | split:
//   enough rows           M = 30000, K = 3584, N = 256 / 384 / 512: 106 / 156 / 212 | 68 / 93 / 109
//                         M = 30000, K = 896, N = 256 / 384 / 512: 37 / 55 / 72 | 24 / 32 / 39
//   columns               M = 16384, K = 3584, N = 128: 50 (36 split) | 55 | 41: the band multiplies 256
//   partials of short K   M = 16384, K = 896, N = 512: 36 | 30 | 47
//   few bands, no split   M = 8192, K = 7168, N = 512, plain: 75 | 146; M = 8192, K = 3584, N = 384: 53 | 67 | 43
inline LinearPlan linear_choose(int64_t M, int32_t N, int32_t K, int param_bytes, int64_t ws_bytes) {
  const int nk = K / kLinearStep;
  constexpr int64_t kBytes = int64_t{1} << 31;
  if (K % (2 * kLinearStep) != 0 || M >= kBytes || (M + 128) * K * 2 >= kBytes || static_cast<int64_t>(N) * K * 2 >= kBytes)
    return {kLinearGeneral, 1, nk};
  struct Cost {
    double fixed, step;
  };
  const bool ln = param_bytes != 0;
  const Cost tile128 = ln ? Cost{4.4, 0.75} : Cost{3.2, 0.51};
  const Cost tile256 = ln ? Cost{9.4, 1.2} : Cost{9.1, 1.0};
  const Cost bands[3] = {ln ? Cost{4.3, 0.78} : Cost{3.6, 0.62}, ln ? Cost{6.6, 0.98} : Cost{6.0, 0.83},
                         ln ? Cost{9.2, 1.18} : Cost{9.2, 1.14}};
  constexpr double kLaunch = 3.0, kFull = 0.55, kReduce = 2.3, kPartial = 1.1e-6;
  const double odd_store = N % 2 ? (ln ? 0.6e-6 : 0.9e-6) : (N % 4 ? 0.15e-6 : 0.0);  // per element stored
  const double mn = static_cast<double>(M) * N;
  const auto split_time = [&](int splits) { return splits > 1 ? kReduce + kPartial * mn * splits : 0.0; };

  LinearPlan tiles{kLinearTile256, 1, nk};
  double tile_time;
  const int64_t t256 = linear_ceil(M, 128) * linear_ceil(N, 256);
  if (t256 >= 2 * kLinearCus) {
    tile_time = kLaunch + linear_ceil(t256, kLinearCus) * (tile256.fixed + tile256.step * nk);
  } else {
    const int64_t t128 = linear_ceil(M, 128) * linear_ceil(N, 128);
    const auto time128 = [&](int splits, int steps) {
      // plain tiles fit a CU twice: a half-filled round takes little more than half the time
      const double rounds = ln ? linear_ceil(t128 * splits, kLinearCus)
                               : t128 * splits <= kLinearCus ? 1.0 : 0.1 + 0.5 * linear_ceil(2 * t128 * splits, kLinearCus);
      return kLaunch + split_time(splits) + rounds * (tile128.fixed + tile128.step * steps);
    };
    tiles.form = kLinearTile128;
    tile_time = time128(1, nk);
    int steps = 0;
    const int splits = linear_split(linear_ceil(kLinearCus, t128), M, N, K, ws_bytes, &steps);
    if (splits > 1 && time128(splits, steps) < tile_time) {
      tiles = {kLinearTile128, splits, steps};
      tile_time = time128(splits, steps);
    }
  }
  if (static_cast<int64_t>(K) * 2 * param_bytes > kLinearBandParams) return tiles;

  const Cost band = bands[linear_band_fragments(N) - 2];
  const int64_t t_band = linear_band_tiles(M, N);
  const auto band_time = [&](int splits, int steps) {
    const int64_t full = t_band * splits / kLinearCus, last = t_band * splits % kLinearCus;
    const double filled = last > kLinearCus / 2 ? 2.0 * last / kLinearCus - 1.0 : 0.0;
    return kLaunch + split_time(splits) + odd_store * mn * splits +
           full * (band.fixed + band.step * steps * (1.0 + kFull)) +
           (last ? band.fixed + band.step * steps * (1.0 + kFull * filled) : 0.0);
  };
  if (band_time(1, nk) < (ln ? 0.97 : 0.93) * tile_time) {
    tiles = {kLinearBand, 1, nk};
    tile_time = band_time(1, nk);
  }
  int steps = 0;
  const int splits = linear_split(kLinearCus / t_band, M, N, K, ws_bytes, &steps);
  if (splits > 1 && band_time(splits, steps) < (ln ? 0.97 : 0.88) * tile_time) return {kLinearBand, splits, steps};
  return tiles;
}

// Bytes of workspace that a shape is given at most, whatever gamma and beta are: what the splits of the
// fastest choice need (0: it is whole).
inline int64_t linear_workspace_bytes(int64_t M, int32_t N, int32_t K) {
  int splits = 1;
  for (int param_bytes : {0, 2, 4}) {
    const LinearPlan plan = linear_choose(M, N, K, param_bytes, INT64_MAX);
    if (plan.splits > splits) splits = plan.splits;
  }
  return splits > 1 ? static_cast<int64_t>(splits) * M * N * 4 : 0;
}

inline LinearPlan linear_plan(int64_t M, int32_t N, int32_t K, int param_bytes, int64_t ws_bytes) {
  const int64_t most = ws_bytes > 0 ? linear_workspace_bytes(M, N, K) : 0;
  return linear_choose(M, N, K, param_bytes, ws_bytes < most ? ws_bytes : most);
}

// ---------------------------------------------------------------------------------------------
// int8 Linear: t [M, N or 2 N] = q [M, K] w^T in int32, K in steps of kLinear8Step bytes.
// ---------------------------------------------------------------------------------------------
constexpr int kLinear8Step = 128;
// |t| <= K * 2^14 (both operands -128 throughout) stays below 2^31
constexpr int kLinear8MaxK = 131071;
constexpr int kLinear8MaxN = 1 << 30;  // 2 N is an int32 too

enum Linear8Form {
  kLinear8Rows,  // 16 rows x 16 outputs, operands straight to registers, K over the wavefronts of a workgroup
  kLinear8Any,   // 128 x 128 tiles of operands at any address, any K
  // K a multiple of 16, 16-byte aligned operands, loaded straight to LDS:
  kLinear8Ring,     // 64 x 64 tiles, a ring of four steps, two to a CU
  kLinear8Tile128,  // 128 x 128 tiles, two steps, two to a CU
  kLinear8Tile256,  // 256 x 256 tiles, two steps, one to a CU
  // rings of four steps, one tile to a CU, when there are about as many tiles as CUs:
  kLinear8RingTall,  // 128 x 64 tiles
  kLinear8Ring128,   // 128 x 128 tiles
  kLinear8Forms,
};
// One launch (two with splits): columns n_begin .. n_end of y.
struct Linear8Part {
  Linear8Form form;
  int splits;  // of K: 1, or as many int32 partial sums as the workspace then has to hold
  int steps;   // per split
  int32_t n_begin, n_end;
};
struct Linear8Plan {
  int parts;
  Linear8Part part[2];
  bool padded;  // operands are copied to rows of whole steps first
};
struct Linear8Tile {
  int rows, cols;  // weight rows (gated: as many gates as values); of the rows forms outputs
};

inline Linear8Tile linear8_tile(Linear8Form form) {
  switch (form) {
    case kLinear8Rows: return {16, 16};
    case kLinear8Ring: return {64, 64};
    case kLinear8RingTall: return {128, 64};
    case kLinear8Tile256: return {256, 256};
    default: return {128, 128};
  }
}

// Bytes of the copies of padded operands, and of a plan's workspace.
inline int64_t linear8_pad_bytes(int64_t M, int32_t N, int32_t K, bool gated) {
  return (M + static_cast<int64_t>(N) * (gated ? 2 : 1)) * linear_ceil(K, kLinear8Step) * kLinear8Step;
}
// (partial sums: rows of whole 16-byte vectors)
constexpr int64_t linear8_part_cols(int64_t cols) { return linear_ceil(cols, 4) * 4; }
inline int64_t linear8_part_bytes(const Linear8Part& part, int64_t M, bool gated) {
  return part.splits > 1 ? part.splits * M * linear8_part_cols(part.n_end - part.n_begin) * (gated ? 8 : 4) : 0;
}
inline int64_t linear8_plan_bytes(const Linear8Plan& plan, int64_t M, int32_t N, int32_t K, bool gated) {
  int64_t most = 0;  // the parts run one after the other
  for (int i = 0; i < plan.parts; ++i) {
    const int64_t b = linear8_part_bytes(plan.part[i], M, gated);
    if (b > most) most = b;
  }
  return most + (plan.padded ? linear8_pad_bytes(M, N, K, gated) : 0);
}

// Tiles of `cols` columns of y.
inline int64_t linear8_tiles(Linear8Form form, int64_t M, int64_t cols, bool gated) {
  const Linear8Tile tile = linear8_tile(form);
  return linear_ceil(M, tile.rows) * linear_ceil(cols, gated && form != kLinear8Rows ? tile.cols / 2 : tile.cols);
}
// The most workgroups of a plan's launches (of one split).
inline int64_t linear8_workgroups(const Linear8Plan& plan, int64_t M, bool gated) {
  int64_t most = 0;
  for (int i = 0; i < plan.parts; ++i) {
    const int64_t t = linear8_tiles(plan.part[i].form, M, plan.part[i].n_end - plan.part[i].n_begin, gated);
    if (t > most) most = t;
  }
  return most;
}

// A launch has fewer than 2^32 threads: the most workgroups of one, by their threads (those of the rows form go by the
// steps of K that it has, see linear8_rows_waves).
constexpr int linear8_rows_waves(int steps) { return steps <= 16 ? 4 : steps <= 32 ? 8 : 16; }
inline int64_t linear8_max_tiles(Linear8Form form, int steps) {
  const int waves = form == kLinear8Rows ? linear8_rows_waves(steps) : form == kLinear8Any || form == kLinear8Ring ? 4 : 8;
  return UINT32_MAX / (waves * 64);
}
// Outputs that are taken, whatever the operands' addresses and the workspace: so many that a row of 256 x 256 tiles has no
// more workgroups than a launch of 1,024 threads each.
inline int64_t linear8_max_out(bool gated) { return static_cast<int64_t>(UINT32_MAX / 1024) * (gated ? 128 : 256); }
// Rows of x in a launch, more take several: so the copy of operands of odd widths stays small beside what they were made
// from (a launch of 2^20 rows leaves at most 1 round of tiles in 16 unfilled), and for outputs past 2^18 (gated 2^17) the
// form that takes every operand has a launch (of 128 rows it has one for every number of outputs that is taken).
constexpr int64_t kLinear8LaunchRows = int64_t{1} << 20;
inline int64_t linear8_launch_rows(int32_t N, bool gated) {
  int64_t rows = kLinear8LaunchRows;
  while (linear8_tiles(kLinear8Any, rows, N, gated) > linear8_max_tiles(kLinear8Any, 0)) rows /= 2;
  return rows;
}

// The estimated time (us) of one part. Workgroups run `slots` at a time (what fits the CUs); a round takes a fixed
// time and a time per step, which grows from `step` to `full` as the round fills the chip. What the operands, the
// output (more where rows of y are not whole 16-byte stores) and the partial sums of a split take beyond that is
// added per million bytes or elements. Fitted to 84,000 timings of 10,600 random shapes (64 to 16,384 rows and outputs, K
// from 64 to 16,384, plain and gated), the first two forms to 61,000 of 9,000 from one row and one output on; the plan chosen
// is on average 1.1% off the best of all forms and splits (4% for rows of odd widths). Measured, in us, rows | ring |
// tall ring | 128 ring | 128 tiles | 256 tiles:
//   16 x 4096 -> 4096: 7.0 | 11.2 | - | - | - | -              64 x 4096 -> 4096: 18.5 | 12.5 | - | - | - | -
//   300 x 3584 -> 512: - | 8.3 | 9.3 | - | - | -               4096 x 3584 -> 512: - | 15.2 | 12.7 | 16.0 | 21.6 | 37.3
//   2048 x 2048 -> 2048: - | 17.6 | 14.8 | 13.5 | 13.2 | 24.6  2048 x 5632 -> 2048: - | 45 | 38 | 27 | 36 | 55
//   2048 x 4096 -> 4096: - | 54 | 48 | 37.7 | 34.4 | 43.6      8192 x 8192 -> 4096: - | 393 | - | - | 268 | 195
inline double linear8_time(const Linear8Part& part, int64_t M, int32_t K, bool gated) {
  struct Cost {
    double launch, fixed, step, full, bytes, split, sums, out, out_odd;
    int slots;
  };
  const int64_t cols = part.n_end - part.n_begin, wrows = cols * (gated ? 2 : 1);
  const auto cost = [&]() -> Cost {
    switch (part.form) {
      case kLinear8Rows: return {2.56, 0.0, 0.108, 0.275, 0.0, 2.35, 1.05, 0.38, 0.26, 512};
      case kLinear8Any: return {3.54, 2.97, 1.052, 1.566, 0.078, 0.31, 1.97, 1.06, 0.0, 512};
      case kLinear8Ring: return {1.38, 2.11, 0.156, 0.408, 0.034, 1.97, 2.48, 0.04, 0.25, 512};
      case kLinear8Tile128: return {0.96, 2.91, 0.540, 0.987, 0.032, 1.99, 1.96, 0.27, 0.36, 512};
      case kLinear8RingTall: return {1.49, 2.21, 0.221, 0.322, 0.042, 2.36, 1.82, 0.0, 0.35, 256};
      case kLinear8Ring128: return {1.65, 3.16, 0.307, 0.496, 0.027, 2.30, 1.59, 0.0, 0.37, 256};
      default: return {2.70, 6.86, 0.984, 1.617, 0.0, 3.21, 1.02, 0.04, 0.44, 256};
    }
  }();
  double slow = 1.0;
  if (part.form == kLinear8Rows) {
    if (gated) slow *= 1.78;
    if (K % 4 != 0) slow *= 2.33;  // loads at odd addresses (at multiples of 4 they cost nothing)
  }
  const int64_t groups = linear8_tiles(part.form, M, cols, gated) * part.splits;
  const int64_t rounds = groups / cost.slots;
  const double filled = static_cast<double>(groups % cost.slots) / cost.slots;
  const double mn = 1e-6 * M * cols;
  double t = cost.launch + rounds * (cost.fixed + cost.full * slow * part.steps);
  if (filled > 0) t += cost.fixed + (cost.step + (cost.full - cost.step) * filled) * slow * part.steps;
  if (part.splits > 1) t += cost.split + cost.sums * 1e-6 * M * wrows * part.splits;
  return t + cost.bytes * 1e-6 * (wrows + M) * K + (cols % 8 == 0 ? cost.out : cost.out + cost.out_odd) * mn;
}

// What the host needs for a call, and for each launch beyond the first: a plan that is faster than that on the GPU
// gains nothing where calls follow each other (where a graph is replayed it would: 1 x 9856 -> 80 by the plan of fewest launches
// is estimated at 11.0 us, 5.4 by the fastest).
constexpr double kLinear8Host = 7.5, kLinear8HostLaunch = 3.5;

// The best single part for columns n_begin .. n_end: its form and splits (at most as many as ws_bytes hold partial
// sums of), and its estimated time.
inline Linear8Part linear8_best(int64_t M, int32_t n_begin, int32_t n_end, int32_t K, bool gated, bool aligned,
                                int64_t ws_bytes, double* time) {
  const int nk = static_cast<int>(linear_ceil(K, kLinear8Step));
  Linear8Part best{kLinear8Any, 1, nk, n_begin, n_end};
  double best_cost = -1.0;
  for (int f = kLinear8Rows; f < kLinear8Forms; ++f) {
    const Linear8Form form = static_cast<Linear8Form>(f);
    if (form != kLinear8Rows && form != kLinear8Any && !aligned) continue;
    const int64_t tiles = linear8_tiles(form, M, n_end - n_begin, gated);
    if (tiles > linear8_max_tiles(form, nk)) continue;  // (never the form for any operand: linear8_launch_rows)
    for (int want = 1; want <= 32; want *= 2) {
      Linear8Part part{form, 1, nk, n_begin, n_end};
      if (want > 1) {
        if (want > nk / 2 || tiles * want > 1024) break;
        part.steps = static_cast<int>(linear_ceil(nk, want));
        part.splits = static_cast<int>(linear_ceil(nk, part.steps));
        if (linear8_part_bytes(part, M, gated) > ws_bytes) break;
      }
      const double t = linear8_time(part, M, K, gated);
      const double host = kLinear8Host + (part.splits > 1 ? kLinear8HostLaunch : 0.0);
      const double cost = t > host ? t : host + 1e-3 * t;  // level with the host: the fewest launches, then the GPU's time
      if (best_cost < 0 || cost < best_cost) {
        best_cost = cost;
        best = part;
        *time = t;
      }
    }
  }
  return best;
}

inline Linear8Plan linear8_plan(int64_t M, int32_t N, int32_t K, bool gated, bool aligned, int64_t ws_bytes) {
  Linear8Plan plan{1, {}, false};
  double time = 0;
  plan.part[0] = linear8_best(M, 0, N, K, gated, aligned, ws_bytes, &time);
  // Operands of odd widths (or addresses) copied to rows of whole steps first (us, not copied | copied): 1531 x 1021 ->
  // 777: 17.7 | 10.9; 2000 x 4094 -> 4096: 57.7 | 52.7; 500 x 8191 -> 2000: 88.9 | 29.1.
  const int64_t pad = linear8_pad_bytes(M, N, K, gated);
  if (!aligned && ws_bytes >= pad && pad / 16 < UINT32_MAX - 1024) {  // (a thread copies 16 bytes)
    const int32_t to = static_cast<int32_t>(linear_ceil(K, kLinear8Step) * kLinear8Step);
    double t = 0;
    const Linear8Part part = linear8_best(M, 0, N, to, gated, true, ws_bytes - pad, &t);
    t += 2.5 + 0.37e-6 * pad;
    const auto cost = [](double t, int launches) {
      const double host = kLinear8Host + kLinear8HostLaunch * (launches - 1);
      return t > host ? t : host + 1e-3 * t;
    };
    if (cost(t, part.splits > 1 ? 3 : 2) < cost(time, plan.part[0].splits > 1 ? 2 : 1)) {
      plan.part[0] = part;
      plan.padded = aligned = true;
      time = t;
      K = to;
      ws_bytes -= pad;
    }
  }
  // Rounds of 256 x 256 tiles that fill the chip, and the columns left over in a form of their own: 8192 x 8192 -> 4352:
  // 17 columns of 32 tiles are two rounds and a rest of 32.
  if (aligned) {
    const int64_t rows = linear_ceil(M, 256), wide = gated ? 128 : 256, tiles = rows * linear_ceil(N, wide);
    const int64_t whole = tiles / kLinearCus * kLinearCus / rows * wide;  // columns of the whole rounds
    if (tiles > kLinearCus && whole > 0 && whole < N && rows * (whole / wide) <= linear8_max_tiles(kLinear8Tile256, 0)) {
      const int nk = static_cast<int>(linear_ceil(K, kLinear8Step));
      const Linear8Part first{kLinear8Tile256, 1, nk, 0, static_cast<int32_t>(whole)};
      double rest = 0;
      const Linear8Part second = linear8_best(M, first.n_end, N, K, gated, true, ws_bytes, &rest);
      if (linear8_time(first, M, K, gated) + rest < 0.95 * time) {
        plan.parts = 2;
        plan.part[0] = first;
        plan.part[1] = second;
      }
    }
  }
  return plan;
}

// Bytes of workspace that a shape's operands, at 16-byte aligned addresses or others, are given at most.
inline int64_t linear8_workspace_bytes(int64_t M, int32_t N, int32_t K, bool gated, bool aligned) {
  const auto of = [&](int64_t rows) {
    return rows > 0 ? linear8_plan_bytes(linear8_plan(rows, N, K, gated, aligned && K % 16 == 0, INT64_MAX), rows, N, K, gated) : 0;
  };
  const int64_t most = linear8_launch_rows(N, gated), rest = of(M % most), whole = M >= most ? of(most) : 0;
  return rest > whole ? rest : whole;
}

// ---------------------------------------------------------------------------------------------
// int8 norms
// ---------------------------------------------------------------------------------------------
// A row in the registers of `waves` wavefronts, `vectors` of 16 bytes (`vec` elements) a lane; waves 0: in a group of lanes
// of one wavefront, a vector each; vectors 0: rows of less than a vector or more than the registers hold, in a loop.
// The time of a row alone counts while rows are few, and a wavefront with 8 vectors per lane leaves too little else on its
// SIMD (16,384 rows of 4,096 bf16 with a residual: 82 us with 4 wavefronts of 2 vectors per lane, 88 with 4 of 4, 101 with
// one of 8; one row: 4.4 us with 8 of 1, 5.2 with 4 of 2, 9.3 with one of 8).
struct Norm8Form {
  int vectors, waves;
};
inline Norm8Form norm8_form(int64_t rows, int64_t cols, int vec) {
  const int64_t n = linear_ceil(cols, vec);  // vectors of a row
  const bool few = rows < 1536;              // too few to fill the card with 8 wavefronts each
  if (cols < vec || n > 4096) return {0, 0};
  if (n <= 32) return {1, 0};
  if (n <= 64) return {1, 1};
  if (n <= 128) return {1, 2};
  if (n <= 256) return {1, 4};
  if (n <= 512) return few ? Norm8Form{1, 8} : Norm8Form{2, 4};
  if (n <= 1024) return {2, 8};
  if (n <= 2048) return few ? Norm8Form{2, 16} : Norm8Form{4, 8};
  return {4, 16};
}

}  // namespace cti
