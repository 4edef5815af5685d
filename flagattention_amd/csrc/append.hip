// Appending keys and values to a paged cache, the keys' rotation on the way.
//
// Row j of sequence s (rows starts[s] .. starts[s + 1] - 1 of key and value; row s where there are no starts) is stored at
// position context_lens[s] - (starts[s + 1] - j) of the sequence: the lengths count the new tokens, as attention over the
// cache needs them right after.  Rows of negative position, behind the last sequence, behind the block table or the
// rotation's tables, or whose block is not one of the cache, are not stored.
//
// A 16-bit cache takes the values rounded once.  An 8-bit cache holds e4m3 codes and an fp32 scale for each block and kv
// head; a code c stands for c * scale.  With `peak` the largest finite magnitude that a call brings into a block,
//   needed = the least power of two with peak / needed <= 448, within 2^-118 .. 2^120
//   scale  = needed where the block was empty, else max(scale, needed)
// and where that grows, the codes that are there are rounded again.  A power of two makes this second rounding exact but for
// numbers that fall below e4m3's normal range, and costs no precision: the codes are floating-point numbers.
//
// Bound by memory (each new value is read and stored once: 16384 rows of 8 heads of 128 to 8 bits 27 us, 109 MB, 4.0 TB/s,
// 8755 of 32 heads of 64 to 16 bits 32 us, 145 MB, 4.5 TB/s) or, for single tokens, by the chain length -> table -> scale ->
// store (4 to 5 us).  A wavefront of the 16-bit kernel holds 1024 / D rows and walks a run of heads; a wavefront or a workgroup of
// the 8-bit kernel has one block of one head, so that the scales are its own.
#include "rotary.hpp"

namespace fa {

constexpr int kAppendWaves = kThreads / 64;

FA_DEVICE int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// The rows of a sequence that exist, and the position that row 0 would have.
struct NewRows { int64_t begin, end, base; };
FA_DEVICE NewRows new_rows(const AppendParams& p, int s) {
  const int64_t ctx = p.lens[s];
  if (!p.starts) return NewRows{s, s + 1, ctx - (s + 1)};
  const int64_t next = p.starts[s + 1], b = clamp64(p.starts[s], 0, p.rows);
  return NewRows{b, clamp64(next, b, p.rows), ctx - next};
}
// The last of n sequences with key(s) <= x (keys do not fall; -1 if there is none), found by the wavefront together: 64 at a
// time, so that up to 64 sequences take one load's latency, up to 4160 two.
template <class Key>
FA_DEVICE int last_not_above(int n, int64_t x, int lane, Key key) {
  int base = 0, found = -1;
  while (base < n) {
    const int step = (n - base + 63) / 64, i = base + lane * step;
    const int count = __builtin_popcountll(hw::ballot(i < n && key(imin(i, n - 1)) <= x));
    if (count == 0) break;
    found = base + (count - 1) * step;
    n = imin(n, found + step);
    base = found + 1;
  }
  return hw::uniform(found);
}
// positions that have a place
FA_DEVICE int64_t position_limit(const AppendParams& p) {
  const int64_t places = (int64_t)p.bt_cols * p.block_size;
  return p.rotary > 0 && p.table_rows < places ? p.table_rows : places;
}
FA_DEVICE int64_t block_of_table(const AppendParams& p, int s, int64_t column) {
  const int64_t at = s * p.bt_stride + column;
  return p.bt64 ? ((const int64_t*)p.block_tables)[at] : ((const int32_t*)p.block_tables)[at];
}

template <class T>
FA_DEVICE void store_raw(T* row, RotaryPlace at, const RawRow& r) {
  *(u32x4*)(row + at.lo) = r.lo;
  *(u32x4*)(row + at.hi) = r.hi;
}

template <class T, int D, bool INTER>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) append_kernel(AppendParams p) {
  const int lane = hw::thread_id() & 63;
  const int item = hw::uniform(hw::block_x() * kAppendWaves + (hw::thread_id() >> 6));
  const int chunks = (p.Hkv + p.heads_per_item - 1) / p.heads_per_item;
  const int h0 = item % chunks * p.heads_per_item, h1 = imin(h0 + p.heads_per_item, p.Hkv);
  const int64_t row0 = (int64_t)(item / chunks) * (1024 / D), row = row0 + lane / (D / 16);
  int s = (int)row;
  if (p.starts) {   // the first row's sequence, and from there to the lane's own in growing and then in shrinking steps
    s = last_not_above(p.num_seqs, row0, lane, [&](int i) { return (int64_t)p.starts[i]; });
    if (s < 0) s = 0;
    int step = 1;
    auto reaches = [&]() { return step < p.num_seqs - s && p.starts[s + step] <= row; };
    for (; reaches(); step *= 2) s += step;
    for (step /= 2; step > 0; step /= 2)
      if (reaches()) s += step;
  }
  if (row >= p.rows || s >= p.num_seqs) return;
  const NewRows rows = new_rows(p, s);
  const int64_t place = rows.base + row;
  if (row < rows.begin || row >= rows.end || place < 0 || place >= position_limit(p)) return;
  const RotaryPlace k_at = rotary_place<D>(lane, p.rotary), v_at = rotary_place<D>(lane, 0);
  const T* k = (const T*)p.side[0].x + row * p.side[0].x_row;
  const T* v = (const T*)p.side[1].x + row * p.side[1].x_row;
  // the first rows and the angles come while the block is looked up
  RawRow next_k = load_row<T, D, true>(k + h0 * p.side[0].x_head, k_at), next_v = load_row<T, D, true>(v + h0 * p.side[1].x_head, v_at);
  Turn tr;
  if (p.rotary > 0) tr = load_turn<INTER>(p.cos, p.sin, p.table_stride, place, p.table_rows, k_at);
  const int64_t blk = block_of_table(p, s, place / p.block_size);
  if (blk < 0 || blk >= p.num_blocks) return;
  const int64_t to = blk * p.c_blk + place % p.block_size * p.c_tok;
  T *kc = (T*)p.side[0].cache + to, *vc = (T*)p.side[1].cache + to;
  for (int h = h0; h < h1; ++h) {
    RawRow row_k = next_k;
    const RawRow row_v = next_v;
    if (h + 1 < h1) {
      next_k = load_row<T, D, true>(k + (h + 1) * p.side[0].x_head, k_at);
      next_v = load_row<T, D, true>(v + (h + 1) * p.side[1].x_head, v_at);
    }
    if (p.rotary > 0) {
      float x[16];
      unpack_row<T>(row_k, x);
      turn<INTER, 1>(x, tr, k_at.turned);
      row_k = RawRow{pack8<T>(x), pack8<T>(x + 8)};
    }
    store_raw(kc + h * p.c_head, k_at, row_k);
    store_raw(vc + h * p.c_head, v_at, row_v);
  }
}

FA_DEVICE float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;   // NaN and infinities do not set the scale
}
// The least power of two s with peak / s <= 448 = 1.75 * 2^8, within 2^-118 .. 2^120: the exponent of peak rounded up where
// its mantissa is above 1.75.
FA_DEVICE float scale_for_peak(float peak) {
  const int e = (int)((__builtin_bit_cast(uint32_t, peak) + 0x1fffffu) >> 23) - 8;
  return __builtin_bit_cast(float, (uint32_t)imin(imax(e, 127 - 118), 127 + 120) << 23);
}
// Eight values as codes of the given scale's inverse: what is not finite has no code but NaN.
FA_DEVICE hw::u32x2 codes8(const float* x, float inverse) {
  hw::u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    hw::f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = x[4 * i + e];
      y[e] = fabsf(v) < __builtin_inff() ? v * inverse : __builtin_nanf("");
    }
    r[i] = hw::to_e4m3(y);
  }
  return r;
}

// SHARED: a workgroup has one block of one head, two wavefronts the keys and two the values, 1024 / D rows in turn.
// Otherwise a wavefront has one block of one head, keys and values one after the other, and a workgroup four heads.
template <class T, int D, bool INTER, bool SHARED>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) append_e4m3_kernel(AppendParams p) {
  FA_LDS_DECL(smem);
  constexpr int ROWS = 1024 / D, TURN = SHARED ? 2 * ROWS : ROWS, SIDES = SHARED ? 1 : 2;   // rows held at a time; sides
  const int lane = hw::thread_id() & 63, wave = hw::uniform(hw::thread_id() >> 6);
  const int per_segment = SHARED ? p.Hkv : (p.Hkv + kAppendWaves - 1) / kAppendWaves;
  const int segment = hw::block_x() / per_segment;   // one block of one sequence
  const int h = hw::block_x() % per_segment * (SHARED ? 1 : kAppendWaves) + (SHARED ? 0 : wave);
  if (h >= p.Hkv) return;
  const int side0 = SHARED ? wave & 1 : 0, r0 = (SHARED ? wave >> 1 : 0) * ROWS + lane / (D / 16);
  // Sequence s has the segments from starts[s] / block + 2 s on: at least as many as the blocks its rows can touch.
  int s = segment, nth = 0;
  if (p.starts) {
    auto first = [&](int i) { return clamp64(p.starts[i], 0, p.rows) / p.block_size + 2 * (int64_t)i; };
    s = last_not_above(p.num_seqs, segment, lane, first);
    if (s < 0) return;   // (this return and the next ones: all that share a block of a head together)
    nth = (int)(segment - first(s));
  }
  const NewRows rows = new_rows(p, s);
  const int64_t begin = rows.base + rows.begin > 0 ? rows.base + rows.begin : 0;
  const int64_t end = rows.base + rows.end < position_limit(p) ? rows.base + rows.end : position_limit(p);
  const int64_t column = begin / p.block_size + nth, at0 = column * p.block_size;
  const int64_t from = at0 > begin ? at0 : begin, to = at0 + p.block_size < end ? at0 + p.block_size : end;
  if (from >= to) return;
  const int64_t blk = block_of_table(p, s, column);   // comes along with the rows, which do not need it
  const int slot0 = (int)(from - at0), count = (int)(to - from);

  // Keys (side 0) and values.  The first TURN rows of each stay in registers as they were loaded; what is behind them is
  // read twice, the second time from the caches (twice as many in registers leave fewer wavefronts: 27.1 and not 26.3 us for
  // 16384 rows of 8 heads, D = 128, in blocks of 16).
  const RotaryPlace turned_at = rotary_place<D>(lane, p.rotary), plain_at = rotary_place<D>(lane, 0);
  RawRow kept[SIDES];
  Turn kept_turn;
  float before[SIDES];
  const T* x[SIDES];
#pragma unroll
  for (int i = 0; i < SIDES; ++i) {
    const AppendSide& sd = p.side[side0 + i];
    x[i] = (const T*)sd.x + (from - rows.base) * sd.x_row + h * sd.x_head;   // row of position `from`
    // (past the last row: the last one again, not counted)
    kept[i] = load_row<T, D, true>(x[i] + imin(r0, count - 1) * sd.x_row, side0 + i ? plain_at : turned_at);
  }
  if (p.rotary > 0 && side0 == 0)
    kept_turn = load_turn<INTER>(p.cos, p.sin, p.table_stride, from + imin(r0, count - 1), p.table_rows, turned_at);
  if (blk < 0 || blk >= p.num_blocks) return;
#pragma unroll
  for (int i = 0; i < SIDES; ++i) before[i] = p.side[side0 + i].scale[blk * p.s_blk + h * p.s_head];

#pragma unroll
  for (int i = 0; i < SIDES; ++i) {
    const int side = side0 + i;
    const AppendSide& sd = p.side[side];
    const bool turns = side == 0 && p.rotary > 0;
    const RotaryPlace at = side ? plain_at : turned_at;
    uint8_t* cache = (uint8_t*)sd.cache + blk * p.c_blk + h * p.c_head;
    // each(row, whether it exists, values): all lanes together, those without a row with the last one.  (The rows that are
    // kept stand in front of the loop, not in it: 28.3 and not 31.9 us at the size above.)
    auto for_rows = [&](auto&& each) {
      float v[16];
      unpack_row<T>(kept[i], v);
      if (turns) turn<INTER, 1>(v, kept_turn, at.turned);
      each(r0, r0 < count, v);
      for (int first = TURN; first < count; first += TURN) {
        const int r = imin(first + r0, count - 1);
        Turn t;
        if (turns) t = load_turn<INTER>(p.cos, p.sin, p.table_stride, from + r, p.table_rows, at);
        unpack_row<T>(load_row<T, D, false>(x[i] + r * sd.x_row, at), v);
        if (turns) turn<INTER, 1>(v, t, at.turned);
        each(r, first + r0 < count, v);
      }
    };
    float peak = 0.f;
    for_rows([&](int, bool, const float* v) {
#pragma unroll
      for (int j = 0; j < 16; ++j) peak = fmaxf(peak, finite_magnitude(v[j]));
    });
#pragma unroll
    for (int m = 1; m < 64; m *= 2) peak = fmaxf(peak, hw::shfl_xor(peak, m));
    if (SHARED) {
      // Also where the other wavefront has no rows: its rows below are those that change to the new scale, and the scale
      // is not written before all have read the old one.
      float* peaks = (float*)smem;
      if (lane == 0) peaks[wave] = peak;
      hw::block_sync();
      peak = fmaxf(peaks[side], peaks[side + 2]);
    }
    float now = scale_for_peak(peak);
    if (slot0 > 0) {
      if (now > before[i]) {
        const float shrink = before[i] / now;
        for (int r = r0; r < slot0; r += TURN) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            hw::u32x2* codes = (hw::u32x2*)(cache + r * p.c_tok + (j ? at.hi : at.lo));
            hw::u32x2 c = *codes;
            c[0] = hw::to_e4m3(hw::from_e4m3(c[0]) * shrink);
            c[1] = hw::to_e4m3(hw::from_e4m3(c[1]) * shrink);
            *codes = c;
          }
        }
      } else {
        now = before[i];
      }
    }
    const float inverse = 1.f / now;
    for_rows([&](int r, bool there, const float* v) {
      uint8_t* row = cache + (slot0 + r) * p.c_tok;
      hw::u32x2 lo = codes8(v, inverse), hi = codes8(v + 8, inverse);
      if (D >= 32 && (!turns || p.rotary % 32 == 0)) {
        // The lanes of a pair have sixteen codes side by side in their first halves, and in their second: one takes those,
        // the other these, so that a row is one store.
        const bool odd = lane & 1;
        const hw::u32x2 give = odd ? lo : hi, keep = odd ? hi : lo;
        hw::u32x2 got;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t word = give[j];   // (a cast of the vector's element itself reads element 0)
          got[j] = __builtin_bit_cast(uint32_t, hw::shfl_xor(__builtin_bit_cast(float, word), 1));
        }
        const u32x4 both = odd ? u32x4{got[0], got[1], keep[0], keep[1]} : u32x4{keep[0], keep[1], got[0], got[1]};
        if (there) {
          uint8_t* to_codes = row + (odd ? at.hi - 8 : at.lo);
          if (D >= 64) hw::store_once(to_codes, both);   // whole lines where a block's rows follow each other
          else *(u32x4*)to_codes = both;
        }
      } else if (there) {
        *(hw::u32x2*)(row + at.lo) = lo;
        *(hw::u32x2*)(row + at.hi) = hi;
      }
    });
    if (lane == 0 && wave < (SHARED ? 2 : kAppendWaves)) sd.scale[blk * p.s_blk + h * p.s_head] = now;
  }
}

template <class T, int D, bool INTER>
static int launch_append_d(AppendParams p, hipStream_t stream) {
  if (p.side[0].scale) {
    const int64_t segments = p.starts ? p.rows / p.block_size + 2 * (int64_t)p.num_seqs : p.num_seqs;
    // A wavefront walks the rows of its block 1024 / D at a time, and twice: a long chain where a block has many, and exposed
    // where few blocks have rows.  Four are worth their exchange of peaks and their empty places then (alone / shared, us:
    // 16384 rows of 8 heads, D = 128, blocks of 64: 35.4 / 30.5, of 32: 27.4 / 31.9, of 16: 29.5 / 37.2; 40 rows for each
    // of 205 sequences in blocks of 64: 18.4 / 21.6; D = 256, blocks of 128: 89.5 / 38.4; 960 rows, D = 128, blocks of 16,
    // 736 wavefronts alone: 8.3 / 6.4, twice as many rows 9.7 / 9.2, four times 12.1 / 14.0).
    const int64_t rows = (p.rows + p.num_seqs - 1) / p.num_seqs, per_block = rows < p.block_size ? rows : p.block_size;
    if (per_block >= 8 * (1024 / D) || segments * p.Hkv <= 4 * (int64_t)num_cus_of_current_device()) {
      const unsigned wgs = workgroups({segments, p.Hkv});
      return wgs ? launch(append_e4m3_kernel<T, D, INTER, true>, dim3(wgs), kAppendWaves * sizeof(float), stream, p) : kBadArgument;
    }
    const unsigned wgs = workgroups({segments, (p.Hkv + kAppendWaves - 1) / kAppendWaves});
    return wgs ? launch(append_e4m3_kernel<T, D, INTER, false>, dim3(wgs), 0, stream, p) : kBadArgument;
  }
  const int64_t groups = (p.rows + 1024 / D - 1) / (1024 / D), cus = num_cus_of_current_device();
  // Heads per item: as many as leave each SIMD four wavefronts, eight where rows are narrower than a line (16384 rows of 8
  // heads, D = 128: 27.6 us with four, 29.3 with eight; 8755 of 32, D = 64: 36.8 and 34.1).
  const int64_t waves = (D >= 128 ? 16 : 32) * cus, n = waves > 0 ? groups * p.Hkv / waves : 1;
  p.heads_per_item = (int)(n < 1 ? 1 : n > p.Hkv ? p.Hkv : n);
  const int chunks = (p.Hkv + p.heads_per_item - 1) / p.heads_per_item;
  const unsigned wgs = workgroups({(groups * chunks + kAppendWaves - 1) / kAppendWaves});
  return wgs ? launch(append_kernel<T, D, INTER>, dim3(wgs), 0, stream, p) : kBadArgument;
}

template <class T, bool INTER>
static int launch_append(const AppendParams& p, hipStream_t stream) {
  switch (p.D) {
    case 16: return launch_append_d<T, 16, INTER>(p, stream);
    case 32: return launch_append_d<T, 32, INTER>(p, stream);
    case 64: return launch_append_d<T, 64, INTER>(p, stream);
    case 128: return launch_append_d<T, 128, INTER>(p, stream);
    case 256: return launch_append_d<T, 256, INTER>(p, stream);
    case 512: return launch_append_d<T, 512, INTER>(p, stream);
  }
  return kUnsupported;
}

int run_append(const AppendParams& p, hipStream_t stream) {
  if (p.rows <= 0 || p.num_seqs <= 0 || p.Hkv <= 0 || p.block_size <= 0 || p.num_blocks <= 0 || p.bt_cols <= 0) return kBadArgument;
  if (p.rows > 0x7fffffff || (!p.starts && p.rows != p.num_seqs)) return kBadArgument;
  if (p.rotary < 0 || p.rotary > p.D || p.rotary % 16 || (p.rotary > 0 && p.table_rows <= 0)) return kBadArgument;
  if (p.dtype == kDtypeF16) return p.interleaved ? launch_append<hw::half_t, true>(p, stream) : launch_append<hw::half_t, false>(p, stream);
  if (p.dtype == kDtypeBF16) return p.interleaved ? launch_append<hw::bf16_t, true>(p, stream) : launch_append<hw::bf16_t, false>(p, stream);
  return kUnsupported;
}

}  // namespace fa
