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
// Bound by memory (each new value is read and stored once) or, for single tokens, by the chain length -> table -> scale ->
// store.  A wavefront of the 16-bit kernel holds 1024 / D rows and walks a run of heads; one of the 8-bit kernel has one
// block of one head, of the keys or of the values, so that the scale is its own.
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
// The last sequence s with key(s) <= x (keys do not fall; -1 if there is none).
template <class Key>
FA_DEVICE int last_not_above(int n, int64_t x, Key key) {
  int lo = -1, hi = n;   // key(lo) <= x < key(hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (key(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
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

template <class T, int D, bool INTER>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) append_kernel(AppendParams p) {
  const int lane = hw::thread_id() & 63;
  const int item = hw::uniform(hw::block_x() * kAppendWaves + (hw::thread_id() >> 6));
  const int chunks = (p.Hkv + p.heads_per_item - 1) / p.heads_per_item;
  const int h0 = item % chunks * p.heads_per_item, h1 = imin(h0 + p.heads_per_item, p.Hkv);
  const int64_t row = (int64_t)(item / chunks) * (1024 / D) + lane / (D / 16);
  if (row >= p.rows) return;
  const int s = p.starts ? last_not_above(p.num_seqs, row, [&](int i) { return (int64_t)p.starts[i]; }) : (int)row;
  if (s < 0 || s >= p.num_seqs) return;
  const NewRows rows = new_rows(p, s);
  const int64_t place = rows.base + row;
  if (row < rows.begin || row >= rows.end || place < 0 || place >= position_limit(p)) return;
  const int64_t blk = block_of_table(p, s, place / p.block_size);
  if (blk < 0 || blk >= p.num_blocks) return;
  const RotaryPlace at = rotary_place<D>(lane, p.rotary);
  Turn tr;
  if (p.rotary > 0) tr = load_turn<INTER>(p.cos, p.sin, p.table_stride, place, p.table_rows, at);
  const int64_t to = blk * p.c_blk + place % p.block_size * p.c_tok;
  const T* k = (const T*)p.side[0].x + row * p.side[0].x_row;
  const T* v = (const T*)p.side[1].x + row * p.side[1].x_row;
  T *kc = (T*)p.side[0].cache + to, *vc = (T*)p.side[1].cache + to;
  for (int h = h0; h < h1; ++h) {
    u32x4 lo = *(const u32x4*)(k + h * p.side[0].x_head + at.lo), hi = *(const u32x4*)(k + h * p.side[0].x_head + at.hi);
    const u32x4 vlo = *(const u32x4*)(v + h * p.side[1].x_head + at.lo), vhi = *(const u32x4*)(v + h * p.side[1].x_head + at.hi);
    if (p.rotary > 0) {
      float x[16];
      unpack8<T>(lo, x);
      unpack8<T>(hi, x + 8);
      turn<INTER, 1>(x, tr, at.turned);
      lo = pack8<T>(x);
      hi = pack8<T>(x + 8);
    }
    *(u32x4*)(kc + h * p.c_head + at.lo) = lo;
    *(u32x4*)(kc + h * p.c_head + at.hi) = hi;
    *(u32x4*)(vc + h * p.c_head + at.lo) = vlo;
    *(u32x4*)(vc + h * p.c_head + at.hi) = vhi;
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

template <class T, int D, bool INTER>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) append_e4m3_kernel(AppendParams p) {
  constexpr int ROWS = 1024 / D;   // rows that a wavefront holds at a time
  const int lane = hw::thread_id() & 63;
  // The four wavefronts of a workgroup share a segment: one block of one sequence.
  const int per_segment = (2 * p.Hkv + kAppendWaves - 1) / kAppendWaves;
  const int segment = hw::block_x() / per_segment;
  const int job = hw::uniform(hw::block_x() % per_segment * kAppendWaves + (hw::thread_id() >> 6));
  if (job >= 2 * p.Hkv) return;
  const int h = job >> 1, side = job & 1;
  // Sequence s has the segments from starts[s] / block + 2 s on: at least as many as the blocks its rows can touch.
  int s = segment, nth = 0;
  if (p.starts) {
    auto first = [&](int i) { return clamp64(p.starts[i], 0, p.rows) / p.block_size + 2 * (int64_t)i; };
    s = hw::uniform(last_not_above(p.num_seqs, segment, first));
    if (s < 0) return;
    nth = (int)(segment - first(s));
  }
  const NewRows rows = new_rows(p, s);
  const int64_t begin = rows.base + rows.begin > 0 ? rows.base + rows.begin : 0;
  const int64_t end = rows.base + rows.end < position_limit(p) ? rows.base + rows.end : position_limit(p);
  const int64_t column = begin / p.block_size + nth, at0 = column * p.block_size;
  const int64_t from = at0 > begin ? at0 : begin, to = at0 + p.block_size < end ? at0 + p.block_size : end;
  if (from >= to) return;
  const int64_t blk = block_of_table(p, s, column);
  if (blk < 0 || blk >= p.num_blocks) return;
  const int slot0 = (int)(from - at0), count = (int)(to - from);

  const AppendSide& sd = p.side[side];
  const bool turns = side == 0 && p.rotary > 0;
  const RotaryPlace at = rotary_place<D>(lane, turns ? p.rotary : 0);
  const int r0 = lane / (D / 16);
  const T* x = (const T*)sd.x + (from - rows.base) * sd.x_row + h * sd.x_head;   // row of position `from`
  uint8_t* cache = (uint8_t*)sd.cache + blk * p.c_blk + h * p.c_head;
  float* scale = sd.scale + blk * p.s_blk + h * p.s_head;

  auto load = [&](int r, float* v) {
    unpack8<T>(*(const u32x4*)(x + r * sd.x_row + at.lo), v);
    unpack8<T>(*(const u32x4*)(x + r * sd.x_row + at.hi), v + 8);
    if (turns) turn<INTER, 1>(v, load_turn<INTER>(p.cos, p.sin, p.table_stride, from + r, p.table_rows, at), at.turned);
  };
  const float before = *scale;   // requested in front of everything that takes time, and of the exchanges that join the lanes
  float peak = 0.f;
  for (int r = r0; r < count; r += ROWS) {
    float v[16];
    load(r, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) peak = fmaxf(peak, finite_magnitude(v[i]));
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) peak = fmaxf(peak, hw::shfl_xor(peak, m));
  float now = scale_for_peak(peak);
  if (slot0 > 0) {
    if (now > before) {
      const float shrink = before / now;
      for (int r = r0; r < slot0; r += ROWS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          hw::u32x2* codes = (hw::u32x2*)(cache + r * p.c_tok + (i ? at.hi : at.lo));
          hw::u32x2 c = *codes;
          c[0] = hw::to_e4m3(hw::from_e4m3(c[0]) * shrink);
          c[1] = hw::to_e4m3(hw::from_e4m3(c[1]) * shrink);
          *codes = c;
        }
      }
    } else {
      now = before;
    }
  }
  const float inverse = 1.f / now;
  for (int r = r0; r < count; r += ROWS) {
    float v[16];
    load(r, v);
    uint8_t* row = cache + (slot0 + r) * p.c_tok;
    *(hw::u32x2*)(row + at.lo) = codes8(v, inverse);
    *(hw::u32x2*)(row + at.hi) = codes8(v + 8, inverse);
  }
  if (lane == 0) *scale = now;
}

template <class T, int D, bool INTER>
static int launch_append_d(AppendParams p, hipStream_t stream) {
  if (p.side[0].scale) {
    const int per_segment = (2 * p.Hkv + kAppendWaves - 1) / kAppendWaves;
    const unsigned wgs = workgroups({p.starts ? p.rows / p.block_size + 2 * (int64_t)p.num_seqs : p.num_seqs, per_segment});
    return wgs ? launch(append_e4m3_kernel<T, D, INTER>, dim3(wgs), 0, stream, p) : kBadArgument;
  }
  const int64_t groups = (p.rows + 1024 / D - 1) / (1024 / D), waves = 32 * (int64_t)num_cus_of_current_device();
  const int64_t n = waves > 0 ? groups * p.Hkv / waves : 1;   // heads per item: as many as leave each SIMD eight wavefronts
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
