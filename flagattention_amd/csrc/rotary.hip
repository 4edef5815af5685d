// Norm and rotation of queries and keys in one pass, forward and backward.
//
// For a row x of D values (one head of one token), a weight w and a position p:
//   n = x * rsqrt(mean(x^2) + eps) * w                      (without weights n = x)
//   y = n with its first `rotary` values turned in pairs:   (a, b) -> (a cos - b sin, b cos + a sin)
// where the pairs are (i, i + rotary / 2) or, interleaved, (2i, 2i + 1), and cos / sin are row p of the tables.
// The turn is orthogonal, so with g = the turn by the opposite angle of dy, r = rsqrt(..) and h = x r:
//   dw = sum over rows of g h,     dx = r (g w - h mean(g w h)).
//
// Bound by memory: a forward reads and writes each row once, a backward reads x and dy and writes dx (without weights it
// reads dy alone); the tables are read once per token and group of heads, from the caches.  So nothing is staged: a row is
// held by D / 16 lanes, each with eight values of the first half of the turned part and the eight they are paired with (the
// rest of the row is dealt the same way), which makes both kinds of pairs local to a lane and the mean a few lane exchanges.
// A wavefront holds 1024 / D tokens at a time and walks a run of heads with their cosines and sines in registers, the next
// head's row on its way.  8192 tokens, 32 + 8 heads of 128, bf16: forward 31 us (172 MB, 5.5 TB/s; a copy of that size
// reaches 4.8 to 6.9, as much of it as the last-level cache holds), backward with weights 50 + 4 us (252 MB); 64 single
// tokens 4.7 us, latency.
#include "rotary.hpp"

namespace fa {

constexpr int kWaves = kThreads / 64;

// sum over the D / 16 lanes of a row
template <int D>
FA_DEVICE float row_sum(float x) {
#pragma unroll
  for (int m = 1; m < D / 16; m *= 2) x += hw::shfl_xor(x, m);
  return x;
}

template <class T>
FA_DEVICE void load_weight(const void* w, int f32, RotaryPlace at, float* out) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    out[i] = f32 ? ((const float*)w)[at.lo + i] : (float)((const T*)w)[at.lo + i];
    out[8 + i] = f32 ? ((const float*)w)[at.hi + i] : (float)((const T*)w)[at.hi + i];
  }
}

// What a wavefront works on: tokens `tokens_at` + its lane's row, heads h0 .. h1 - 1 of the queries or of the keys.
struct RotaryItem {
  int side, h0, h1;
  int64_t token;   // this lane's
};
template <int D>
FA_DEVICE RotaryItem rotary_item(const RotaryParams& p, int64_t item, int lane) {
  const int chunks = p.side[0].chunks + p.side[1].chunks, c = (int)(item % chunks);
  RotaryItem r;
  r.side = c < p.side[0].chunks ? 0 : 1;
  const RotarySide& s = p.side[r.side];
  r.h0 = (r.side ? c - p.side[0].chunks : c) * p.heads_per_item;
  r.h1 = imin(r.h0 + p.heads_per_item, s.heads);
  r.token = item / chunks * (1024 / D) + lane / (D / 16);
  return r;
}

// A lane's share of a row as it lies in memory.  From head size 128 on, each of its two accesses takes whole 128-byte lines,
// and a row's are requested while the row before it is worked on (narrower rows have one or two heads to an item where it
// matters, and lost 0.8 of 6.9 us to that).  The forward's stores and the backward's loads are marked non-temporal; with the
// loads in place of the stores the forward of 8192 tokens, 32 + 8 heads, D = 128 takes 34.4 us and not 32.0, with neither
// 41.7; the backward takes 58.5 with stores in place of loads, 55.0 so.
template <class T, int D, bool ONCE>
FA_DEVICE void store_row(T* row, RotaryPlace at, const float* x) {
  if constexpr (D >= 128 && ONCE) {
    hw::store_once(row + at.lo, pack8<T>(x));
    hw::store_once(row + at.hi, pack8<T>(x + 8));
  } else {
    *(u32x4*)(row + at.lo) = pack8<T>(x);
    *(u32x4*)(row + at.hi) = pack8<T>(x + 8);
  }
}

FA_DEVICE int64_t rotary_position(const RotaryParams& p, int b, int t) {
  if (!p.positions) return t;
  const int64_t at = b * p.pos_sb + t * p.pos_st;
  return p.pos64 ? ((const int64_t*)p.positions)[at] : ((const int32_t*)p.positions)[at];
}

template <class T, int D, bool NORM, bool INTER>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) rotary_kernel(RotaryParams p) {
  const int lane = hw::thread_id() & 63;
  const int64_t item = hw::uniform((int)((int64_t)hw::block_x() * kWaves + (hw::thread_id() >> 6)));
  const RotaryItem it = rotary_item<D>(p, item, lane);
  const RotarySide& s = p.side[it.side];
  const int64_t tokens = (int64_t)p.B * p.T;
  const bool there = it.token < tokens;   // the lanes of a token that does not exist work on the last one and do not store
  const int64_t n = there ? it.token : tokens - 1;
  const int b = (int)(n / p.T), t = (int)(n % p.T);
  const RotaryPlace at = rotary_place<D>(lane, p.rotary);
  const T* x = (const T*)s.x.ptr + b * s.x.sb + t * s.x.st;
  T* y = (T*)s.y.ptr + b * s.y.sb + t * s.y.st;
  RawRow next = load_row<T, D, false>(x + it.h0 * s.x.sh, at);   // on its way while the position finds its row of the tables
  const Turn tr = load_turn<INTER>(p.cos, p.sin, p.table_stride, rotary_position(p, b, t), p.table_rows, at);
  float w[16];
  if (NORM) load_weight<T>(s.w, p.w_f32, at, w);
  for (int h = it.h0; h < it.h1; ++h) {
    float v[16];
    const RawRow row = D < 128 && h > it.h0 ? load_row<T, D, false>(x + h * s.x.sh, at) : next;
    if (D >= 128 && h + 1 < it.h1) next = load_row<T, D, false>(x + (h + 1) * s.x.sh, at);
    unpack_row<T>(row, v);
    if (NORM) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sq = fmaf(v[i], v[i], sq);
      const float r = hw::rsqrt_fast(row_sum<D>(sq) * (1.f / D) + p.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * r * w[i];
    }
    turn<INTER, 1>(v, tr, at.turned);
    if (there) {
      store_row<T, D, true>(y + h * s.y.sh, at, v);
    }
  }
}

// A workgroup takes items of one side only, so that its share of dw is one row of the workspace: its wavefronts' sums, added
// in LDS.  rotary_weight_grad_kernel adds the workgroups' rows in a fixed order.
template <class T, int D, bool NORM, bool INTER>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) rotary_bwd_kernel(RotaryParams p) {
  FA_LDS_DECL(smem);
  const int tid = hw::thread_id(), lane = tid & 63, wave = hw::uniform(tid >> 6);
  const int side = hw::block_x() < p.side[0].workgroups ? 0 : 1;
  const RotarySide& s = p.side[side];
  const int wg = hw::block_x() - (side ? p.side[0].workgroups : 0);
  const RotaryPlace at = rotary_place<D>(lane, p.rotary);
  float w[16], dw[16];
  if (NORM) load_weight<T>(s.w, p.w_f32, at, w);
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f;
  const int64_t tokens = (int64_t)p.B * p.T, items = (tokens + 1024 / D - 1) / (1024 / D) * s.chunks;
  for (int64_t item = (int64_t)wg * kWaves + wave; item < items; item += (int64_t)s.workgroups * kWaves) {
    const int h0 = (int)(item % s.chunks) * p.heads_per_item, h1 = imin(h0 + p.heads_per_item, s.heads);
    const int64_t token = item / s.chunks * (1024 / D) + lane / (D / 16);
    const bool there = token < tokens;   // as in the forward; and do not count
    const int64_t n = there ? token : tokens - 1;
    const int b = (int)(n / p.T), t = (int)(n % p.T);
    const T* x = NORM ? (const T*)s.x.ptr + b * s.x.sb + t * s.x.st : nullptr;
    const T* dy = (const T*)s.dy.ptr + b * s.dy.sb + t * s.dy.st;
    T* dx = (T*)s.y.ptr + b * s.y.sb + t * s.y.st;
    RawRow next_x, next_dy;
    auto fetch = [&](int h) {
      next_dy = load_row<T, D, true>(dy + h * s.dy.sh, at);
      if (NORM) next_x = load_row<T, D, true>(x + h * s.x.sh, at);
    };
    fetch(h0);
    const Turn tr = load_turn<INTER>(p.cos, p.sin, p.table_stride, rotary_position(p, b, t), p.table_rows, at);
    for (int h = h0; h < h1; ++h) {
      float g[16];
      if (D < 128 && h > h0) fetch(h);
      const RawRow row_dy = next_dy, row_x = next_x;
      if (D >= 128 && h + 1 < h1) fetch(h + 1);
      unpack_row<T>(row_dy, g);
      if (NORM) {
        float v[16];
        unpack_row<T>(row_x, v);
        turn<INTER, -1>(g, tr, at.turned);
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { sq = fmaf(v[i], v[i], sq); dot = fmaf(g[i] * w[i], v[i], dot); }
        sq = row_sum<D>(sq);
        dot = row_sum<D>(dot);
        const float r = hw::rsqrt_fast(sq * (1.f / D) + p.eps), mean = dot * r * (1.f / D);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float hat = v[i] * r;
          if (there) dw[i] = fmaf(g[i], hat, dw[i]);
          g[i] = r * (g[i] * w[i] - hat * mean);
        }
      } else {
        turn<INTER, -1>(g, tr, at.turned);
      }
      if (there) {
        store_row<T, D, false>(dx + h * s.y.sh, at, g);
      }
    }
  }
  if (!NORM) return;
  // lanes of one place in the row, then the four wavefronts
  float* area = (float*)smem;   // [kWaves][D]
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int m = D / 16; m < 64; m *= 2) dw[i] += hw::shfl_xor(dw[i], m);
    if (lane < D / 16) area[wave * D + (i < 8 ? at.lo + i : at.hi + i - 8)] = dw[i];
  }
  hw::block_sync();
  for (int d = tid; d < D; d += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) sum += area[u * D + d];
    p.partial[(int64_t)hw::block_x() * D + d] = sum;
  }
}

// dw[d .. d + 3] = sum over the side's workgroups of their rows: one workgroup per four columns and side.
template <class T>
FA_KERNEL void FA_LAUNCH_BOUNDS(kThreads) rotary_weight_grad_kernel(RotaryParams p) {
  FA_LDS_DECL(smem);
  const int tid = hw::thread_id(), side = hw::block_y(), d = 4 * hw::block_x();
  const RotarySide& s = p.side[side];
  const float* rows = p.partial + (int64_t)(side ? p.side[0].workgroups : 0) * p.D + d;
  hw::f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = tid; i < s.workgroups; i += kThreads) sum += *(const hw::f32x4*)(rows + (int64_t)i * p.D);
#pragma unroll
  for (int m = 1; m < 64; m *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += hw::shfl_xor(sum[e], m);
  float* area = (float*)smem;
  if ((tid & 63) == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) area[4 * (tid >> 6) + e] = sum[e];
  hw::block_sync();
  if (tid < 4) {
    float total = 0.f;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) total += area[4 * u + tid];
    if (p.w_f32) ((float*)s.dw)[d + tid] = total;
    else ((T*)s.dw)[d + tid] = (T)total;
  }
}

// Heads per item: as many as leave each SIMD about four wavefronts (what is loaded once per token is then shared most), all
// of them at most.
static void plan_rotary(RotaryParams& p) {
  const int64_t groups = ((int64_t)p.B * p.T + 1024 / p.D - 1) / (1024 / p.D);
  const int64_t waves = 16 * (int64_t)num_cus_of_current_device();
  const int most = p.side[0].heads > p.side[1].heads ? p.side[0].heads : p.side[1].heads;
  const int64_t heads = p.side[0].heads + p.side[1].heads;
  int64_t n = waves > 0 ? groups * heads / waves : 1;
  p.heads_per_item = (int)(n < 1 ? 1 : n > most ? most : n);
  for (RotarySide& s : p.side) s.chunks = (s.heads + p.heads_per_item - 1) / p.heads_per_item;
}

static int64_t rotary_items(const RotaryParams& p, int chunks) {
  return ((int64_t)p.B * p.T + 1024 / p.D - 1) / (1024 / p.D) * chunks;
}

static bool rotary_args_ok(const RotaryParams& p) {
  if (p.B <= 0 || p.T <= 0 || p.side[0].heads <= 0 || p.side[1].heads <= 0) return false;
  if ((int64_t)p.B * p.T > 0x7fffffff || (int64_t)p.B * p.T * (p.side[0].heads + (int64_t)p.side[1].heads) / (1024 / p.D) > 0x7fffffff) return false;
  return p.rotary >= 16 && p.rotary <= p.D && p.rotary % 16 == 0 && p.eps > 0.f && p.table_rows > 0;
}

// Workgroups of the backward: those of a side that fit its items, at most eight per compute unit for both (a row of the
// workspace each), dealt to the sides by their heads.
static void plan_rotary_bwd(RotaryParams& p) {
  plan_rotary(p);
  const int cus = num_cus_of_current_device();
  const int64_t limit = 8 * (int64_t)(cus > 0 ? cus : 1);
  const int64_t heads = p.side[0].heads + p.side[1].heads;
  for (RotarySide& s : p.side) {
    const int64_t all = (rotary_items(p, s.chunks) + kWaves - 1) / kWaves, share = limit * s.heads / heads;
    const int64_t n = share < 1 ? 1 : share;
    s.workgroups = (int)(all < n ? all : n);
  }
}

int64_t rotary_workspace_bytes(int D) {
  const int cus = num_cus_of_current_device();
  return (8 * (int64_t)(cus > 0 ? cus : 1) + 2) * D * (int64_t)sizeof(float);
}

template <class T, int D, bool INTER>
static int launch_rotary_d(const RotaryParams& p, hipStream_t stream) {
  const unsigned wgs = workgroups({(rotary_items(p, p.side[0].chunks + p.side[1].chunks) + kWaves - 1) / kWaves});
  if (!wgs) return kBadArgument;
  return p.side[0].w ? launch(rotary_kernel<T, D, true, INTER>, dim3(wgs), 0, stream, p)
                     : launch(rotary_kernel<T, D, false, INTER>, dim3(wgs), 0, stream, p);
}
template <class T, int D, bool INTER>
static int launch_rotary_bwd_d(const RotaryParams& p, hipStream_t stream) {
  const dim3 grid(p.side[0].workgroups + p.side[1].workgroups);
  if (!p.side[0].w) return launch(rotary_bwd_kernel<T, D, false, INTER>, grid, 0, stream, p);
  const int rc = launch(rotary_bwd_kernel<T, D, true, INTER>, grid, kWaves * D * sizeof(float), stream, p);
  return rc ? rc : launch(rotary_weight_grad_kernel<T>, dim3(D / 4, 2), 4 * kWaves * sizeof(float), stream, p);
}

template <class T, bool INTER, bool BWD>
static int launch_rotary(const RotaryParams& p, hipStream_t stream) {
  auto at = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if constexpr (BWD) return launch_rotary_bwd_d<T, D, INTER>(p, stream);
    else return launch_rotary_d<T, D, INTER>(p, stream);
  };
  switch (p.D) {
    case 16: return at(hw::int_tag<16>{});
    case 32: return at(hw::int_tag<32>{});
    case 64: return at(hw::int_tag<64>{});
    case 128: return at(hw::int_tag<128>{});
    case 256: return at(hw::int_tag<256>{});
    case 512: return at(hw::int_tag<512>{});
  }
  return kUnsupported;
}

template <bool BWD>
static int launch_rotary_any(const RotaryParams& p, hipStream_t stream) {
  if (p.dtype == kDtypeF16) return p.interleaved ? launch_rotary<hw::half_t, true, BWD>(p, stream) : launch_rotary<hw::half_t, false, BWD>(p, stream);
  if (p.dtype == kDtypeBF16) return p.interleaved ? launch_rotary<hw::bf16_t, true, BWD>(p, stream) : launch_rotary<hw::bf16_t, false, BWD>(p, stream);
  return kUnsupported;
}

int run_rotary(RotaryParams p, hipStream_t stream) {
  if (!rotary_args_ok(p)) return kBadArgument;
  plan_rotary(p);
  return launch_rotary_any<false>(p, stream);
}

int run_rotary_bwd(RotaryParams p, hipStream_t stream) {
  if (!rotary_args_ok(p)) return kBadArgument;
  plan_rotary_bwd(p);
  return launch_rotary_any<true>(p, stream);
}

}  // namespace fa
