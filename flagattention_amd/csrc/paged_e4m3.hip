// Paged attention decode over a cache of e4m3 codes with an fp32 scale for each block and kv head:
//   o = sum_n p_n vs_b(n) v_n / sum_n p_n,   p_n = exp(scale ks_b(n) q.k_n),   b(n) the cache block of key n.
//
// Bound by memory: a key costs 2 D bytes per kv head, half of what a 16-bit cache costs, so half of the time is left for
// everything else.  What carries it:
//   * No LDS on the way.  e4m3 becomes bf16 or fp16 exactly, two numbers per instruction, so the codes are converted in
//     registers between the load and the matrix product; and the loads put every code where the product wants it, because
//     the order of the contraction index of a product, and of its rows, is free as long as both operands (and the reader of
//     the result) agree on it.
//   * The scales never touch the codes: ks multiplies the scores, vs the probabilities.
//   * S^T = K Q^T (keys x queries) by 16x16x32 products, as in decode.hpp: lane l = 16 g + i.  Row i of score block kb of a
//     group of 32 keys is key 8 (i / 4) + 4 kb + i % 4, so that lane (g, i) of the result has keys 8g + 4kb + 0..3 of query
//     i: the two blocks of a group are, as they are, the B operand of O^T += V^T P^T with contraction index 8g + e for key
//     8g + e.  The A operand is eight keys' codes of one value index d: lane (g, i) loads, of each of its eight keys, the
//     D / 16 codes that start at d = i D / 16, and pairs the codes of two keys by byte selection before converting them.
//     (At D = 512: 16 codes from 16 i and 16 from 256 + 16 i.)
//   * The eight keys of a lane lie in one cache block where the block size is a multiple of eight: one table entry, one
//     address and two scales for all of them.  Other block sizes look up every key.
//   * The reference of the exponentials is raised only when a score passes it by more than 2^8 (base 2): most steps need
//     no exchange between lanes.
//
// A table entry outside the cache (or a column behind the table) makes its keys' scores NaN, and with them the rows that
// see them; nothing is read outside the cache.
#include "paged_balance.hpp"

namespace fa {

template <int D>
struct E4m3Cfg {
  static constexpr int GROUPS = D <= 128 ? 2 : 1;      // groups of 32 keys per wavefront step
  static constexpr int TK = 32 * GROUPS;
  static constexpr int KB_BYTES = D / 4;               // codes of a key that a lane holds for the first product
  static constexpr int KW = KB_BYTES / 4;              // in dwords
  static constexpr int KSTEPS = D < 32 ? 1 : D / 32;   // products over the head size
  static constexpr int VB_BYTES = D / 16;              // codes of a key that a lane holds for the second product
  static constexpr int VW = VB_BYTES < 4 ? 1 : VB_BYTES / 4;
  static constexpr int SLICES = D / 16;
  static constexpr size_t MERGE_BYTES = 4 * 16 * (D + 2) * sizeof(float);
};

// d of row i of output slice u (the u-th code that a lane holds of a key)
template <int D>
FA_DEVICE int e4m3_value_index(int i, int u) {
  return D == 512 ? 256 * (u / 16) + 16 * i + u % 16 : i * (D / 16) + u;
}

template <int BYTES>
FA_DEVICE void load_codes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES >= 16) { const u32x4 x = *(const u32x4*)p; w[0] = x[0]; w[1] = x[1]; w[2] = x[2]; w[3] = x[3]; }
  else if constexpr (BYTES == 8) { const hw::u32x2 x = *(const hw::u32x2*)p; w[0] = x[0]; w[1] = x[1]; }
  else if constexpr (BYTES == 4) w[0] = *(const uint32_t*)p;
  else if constexpr (BYTES == 2) w[0] = *(const uint16_t*)p;
  else w[0] = *p;
}

// The cache of one sequence and kv head.  OCTETS: eight keys from a multiple of eight on lie in one block.
template <bool OCTETS>
struct E4m3Source {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const char* table;
  int bt64, bs, bs_shift, columns, num_blocks;
  int64_t s_blk, s_tok, s_scale;
  // a block number that can be used and whether it is the table's; n: any key
  FA_DEVICE int lookup(int n) const {
    int c = bs_shift >= 0 ? n >> bs_shift : n / bs;
    const bool inside = c < columns;
    c = inside ? c : columns - 1;
    const int64_t b = bt64 ? ((const int64_t*)table)[c] : ((const int32_t*)table)[c];
    return inside && b >= 0 && b < num_blocks ? (int)b : -1;
  }
  FA_DEVICE int slot(int n) const { return bs_shift >= 0 ? n & (bs - 1) : n % bs; }
};

template <class T, int D, bool OCTETS>
FA_DEVICE void decode_e4m3(const E4m3Source<OCTETS>& src, const T* q_row /* query row of lane % 16, or nullptr */, int n_rows,
                           int n_begin, int n_end, float c2, unsigned char* smem, DecodeOut<D>& out) {
  using C = E4m3Cfg<D>;
  using V8 = typename hw::Elem<T>::v8;
  using B8 = hw::bf16x8;
  // fp16 queries: probabilities times scales as the sum of two bf16 numbers (16 bits), since vs has no bound that fp16 could
  // hold them to; bf16 queries: one, as the result has no more
  constexpr bool TWO = std::is_same<T, hw::half_t>::value;
  constexpr int NK = OCTETS ? 1 : 2, NV = OCTETS ? 1 : 8;
  const int tid = hw::thread_id(), lane = tid & 63, wave = hw::uniform(tid >> 6);
  const int li = lane & 15, g = lane >> 4;

  // this lane's query row as B operand, in the order in which it holds a key's codes
  V8 qreg[C::KSTEPS];
#pragma unroll
  for (int ks = 0; ks < C::KSTEPS; ++ks) {
    u32x4 z = {0u, 0u, 0u, 0u};
    if (q_row) {
      if constexpr (D >= 64) z = *(const u32x4*)(q_row + 64 * (ks / 2) + 16 * g + 8 * (ks % 2));
      else if constexpr (D == 32) z = *(const u32x4*)(q_row + 8 * g);
      else { const hw::u32x2 x = *(const hw::u32x2*)(q_row + 4 * g); z[0] = x[0]; z[1] = x[1]; }
    }
    qreg[ks] = hw::as_v8<T>(z);
  }

  float m_ref = neg_inf(), l_i = 0.f;
  hw::f32x4 oacc[C::SLICES];
#pragma unroll
  for (int i = 0; i < C::SLICES; ++i) oacc[i] = hw::f32x4{0.f, 0.f, 0.f, 0.f};

  const int total_steps = n_end > n_begin ? cdiv(n_end - n_begin, C::TK) : 0;
  const int my_steps = total_steps > wave ? (total_steps - wave + 3) / 4 : 0;
  auto step_start = [&](int j) { return n_begin + (wave + 4 * j) * C::TK; };
  const int last = n_end - 1;

  // blocks of the lane's keys: rows of the score blocks, contraction indices of the second product
  struct Blocks { int k[C::GROUPS][NK], v[C::GROUPS][NV]; } blocks;
  auto k_key = [&](int n0, int grp, int kb) { return n0 + 32 * grp + 8 * (li >> 2) + 4 * kb + (li & 3); };
  auto v_key = [&](int n0, int grp, int e) { return n0 + 32 * grp + 8 * g + e; };
  auto lookup = [&](int n0) {
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp) {
#pragma unroll
      for (int i = 0; i < NK; ++i) blocks.k[grp][i] = src.lookup(imin(k_key(n0, grp, i), last));
#pragma unroll
      for (int i = 0; i < NV; ++i) blocks.v[grp][i] = src.lookup(imin(v_key(n0, grp, i), last));
    }
  };

  uint32_t kw[C::GROUPS][2][C::KW], vw[C::GROUPS][8][C::VW];
  float ksc[C::GROUPS][NV], vsc[C::GROUPS][NV];
  // keys past the end are read from the last one: their scores are masked, and what their codes hold must not be NaN where
  // no visible key's do
  auto fetch_k = [&](int n0) {
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int n = imin(k_key(n0, grp, kb), last);
        const uint8_t* row = src.kc + (int64_t)imax(blocks.k[grp][OCTETS ? 0 : kb], 0) * src.s_blk + (int64_t)src.slot(n) * src.s_tok;
        if constexpr (D >= 64) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) load_codes<16>(row + 64 * c + 16 * g, &kw[grp][kb][4 * c]);
        } else {
          load_codes<C::KB_BYTES>(row + C::KB_BYTES * g, kw[grp][kb]);
        }
      }
    }
  };
  auto fetch_v = [&](int n0) {
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int b = blocks.v[grp][i];
        const float k = src.ks[(int64_t)imax(b, 0) * src.s_scale], v = src.vs[(int64_t)imax(b, 0) * src.s_scale];
        ksc[grp][i] = b >= 0 ? k : __builtin_nanf("");
        vsc[grp][i] = v;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int n = imin(v_key(n0, grp, e), last);
        const uint8_t* row = src.vc + (int64_t)imax(blocks.v[grp][OCTETS ? 0 : e], 0) * src.s_blk + (int64_t)src.slot(n) * src.s_tok;
        load_codes<C::VB_BYTES>(row + (D == 512 ? 16 : C::VB_BYTES) * li, vw[grp][e]);
        if constexpr (D == 512) load_codes<16>(row + 256 + 16 * li, &vw[grp][e][4]);
      }
    }
  };

  if (my_steps > 0) {
    lookup(step_start(0));
    fetch_k(step_start(0));
    fetch_v(step_start(0));
    if (my_steps > 1) lookup(step_start(1));
  }
  for (int j = 0; j < my_steps; ++j) {
    const int n0 = step_start(j);
    // ---- S^T ----
    hw::f32x4 s[C::GROUPS][2];
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        hw::f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < C::KSTEPS; ++ks) {
          const uint32_t a = kw[grp][kb][2 * ks < C::KW ? 2 * ks : 0], b = 2 * ks + 1 < C::KW ? kw[grp][kb][2 * ks + 1] : 0u;
          u32x4 x;
          x[0] = hw::from_e4m3<false>(T{}, a);
          x[1] = hw::from_e4m3<true>(T{}, a);
          x[2] = hw::from_e4m3<false>(T{}, b);
          x[3] = hw::from_e4m3<true>(T{}, b);
          acc = hw::mfma16(hw::as_v8<T>(x), qreg[ks], acc);
        }
        s[grp][kb] = acc;
      }
    // ---- scores in the base-2 exponent, probabilities ----
    float mx = neg_inf();
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float t = s[grp][kb][r] * (ksc[grp][OCTETS ? 0 : 4 * kb + r] * c2);
          t = v_key(n0, grp, 4 * kb + r) < n_end ? t : neg_inf();
          s[grp][kb][r] = t;
          mx = fmaxf(mx, t);
        }
    if (hw::wave_any(mx > m_ref + 8.f)) {   // m_ref is the same in the four lanes of a query row
      mx = fmaxf(mx, hw::shfl_xor(mx, 16));
      mx = fmaxf(mx, hw::shfl_xor(mx, 32));
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = hw::exp2_fast(m_ref - (m_new == neg_inf() ? 0.f : m_new));
      m_ref = m_new;
      l_i *= alpha;
#pragma unroll
      for (int i = 0; i < C::SLICES; ++i) oacc[i] *= alpha;
    }
    const float m_use = m_ref == neg_inf() ? 0.f : m_ref;
    B8 p1[C::GROUPS], p2[C::GROUPS];
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = hw::exp2_fast(s[grp][kb][r] - m_use);
          l_i += e;
          const float pv = e * vsc[grp][OCTETS ? 0 : 4 * kb + r];
          p1[grp][4 * kb + r] = (hw::bf16_t)pv;
          if (TWO) p2[grp][4 * kb + r] = (hw::bf16_t)(pv - (float)p1[grp][4 * kb + r]);
        }
    const bool more = j + 1 < my_steps;
    if (more) fetch_k(step_start(j + 1));
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int grp = 0; grp < C::GROUPS; ++grp)
#pragma unroll
      for (int w = 0; w < C::VW; ++w) {
        uint32_t lo[4], hi[4];   // codes 4w, 4w + 1 and 4w + 2, 4w + 3 of keys 2e and 2e + 1, alternating
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = vw[grp][2 * e][w], b = vw[grp][2 * e + 1][w];
          lo[e] = hw::byte_perm(b, a, 0x05010400u);
          hi[e] = hw::byte_perm(b, a, 0x07030602u);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (4 * w + u >= C::SLICES) break;
          u32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t c = u < 2 ? lo[e] : hi[e];
            x[e] = u % 2 ? hw::from_e4m3<true>(hw::bf16_t{}, c) : hw::from_e4m3<false>(hw::bf16_t{}, c);
          }
          const B8 va = hw::as_v8<hw::bf16_t>(x);
          hw::f32x4 o = hw::mfma16(va, p1[grp], oacc[4 * w + u]);
          if (TWO) o = hw::mfma16(va, p2[grp], o);
          oacc[4 * w + u] = o;
        }
      }
    if (more) {
      fetch_v(step_start(j + 1));
      if (j + 2 < my_steps) lookup(step_start(j + 2));
    }
  }

  l_i += hw::shfl_xor(l_i, 16);
  l_i += hw::shfl_xor(l_i, 32);
  float* area = (float*)smem;
  constexpr int RS = D + 2;
  if (li < n_rows) {
    float* mine = area + (wave * 16 + li) * RS;
#pragma unroll
    for (int u = 0; u < C::SLICES; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[e4m3_value_index<D>(4 * g + r, u)] = oacc[u][r];
    if (g == 0) { mine[D] = m_ref; mine[D + 1] = l_i; }
  }
  merge_wavefronts<D>(area, n_rows, 1.f, out);
}

template <bool OCTETS>
FA_DEVICE E4m3Source<OCTETS> e4m3_source(const PagedParams& p, int seq, int hk) {
  E4m3Source<OCTETS> src;
  src.kc = (const uint8_t*)p.kc + (int64_t)hk * p.kv_sh;
  src.vc = (const uint8_t*)p.vc + (int64_t)hk * p.kv_sh;
  src.ks = p.k_scales + (int64_t)hk * p.scale_sh;
  src.vs = p.v_scales + (int64_t)hk * p.scale_sh;
  src.table = (const char*)p.block_tables + (((int64_t)seq * p.bt_stride) << (p.bt64 ? 3 : 2));
  src.bt64 = p.bt64;
  src.bs = p.block_size;
  src.bs_shift = (p.block_size & (p.block_size - 1)) == 0 ? __builtin_ctz(p.block_size) : -1;
  src.columns = p.bt_cols;
  src.num_blocks = p.num_blocks;
  src.s_blk = p.kv_sblk;
  src.s_tok = p.kv_stok;
  src.s_scale = p.scale_sblk;
  return src;
}

// One workgroup per (sequence, kv head, 16 query heads).
template <class T, int D, bool OCTETS>
FA_KERNEL void FA_LAUNCH_BOUNDS2(kThreads, (D <= 128 ? 2 : 1)) paged_e4m3_kernel(PagedParams p) {
  FA_LDS_DECL(smem);
  const int li = hw::thread_id() & 15;
  const int G = p.Hq / p.Hkv, row_blocks = (G + 15) / 16;
  const int rb = hw::block_x() % row_blocks, hk = hw::block_x() / row_blocks % p.Hkv, seq = hw::block_x() / row_blocks / p.Hkv;
  const int g_lane = rb * 16 + li;
  const T* q_row = nullptr;
  if (g_lane < G) q_row = (const T*)p.q + (int64_t)seq * p.q_ss + (int64_t)(hk * G + g_lane) * p.q_sh;
  DecodeOut<D> res;
  decode_e4m3<T, D, OCTETS>(e4m3_source<OCTETS>(p, seq, hk), q_row, imin(16, G - rb * 16), 0, imax(0, p.context_lens[seq]),
                            p.scale * kLog2e, smem, res);
  store_balanced<T, D>(p, res, kLn2, seq, hk, rb, true, 0);
}

template <class T, int D, bool OCTETS>
FA_KERNEL void FA_LAUNCH_BOUNDS2(kThreads, (D <= 128 ? 2 : 1)) paged_e4m3_balanced_kernel(PagedParams p) {
  FA_LDS_DECL(smem);
  const int li = hw::thread_id() & 15;
  const int G = p.Hq / p.Hkv;
  balanced_walk<T, E4m3Cfg<D>::TK>(p, D, [&](int seq, int hk, int rb, int n_begin, int n_end, bool whole, int slot_index) {
    const int g_lane = rb * 16 + li;
    const T* q_row = nullptr;
    if (g_lane < G) q_row = (const T*)p.q + (int64_t)seq * p.q_ss + (int64_t)(hk * G + g_lane) * p.q_sh;
    hw::block_sync();  // the previous pair's merge area has been read out
    DecodeOut<D> res;
    decode_e4m3<T, D, OCTETS>(e4m3_source<OCTETS>(p, seq, hk), q_row, imin(16, G - rb * 16), n_begin, n_end, p.scale * kLog2e, smem, res);
    store_balanced<T, D>(p, res, kLn2, seq, hk, rb, whole, slot_index);
  });
}

template <class T, int D, bool OCTETS>
static int launch_e4m3_d(const PagedParams& p, hipStream_t stream) {
  const size_t lds = E4m3Cfg<D>::MERGE_BYTES;
  if (p.num_wgs > 0) {
    const int rc = launch(paged_e4m3_balanced_kernel<T, D, OCTETS>, dim3(p.num_wgs), lds, stream, p);
    return rc ? rc : run_balanced_reduce(p, stream);
  }
  const unsigned wgs = workgroups({p.num_seqs, p.Hkv, (p.Hq / p.Hkv + 15) / 16});
  return wgs ? launch(paged_e4m3_kernel<T, D, OCTETS>, dim3(wgs), lds, stream, p) : kBadArgument;
}

template <class T, bool OCTETS>
static int launch_e4m3(const PagedParams& p, hipStream_t stream) {
  switch (p.D) {
    case 16: return launch_e4m3_d<T, 16, OCTETS>(p, stream);
    case 32: return launch_e4m3_d<T, 32, OCTETS>(p, stream);
    case 64: return launch_e4m3_d<T, 64, OCTETS>(p, stream);
    case 128: return launch_e4m3_d<T, 128, OCTETS>(p, stream);
    case 256: return launch_e4m3_d<T, 256, OCTETS>(p, stream);
    case 512: return launch_e4m3_d<T, 512, OCTETS>(p, stream);
  }
  return kUnsupported;
}

int run_paged_e4m3(const PagedParams& p, hipStream_t stream) {
  if (p.num_seqs <= 0 || p.Hq <= 0 || p.Hkv <= 0 || p.Hq % p.Hkv || p.block_size <= 0 || p.bt_cols <= 0 || p.num_blocks <= 0) return kBadArgument;
  if (p.num_wgs < 0 || (p.num_wgs > 0 && !p.ws)) return kBadArgument;
  const bool octets = p.block_size % 8 == 0;
  if (p.dtype == kDtypeF16) return octets ? launch_e4m3<hw::half_t, true>(p, stream) : launch_e4m3<hw::half_t, false>(p, stream);
  if (p.dtype == kDtypeBF16) return octets ? launch_e4m3<hw::bf16_t, true>(p, stream) : launch_e4m3<hw::bf16_t, false>(p, stream);
  return kUnsupported;
}

}  // namespace fa
