// Paged attention decode over a cache of e4m3 codes with an fp32 scale for each block and kv head:
//   o = sum_n p_n vs_b(n) v_n / sum_n p_n,   p_n = exp(scale ks_b(n) q.k_n),   b(n) the cache block of key n.
//
// Bound by memory: a key costs 2 D bytes per kv head, half of what a 16-bit cache costs, so half of the time is left for
// everything else.  64 sequences of 512 .. 8192 keys, 32 / 8 heads of 128: 97 us for 573 MB, 5.9 TB/s, where loads that do
// nothing else reach 6.5 (and the merge behind it 5); one workgroup per pair, 300 sequences of 1 .. 700 keys, 16 heads of 64:
// 42 us for 198 MB, 4.7 TB/s; three sequences of 40000 .. 120000 keys, 48 / 4 heads of 256: 88 us for 492 MB, 5.6 TB/s.  What
// carries it:
//   * Codes are read once and past the caches (load_once), whole 128-byte lines of an instruction: 6.5 TB/s and not 5.9 for
//     loads alone.  Lines that two instructions halve must stay in the cache between them, so a row narrower than a line is
//     not split over instructions.
//   * e4m3 becomes bf16 or fp16 exactly, two numbers per instruction, so the codes are converted in registers in front of the
//     matrix product, and whatever passes through LDS does so as codes, half the bytes.  One of the two operands passes: the
//     keys of wide rows (D >= 128), loaded as rows and read as the product wants them; the values of narrow ones.  The other
//     is loaded as the product wants it, because the order of the contraction index of a product, and of its rows, is free
//     as long as both operands (and the reader of the result) agree on it.
//   * The scales never touch the codes: ks multiplies the scores, vs the probabilities.
//   * S^T = K Q^T (keys x queries) by 16x16x32 products, as in decode.hpp: lane l = 16 g + i.  Row i of score block kb of a
//     group of 32 keys is key 8 (i / 4) + 4 kb + i % 4, so that lane (g, i) of the result has keys 8g + 4kb + 0..3 of query
//     i: the two blocks of a group are, as they are, the B operand of O^T += V^T P^T with contraction index 8g + e for key
//     8g + e.  The A operand is eight keys' codes of one value index d: lane (g, i) loads, of each of its eight keys, the
//     D / 16 codes that start at d = i D / 16, and pairs the codes of two keys by byte selection before converting them.
//     (At D = 512: 16 codes from 16 i and 16 from 256 + 16 i.)
//   * Eight keys from a multiple of eight on lie in one cache block where the block size is a power of two of at least eight:
//     one table entry, one address and two scales for all of them, and whole rows that a load instruction of all lanes takes
//     from one scalar address.  With other block sizes every lane looks up one key of a step, and the lanes that need its
//     block, row or scale get them by an exchange (the 64 sequences in blocks of 32: 105 us, of 24: 113).
//   * The chain table -> codes is a step long: entries are requested a step ahead of the codes that they lead to, between the
//     loads of this step's keys and values, since loads return in order and waiting for a later one waits for all before it.
//   * The reference of the exponentials is raised only when a score passes it by more than 2^8 (base 2): most steps need
//     no exchange between lanes.
//   * Many pairs that are cut: a range of keys to every wavefront, no barrier from the first load to the last store (100 us
//     for 64 sequences and their merge, 124 with a range to every workgroup).  Few pairs: pieces to workgroups, which leave a
//     quarter of the partial results.  Short sequences: a workgroup per pair, one kernel.  (The rule: choose_workgroups in
//     paged_fp8.py.)
//
// A table entry outside the cache (or a column behind the table) makes its keys' scores NaN, and with them the rows that
// see them; nothing is read outside the cache.
#include "paged_balance.hpp"

namespace fa {

template <int D>
struct E4m3Cfg {
  static constexpr int TK = 32;                        // keys per wavefront step: the contraction of one second product
  // wavefronts per SIMD that the registers allow, in a balanced launch and with a workgroup to a pair (300 sequences of 1 ..
  // 700 keys, 16 heads, D = 64: 43.5 us with five, 47.2 with four)
  static constexpr int WAVES = D <= 64 ? 4 : D == 128 ? 3 : D == 256 ? 2 : 1, WAVES_ALONE = D <= 64 ? 5 : WAVES;
  static constexpr int KB_BYTES = D / 4;               // codes of a key that a lane holds for the first product
  static constexpr int KW = KB_BYTES / 4;              // in dwords
  static constexpr int KSTEPS = D < 32 ? 1 : D / 32;   // products over the head size
  static constexpr int VB_BYTES = D / 16;              // codes of a key that a lane holds for the second product
  static constexpr int VW = VB_BYTES < 4 ? 1 : VB_BYTES / 4;
  static constexpr int SLICES = D / 16;
  // What passes through a patch of LDS of its wavefront, rows of D codes: the keys (wide rows) or the values (narrow ones).
  static constexpr bool STAGE_K = D >= 128;
  static constexpr int LD = D + 16 < 32 ? 32 : D + 16;  // 16 bytes behind a row: rows that are read together start in other banks
  static constexpr int PATCH = TK * LD;
  static constexpr int RPI = 1024 / D;                 // staged keys: rows of a load instruction (64 lanes of 16 bytes)
  static constexpr int NKI = STAGE_K ? TK / RPI : 0;   // and load instructions per step
  static constexpr size_t MERGE_BYTES = 4 * 16 * (D + 2) * sizeof(float);
  static constexpr size_t LDS_BYTES = 4 * PATCH > (int)MERGE_BYTES ? 4 * PATCH : MERGE_BYTES;
};

// d of row i of output slice u (the u-th code that a lane holds of a key)
template <int D>
FA_DEVICE int e4m3_value_index(int i, int u) {
  return D == 512 ? 256 * (u / 16) + 16 * i + u % 16 : i * (D / 16) + u;
}

template <int BYTES>
FA_DEVICE void load_codes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES >= 16) { const u32x4 x = hw::load_once<u32x4>(p); w[0] = x[0]; w[1] = x[1]; w[2] = x[2]; w[3] = x[3]; }
  else if constexpr (BYTES == 8) { const hw::u32x2 x = hw::load_once<hw::u32x2>(p); w[0] = x[0]; w[1] = x[1]; }
  else w[0] = hw::load_once<uint32_t>(p);
}
// the same into and out of LDS
template <int BYTES>
FA_DEVICE void put_codes(unsigned char* p, const uint32_t* w) {
  if constexpr (BYTES >= 16) *(u32x4*)p = u32x4{w[0], w[1], w[2], w[3]};
  else if constexpr (BYTES == 8) *(hw::u32x2*)p = hw::u32x2{w[0], w[1]};
  else *(uint32_t*)p = w[0];
}
template <int BYTES>
FA_DEVICE uint32_t get_codes(const unsigned char* p) {
  if constexpr (BYTES == 4) return *(const uint32_t*)p;
  else if constexpr (BYTES == 2) return *(const uint16_t*)p;
  else return *p;
}

// The cache of one sequence and kv head.  OCTETS: the block size is a power of two of at least eight, so that eight keys from
// a multiple of eight on lie in one block, and rows are 32-bit offsets apart (e4m3_octets checks).
struct E4m3Source {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const char* table;
  int entry_shift;    // log2 of the bytes of a table entry
  int bs, bs_shift, columns, num_blocks;
  int64_t s_blk, s_tok, s_scale;
  // An entry's two halves (an int32 entry twice), requested; and the block it names, or -1 where that is not one of the cache.
  struct Entry { int lo, hi, inside; };
  FA_DEVICE Entry request(int column) const {
    const char* at = table + ((int64_t)imin(column, columns - 1) << entry_shift);
    return Entry{*(const int32_t*)at, *(const int32_t*)(at + 4 * (entry_shift - 2)), column < columns};
  }
  FA_DEVICE int block(const Entry& e) const {
    const int sign = entry_shift == 3 ? 0 : e.lo;
    return e.inside && e.hi == sign && (uint32_t)e.lo < (uint32_t)num_blocks ? e.lo : -1;
  }
};

// Un-normalised result of a wavefront: lane (g, i) has values e4m3_value_index(4g + r, u) of query row i in o[u][r],
// relative to `top` (base 2), and the row's sum.
template <int D>
struct E4m3Result {
  hw::f32x4 o[D / 16];
  float top, sum;
};

// WAVES: wavefronts that share the keys, step by step in turn.
template <class T, int D, bool OCTETS, int WAVES>
FA_DEVICE void decode_e4m3(const E4m3Source& src, const T* q_row /* query row of lane % 16, or nullptr */, int n_begin,
                           int n_end, float c2, unsigned char* smem, E4m3Result<D>& out) {
  using C = E4m3Cfg<D>;
  using V8 = typename hw::Elem<T>::v8;
  using B8 = hw::bf16x8;
  // fp16 queries: probabilities times scales as the sum of two bf16 numbers (16 bits), since vs has no bound that fp16 could
  // hold them to; bf16 queries: one, as the result has no more
  constexpr bool TWO = std::is_same<T, hw::half_t>::value;
  const int tid = hw::thread_id(), lane = tid & 63, patch_index = hw::uniform(tid >> 6), wave = WAVES > 1 ? patch_index : 0;
  const int li = lane & 15, g = lane >> 4;

  // OCTETS: lane o has the table's entry for octet o of a step, otherwise lane n that for key n and the key's row in its block;
  // requested a step ahead and resolved when its keys are fetched.
  // (The first is requested in front of everything else: the context length, which bounds the steps, may still be on its way.
  // Entries behind it are columns like others, and not used.)
  E4m3Source::Entry ahead = {0, 0, 0};
  int found_block = 0, found_row = 0, ahead_row = 0;
  auto lookup = [&](int n0) {
    if constexpr (OCTETS) {
      ahead = src.request((n0 + 8 * (lane & (C::TK / 8 - 1))) >> src.bs_shift);
    } else {
      const uint32_t n = n0 + (lane & (C::TK - 1)), column = n / (uint32_t)src.bs;
      ahead = src.request((int)column);
      ahead_row = (int)(n - column * (uint32_t)src.bs);
    }
  };
  lookup(n_begin + wave * C::TK);

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
  hw::f32x4 (&oacc)[C::SLICES] = out.o;
#pragma unroll
  for (int i = 0; i < C::SLICES; ++i) oacc[i] = hw::f32x4{0.f, 0.f, 0.f, 0.f};

  const int total_steps = n_end > n_begin ? cdiv(n_end - n_begin, C::TK) : 0;
  const int my_steps = total_steps > wave ? (total_steps - wave + WAVES - 1) / WAVES : 0;
  auto step_start = [&](int j) { return n_begin + (wave + WAVES * j) * C::TK; };
  const int last = n_end - 1;

  // Keys past the end are read from the last one: their scores are masked, and what their codes hold must not be NaN where
  // no visible key's do.
  constexpr int CPR = D / 16;   // 16-byte chunks of a row
  auto k_key = [&](int n0, int kb) { return n0 + 8 * (li >> 2) + 4 * kb + (li & 3); };
  auto v_key = [&](int n0, int e) { return n0 + 8 * g + e; };
  uint32_t kw[2][C::KW], vw[8][C::VW], sw[2][C::STAGE_K ? 1 : C::KW];
  float ksc = 0.f, vsc = 0.f;   // scales of the lane's octet, or of its key
  // Element offset of a row (key of the step, at most the last), where a lane's rows are not those of one octet: the block and
  // the row in it from the lane that has looked them up.
  auto row_at = [&](int key) {
    return (int64_t)imax(hw::lane_value(found_block, key), 0) * src.s_blk + (int64_t)hw::lane_value(found_row, key) * src.s_tok;
  };
  auto scale_of = [&](float scale, int key) {
    return OCTETS ? scale : hw::lane_value(scale, key);
  };
  unsigned char* patch = smem + patch_index * C::PATCH;
  auto fetch_k = [&](int n0) {
    const uint32_t s_tok = (uint32_t)src.s_tok;
    found_block = src.block(ahead);
    found_row = ahead_row;
    if constexpr (C::STAGE_K) {
      const uint32_t col = 16 * (lane % CPR);
      if (OCTETS && n0 + C::TK <= n_end) {
        const uint32_t off = (uint32_t)(lane / CPR) * s_tok + col;
#pragma unroll
        for (int i = 0; i < C::NKI; ++i) {   // the keys of an instruction lie in one octet: one address for all lanes
          const int n = n0 + i * C::RPI;
          const int64_t at = (int64_t)imax(hw::read_lane(found_block, i * C::RPI / 8), 0) * src.s_blk + (int64_t)(n & (src.bs - 1)) * src.s_tok;
          load_codes<16>(src.kc + at + off, &kw[0][0] + 4 * i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < C::NKI; ++i) {
          const int key = imin(i * C::RPI + lane / CPR, last - n0);
          int64_t at;
          if constexpr (OCTETS) at = (int64_t)imax(hw::lane_value(found_block, key >> 3), 0) * src.s_blk + (int64_t)((n0 + key) & (src.bs - 1)) * src.s_tok;
          else at = row_at(key);
          load_codes<16>(src.kc + at + col, &kw[0][0] + 4 * i);
        }
      }
    } else {
      const int64_t octet_at = OCTETS ? (int64_t)imax(hw::lane_value(found_block, imin(li >> 2, (last - n0) >> 3)), 0) * src.s_blk : 0;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int key = imin(k_key(0, kb), last - n0);
        int64_t at = C::KB_BYTES * g;
        if constexpr (OCTETS) at += octet_at + (int64_t)((n0 + key) & (src.bs - 1)) * src.s_tok;
        else at += row_at(key);
        load_codes<C::KB_BYTES>(src.kc + at, kw[kb]);
        load_codes<C::KB_BYTES>(src.vc + at, sw[kb]);
      }
    }
  };
  // (behind fetch_k of the same step)
  auto fetch_v = [&](int n0) {
    const bool full = n0 + C::TK <= n_end;
    const int b = OCTETS ? hw::lane_value(found_block, imin(g, (last - n0) >> 3)) : found_block, blk = imax(b, 0);
    const float k = src.ks[(int64_t)blk * src.s_scale];
    vsc = src.vs[(int64_t)blk * src.s_scale];
    ksc = b >= 0 ? k : __builtin_nanf("");
    if constexpr (C::STAGE_K) {
      auto load = [&](int e, const uint8_t* row) {
        load_codes<C::VB_BYTES>(row + (D == 512 ? 16 : C::VB_BYTES) * li, vw[e]);
        if constexpr (D == 512) load_codes<16>(row + 256 + 16 * li, &vw[e][4]);
      };
      if (OCTETS && full) {
        const uint8_t* row = src.vc + (int64_t)blk * src.s_blk + (int64_t)(v_key(n0, 0) & (src.bs - 1)) * src.s_tok;
#pragma unroll
        for (int e = 0; e < 8; ++e) load(e, row + e * src.s_tok);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = imin(v_key(0, e), last - n0);
          if constexpr (OCTETS) load(e, src.vc + (int64_t)blk * src.s_blk + (int64_t)((n0 + key) & (src.bs - 1)) * src.s_tok);
          else load(e, src.vc + row_at(key));
        }
      }
    }
  };

  if (my_steps > 0) {
    fetch_k(step_start(0));
    if (my_steps > 1) lookup(step_start(1));
    fetch_v(step_start(0));
  }
  // Loads return in order: the table entries of the step after next are requested behind its keys and in front of its
  // values, so that waiting for them waits for neither these nor those.
  auto request_next = [&](int j) {
    fetch_k(step_start(j + 1));
    if (j + 2 < my_steps) lookup(step_start(j + 2));
  };
  for (int j = 0; j < my_steps; ++j) {
    const int n0 = step_start(j);
    const bool more = j + 1 < my_steps;
    // ---- the staged rows: as they were loaded into the patch ----
    hw::wave_sync();
    if constexpr (C::STAGE_K) {
#pragma unroll
      for (int i = 0; i < C::NKI; ++i) put_codes<16>(patch + (i * C::RPI + lane / CPR) * C::LD + 16 * (lane % CPR), &kw[0][0] + 4 * i);
      if (more) request_next(j);
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) put_codes<C::KB_BYTES>(patch + k_key(0, kb) * C::LD + C::KB_BYTES * g, sw[kb]);
    }
    hw::wave_sync();
    // ---- S^T ----
    hw::f32x4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      hw::f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < C::KSTEPS; ++ks) {
        uint32_t a, b;
        if constexpr (C::STAGE_K) {
          const hw::u32x2 x = *(const hw::u32x2*)(patch + k_key(0, kb) * C::LD + 64 * (ks / 2) + 16 * g + 8 * (ks % 2));
          a = x[0];
          b = x[1];
        } else {
          a = kw[kb][2 * ks < C::KW ? 2 * ks : 0];
          b = 2 * ks + 1 < C::KW ? kw[kb][2 * ks + 1] : 0u;
        }
        u32x4 x;
        x[0] = hw::from_e4m3<false>(T{}, a);
        x[1] = hw::from_e4m3<true>(T{}, a);
        x[2] = hw::from_e4m3<false>(T{}, b);
        x[3] = hw::from_e4m3<true>(T{}, b);
        acc = hw::mfma16(hw::as_v8<T>(x), qreg[ks], acc);
      }
      s[kb] = acc;
    }
    // ---- scores in the base-2 exponent, probabilities ----
    float mx = neg_inf();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float t = s[kb][r] * (scale_of(ksc, imin(v_key(0, 4 * kb + r), last - n0)) * c2);
        t = v_key(n0, 4 * kb + r) < n_end ? t : neg_inf();
        s[kb][r] = t;
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
    B8 p1, p2;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = hw::exp2_fast(s[kb][r] - m_use);
        l_i += e;
        const float pv = e * scale_of(vsc, imin(v_key(0, 4 * kb + r), last - n0));
        p1[4 * kb + r] = (hw::bf16_t)pv;
        if (TWO) p2[4 * kb + r] = (hw::bf16_t)(pv - (float)p1[4 * kb + r]);
      }
    if (!C::STAGE_K && more) request_next(j);
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int w = 0; w < C::VW; ++w) {
      uint32_t lo[4], hi[4];   // codes 4w, 4w + 1 and 4w + 2, 4w + 3 of keys 2e and 2e + 1, alternating
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t a, b;   // keys 2e and 2e + 1 of the lane
        if constexpr (C::STAGE_K) {
          a = vw[2 * e][w];
          b = vw[2 * e + 1][w];
        } else {
          const unsigned char* row = patch + v_key(0, 2 * e) * C::LD + C::VB_BYTES * li;
          a = get_codes<C::VB_BYTES>(row);
          b = get_codes<C::VB_BYTES>(row + C::LD);
        }
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
        hw::f32x4 o = hw::mfma16(va, p1, oacc[4 * w + u]);
        if (TWO) o = hw::mfma16(va, p2, o);
        oacc[4 * w + u] = o;
      }
    }
    if (more) fetch_v(step_start(j + 1));
  }

  l_i += hw::shfl_xor(l_i, 16);
  l_i += hw::shfl_xor(l_i, 32);
  out.top = m_ref;
  out.sum = l_i;
}

// The four wavefronts of a workgroup to one result per row.
template <int D>
FA_DEVICE void join_wavefronts(const E4m3Result<D>& res, int n_rows, unsigned char* smem, DecodeOut<D>& out) {
  const int lane = hw::thread_id() & 63, li = lane & 15, g = lane >> 4;
  hw::block_sync();   // every wavefront is done with its patch
  float* area = (float*)smem;
  constexpr int RS = D + 2;
  if (li < n_rows) {
    float* mine = area + ((hw::thread_id() >> 6) * 16 + li) * RS;
#pragma unroll
    for (int u = 0; u < D / 16; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[e4m3_value_index<D>(4 * g + r, u)] = res.o[u][r];
    if (g == 0) { mine[D] = res.top; mine[D + 1] = res.sum; }
  }
  merge_wavefronts<D>(area, n_rows, 1.f, out);
}

// What a wavefront has of a pair by itself, as store_balanced.
template <class T, int D>
FA_DEVICE void store_wavefront(const PagedParams& p, const E4m3Result<D>& res, int seq, int hk, int rb, bool whole, int slot_index) {
  const int lane = hw::thread_id() & 63, li = lane & 15, g = lane >> 4;
  const int G = p.Hq / p.Hkv;
  if (rb * 16 + li >= G) return;
  const float inv = res.sum == 0.f ? 0.f : 1.f / res.sum;
  constexpr int RUN = D == 512 ? 16 : D / 16;   // consecutive values of a lane
  T* out = (T*)p.out + (int64_t)seq * p.o_ss + (int64_t)(hk * G + rb * 16 + li) * p.o_sh;
  float* slot = p.ws + (int64_t)slot_index * balanced_slot_floats(D);
  if (!whole && g == 0) {
    slot[16 * D + li] = res.top * kLn2;
    slot[16 * D + 16 + li] = res.sum;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int u = 0; u < D / 16; u += RUN) {
      const int d = e4m3_value_index<D>(4 * g + r, u);
      float v[RUN];
#pragma unroll
      for (int e = 0; e < RUN; ++e) v[e] = res.o[u + e][r] * inv;
      if (whole) {
        if constexpr (RUN >= 8) {
#pragma unroll
          for (int e = 0; e < RUN; e += 8) {
            u32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = hw::pack2(T{}, v[e + 2 * i], v[e + 2 * i + 1]);
            *(u32x4*)(out + d + e) = x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < RUN; ++e) out[d + e] = (T)v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < RUN; ++e) slot[li * D + d + e] = v[e];
      }
    }
}

FA_DEVICE E4m3Source e4m3_source(const PagedParams& p, int seq, int hk) {
  E4m3Source src;
  src.kc = (const uint8_t*)p.kc + (int64_t)hk * p.kv_sh;
  src.vc = (const uint8_t*)p.vc + (int64_t)hk * p.kv_sh;
  src.ks = p.k_scales + (int64_t)hk * p.scale_sh;
  src.vs = p.v_scales + (int64_t)hk * p.scale_sh;
  src.entry_shift = p.bt64 ? 3 : 2;
  src.table = (const char*)p.block_tables + (((int64_t)seq * p.bt_stride) << src.entry_shift);
  src.bs = p.block_size;
  src.bs_shift = __builtin_ctz(p.block_size);
  src.columns = p.bt_cols;
  src.num_blocks = p.num_blocks;
  src.s_blk = p.kv_sblk;
  src.s_tok = p.kv_stok;
  src.s_scale = p.scale_sblk;
  return src;
}
static bool e4m3_octets(const PagedParams& p) {
  return p.block_size >= 8 && (p.block_size & (p.block_size - 1)) == 0 && p.kv_stok < (1 << 25);
}

template <class T>
FA_DEVICE const T* e4m3_query_row(const PagedParams& p, int seq, int hk, int rb) {
  const int G = p.Hq / p.Hkv, g = rb * 16 + (hw::thread_id() & 15);
  return g < G ? (const T*)p.q + (int64_t)seq * p.q_ss + (int64_t)(hk * G + g) * p.q_sh : nullptr;
}

// One workgroup per (sequence, kv head, 16 query heads).
template <class T, int D, bool OCTETS>
FA_KERNEL void FA_LAUNCH_BOUNDS2(kThreads, E4m3Cfg<D>::WAVES_ALONE) paged_e4m3_kernel(PagedParams p) {
  FA_LDS_DECL(smem);
  const int G = p.Hq / p.Hkv, row_blocks = (G + 15) / 16;
  const int rb = hw::block_x() % row_blocks, hk = hw::block_x() / row_blocks % p.Hkv, seq = hw::block_x() / row_blocks / p.Hkv;
  E4m3Result<D> res;
  DecodeOut<D> out;
  decode_e4m3<T, D, OCTETS, 4>(e4m3_source(p, seq, hk), e4m3_query_row<T>(p, seq, hk, rb), 0, bounded_length(p, seq),
                               p.scale * kLog2e, smem, res);
  join_wavefronts<D>(res, imin(16, G - rb * 16), smem, out);
  store_balanced<T, D>(p, out, kLn2, seq, hk, rb, true, 0);
}

// Balanced, a piece of a pair to a workgroup.
template <class T, int D, bool OCTETS>
FA_KERNEL void FA_LAUNCH_BOUNDS2(kThreads, E4m3Cfg<D>::WAVES) paged_e4m3_pieces_kernel(PagedParams p) {
  FA_LDS_DECL(smem);
  const int G = p.Hq / p.Hkv;
  balanced_walk<T, E4m3Cfg<D>::TK>(p, D, [&](int seq, int hk, int rb, int n_begin, int n_end, bool whole, int slot_index) {
    hw::block_sync();  // the previous pair's merge area has been read out
    E4m3Result<D> res;
    DecodeOut<D> out;
    decode_e4m3<T, D, OCTETS, 4>(e4m3_source(p, seq, hk), e4m3_query_row<T>(p, seq, hk, rb), n_begin, n_end, p.scale * kLog2e, smem, res);
    join_wavefronts<D>(res, imin(16, G - rb * 16), smem, out);
    store_balanced<T, D>(p, out, kLn2, seq, hk, rb, whole, slot_index);
  });
}

// Balanced, a range to every wavefront: no barrier, so that one's change from pair to pair hides behind the others' loads.
template <class T, int D, bool OCTETS>
FA_KERNEL void FA_LAUNCH_BOUNDS2(kThreads, E4m3Cfg<D>::WAVES) paged_e4m3_ranges_kernel(PagedParams p) {
  FA_LDS_DECL(smem);
  balanced_walk<T, E4m3Cfg<D>::TK, true>(p, D, [&](int seq, int hk, int rb, int n_begin, int n_end, bool whole, int slot_index) {
    E4m3Result<D> res;
    decode_e4m3<T, D, OCTETS, 1>(e4m3_source(p, seq, hk), e4m3_query_row<T>(p, seq, hk, rb), n_begin, n_end, p.scale * kLog2e, smem, res);
    store_wavefront<T, D>(p, res, seq, hk, rb, whole, slot_index);
  });
}

template <class T, int D, bool OCTETS>
static int launch_e4m3_d(const PagedParams& p, hipStream_t stream) {
  const size_t lds = E4m3Cfg<D>::LDS_BYTES;
  const int row_blocks = (p.Hq / p.Hkv + 15) / 16;
  if (p.num_wgs > 0) {
    PagedParams r = p;
    int rc;
    const int64_t pairs = (int64_t)p.num_seqs * p.Hkv * row_blocks;
    if (4 * pairs <= p.num_wgs) {
      // Of the threads that the merge has for the rows of a pair, as many share a row as leave each about eight of its partial
      // results, what it loads at once (three sequences of 80000 keys, 48 / 4 heads of 256: 89.1 us, with sixteen 90.7).
      constexpr int kSets = 1024 / D;
      int shares = 1;
      while (shares < kSets && 16 * shares * pairs <= p.num_wgs) shares *= 2;
      r.merge_rows = kSets / shares;
      rc = launch(paged_e4m3_pieces_kernel<T, D, OCTETS>, dim3(p.num_wgs), lds, stream, p);
    } else {
      rc = launch(paged_e4m3_ranges_kernel<T, D, OCTETS>, dim3(p.num_wgs), 4 * E4m3Cfg<D>::PATCH, stream, p);
      r.num_wgs = 4 * p.num_wgs;   // a record and two slots to every wavefront
    }
    return rc ? rc : run_balanced_reduce(r, stream);
  }
  const unsigned wgs = workgroups({p.num_seqs, p.Hkv, row_blocks});
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

int run_paged_e4m3(PagedParams p, hipStream_t stream) {
  if (p.num_seqs <= 0 || p.Hq <= 0 || p.Hkv <= 0 || p.Hq % p.Hkv || p.block_size <= 0 || p.bt_cols <= 0 || p.num_blocks <= 0) return kBadArgument;
  if (p.num_wgs < 0 || (p.num_wgs > 0 && !p.ws)) return kBadArgument;
  // One key behind the table says as much as all of them: a length that is not one ends soon (and the steps' arithmetic, which
  // goes up to 255 keys past the end, stays below 2^31).
  const int64_t keys = (int64_t)p.bt_cols * p.block_size + 1;
  p.max_keys = (int)(keys < 0x7fffffff - 255 ? keys : 0x7fffffff - 255);
  const bool octets = e4m3_octets(p);
  if (p.dtype == kDtypeF16) return octets ? launch_e4m3<hw::half_t, true>(p, stream) : launch_e4m3<hw::half_t, false>(p, stream);
  if (p.dtype == kDtypeBF16) return octets ? launch_e4m3<hw::bf16_t, true>(p, stream) : launch_e4m3<hw::bf16_t, false>(p, stream);
  return kUnsupported;
}

}  // namespace fa
