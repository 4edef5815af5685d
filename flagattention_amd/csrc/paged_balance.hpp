// Balanced launch of the paged decode kernels: which keys a workgroup streams, and where its results go.
//
// The keys of all (sequence, kv head) pairs, counted in units, are laid end
// to end and cut into num_wgs equal ranges, one per workgroup, so that every workgroup streams the
// same number of bytes whatever the spread of context lengths and the launch is exactly one
// resident wave of workgroups.
//
// A unit is four steps of a wavefront (128 keys where a step has 32) where there are pairs enough (more than a quarter of
// the workgroups).  With few pairs a unit
// is at least that and as many steps as make at most one unit per workgroup: every workgroup then takes one unit of one
// pair.  A workgroup whose range held the end of one pair and the beginning of the next would run two of them one
// after the other, each with its own chain of dependent loads (table, keys) and merge, 4-5 us of which a short
// launch has little else: 4 sequences of 100 .. 2000 keys, 8 kv heads: 12.7 -> 9.1 us.
//
// A pair that lies inside one range is finished by that workgroup
// and written to `out`; a pair cut by range boundaries leaves one partial result per workgroup it
// touches (at most two per workgroup: the pair it starts in the middle of, slot 2w, and the pair it
// leaves unfinished, slot 2w + 1), which paged_balanced_reduce_kernel merges.
//
// Workspace (floats): 2 * num_wgs slots of [16][D] normalised outputs, [16] max logits, [16] sums of
// exponentials; then num_wgs records of 4 ints {sequence, kv head, row block, number of following
// workgroups that continue the pair left unfinished} (the last is 0 when there is no such pair).
#pragma once
#include "decode.hpp"
#include "params.hpp"

namespace fa {

constexpr int kMinUnitsPerWg = 2;   // where a range may cross pairs

FA_DEVICE int balanced_slot_floats(int D) { return 16 * D + 32; }

FA_DEVICE int bounded_length(const PagedParams& p, int seq) {
  const int n = imax(0, p.context_lens[seq]);
  return p.max_keys > 0 ? imin(n, p.max_keys) : n;
}

// Runs pair(seq, hk, rb, n_begin, n_end, whole, slot index) for every piece of a pair in this workgroup's range, and clears
// the output rows of empty sequences.  STEP_KEYS: the keys of a wavefront's step.  WAVES: every wavefront has a range of its
// own, in units of one step (the workgroups above are wavefronts then, four times as many), and pieces are dealt so however
// few pairs there are.
template <class T, int STEP_KEYS, bool WAVES = false, class Pair>
FA_DEVICE void balanced_walk(const PagedParams& p, const int D, Pair pair) {
  constexpr int kUnitKeys = WAVES ? STEP_KEYS : 4 * STEP_KEYS, kStepKeys = STEP_KEYS;
  constexpr int kMembers = WAVES ? 64 : kThreads;
  const int lane = hw::thread_id() & 63, tid = WAVES ? lane : hw::thread_id();
  const int w = WAVES ? hw::uniform(4 * hw::block_x() + (hw::thread_id() >> 6)) : hw::block_x();
  const int num_wgs = WAVES ? 4 * p.num_wgs : p.num_wgs;
  const int G = p.Hq / p.Hkv;
  const int row_blocks = (G + 15) / 16;
  const int pairs_per_seq = p.Hkv * row_blocks;

  // ---- every wavefront scans the context lengths for itself, 64 at a time: no LDS, no barrier ----
  auto length_of = [&](int s) { return s < p.num_seqs ? bounded_length(p, s) : 0; };
  const int first_lengths = length_of(lane);   // both scans begin with these
  const int64_t num_pairs = (int64_t)p.num_seqs * pairs_per_seq;
  const bool one_each = !WAVES && 4 * num_pairs <= num_wgs;
  const int grain = one_each ? kStepKeys : kUnitKeys;
  int total_units = 0;
  for (int base = 0; base < p.num_seqs; base += 64) {
    const int s = base + lane;
    const int u = cdiv(base == 0 ? first_lengths : length_of(s), grain);
    // An empty sequence has no keys to stream: its output rows are zero.  Every wavefront sees the same
    // empty sequences here; they are dealt round-robin to the workgroups, and the threads of the one
    // that takes a sequence clear its rows together.
    for (uint64_t todo = hw::ballot(s < p.num_seqs && u == 0 && s % num_wgs == w); todo; todo &= todo - 1) {
      const int e = base + __builtin_ctzll(todo);
      for (int i = tid; i < p.Hq * D; i += kMembers) ((T*)p.out)[(int64_t)e * p.o_ss + (int64_t)(i / D) * p.o_sh + i % D] = (T)0.f;
    }
    total_units += hw::last_lane(hw::wave_prefix_sum(u));
  }
  // everything derived from the total (the key ranges, the step counts of the wavefronts) stays in scalar registers
  const int64_t total0 = (int64_t)total_units * pairs_per_seq;
  const int64_t per = one_each ? 1 : (int64_t)imax(kMinUnitsPerWg, (int)((total0 + num_wgs - 1) / num_wgs));
  int unit_keys = kUnitKeys;
  if (one_each) {
    // Pieces of n steps' worth of keys: sum over pairs of ceil(steps / n) is at most total / n + pairs, and about
    // total / n + pairs / 2.  The n that makes the latter num_wgs is taken if the pieces really fit, else the safe one.
    auto steps_for = [&](int64_t wgs) { return (int)imax(kUnitKeys / kStepKeys, (int)((total0 + wgs - 1) / wgs)); };
    const int tight = steps_for(num_wgs - num_pairs / 2);
    int pieces = 0;
    for (int base = 0; base < p.num_seqs; base += 64)
      pieces += hw::last_lane(hw::wave_prefix_sum(cdiv(base == 0 ? first_lengths : length_of(base + lane), tight * kStepKeys)));
    unit_keys = kStepKeys * ((int64_t)pieces * pairs_per_seq <= num_wgs ? tight : steps_for(num_wgs - num_pairs));
  }
  const int64_t u_begin = (int64_t)w * per;
  int* meta = (int*)(p.ws + (int64_t)2 * num_wgs * balanced_slot_floats(D)) + 4 * w;
  // the sequence whose pairs hold unit u_begin, and the units of the sequences before it
  int seq = 0, before = 0, all_units = 0;
  {
    int running = 0;
    for (int base = 0; base < p.num_seqs; base += 64) {
      const int s = base + lane;
      const int u = cdiv(base == 0 ? first_lengths : length_of(s), unit_keys);
      const int incl = hw::wave_prefix_sum(u), excl = incl - u;
      const bool here = u > 0 && (int64_t)(running + excl) * pairs_per_seq <= u_begin &&
                        u_begin < (int64_t)(running + incl) * pairs_per_seq;
      const uint64_t hit = hw::ballot(here);
      const int first = hit ? __builtin_ctzll(hit) : 0;
      const int excl_first = hw::lane_value(excl, first);
      if (hit) { seq = base + first; before = running + excl_first; }
      running += hw::last_lane(incl);
    }
    seq = hw::uniform(seq);
    before = hw::uniform(before);
    all_units = hw::uniform(running);
  }
  const int64_t total = (int64_t)all_units * pairs_per_seq;
  const int64_t u_end = u_begin + per < total ? u_begin + per : total;
  if (u_begin >= total) {  // whole workgroup
    if (tid == 0) meta[3] = 0;
    return;
  }
  int64_t u = u_begin;
  int unfinished = 0;

  while (u < u_end) {
    const int ctx = hw::uniform(bounded_length(p, seq));
    const int us = ctx > 0 ? cdiv(ctx, unit_keys) : 0;
    const int local = (int)(u - (int64_t)before * pairs_per_seq);  // unit index inside this sequence's pairs
    if (us == 0 || local >= us * pairs_per_seq) { before += us; ++seq; continue; }
    const int pr = local / us, lo = local % us;
    const int hk = pr / row_blocks, rb = pr % row_blocks;
    const int hi = (int)(u_end - u < (int64_t)(us - lo) ? lo + (u_end - u) : us);
    const int n_begin = lo * unit_keys, n_end = imin((int64_t)ctx, (int64_t)hi * unit_keys);

    pair(seq, hk, rb, n_begin, n_end, lo == 0 && hi == us, 2 * w + (lo == 0 ? 1 : 0));
    if (lo == 0 && hi < us) {  // this pair continues in the following workgroups, `per` units each
      unfinished = (int)(((int64_t)(us - hi) + per - 1) / per);
      if (tid == 0) { meta[0] = seq; meta[1] = hk; meta[2] = rb; }
    }
    u += hi - lo;
  }
  if (tid == 0) meta[3] = unfinished;
}

// What a workgroup has of a pair: the output rows themselves where it has the whole pair, else a partial result.
// row_max * max_scale is the maximum in the natural exponent.
template <class T, int D>
FA_DEVICE void store_balanced(const PagedParams& p, const DecodeOut<D>& res, float max_scale, int seq, int hk, int rb, bool whole,
                              int slot_index) {
  const int G = p.Hq / p.Hkv;
  float* slot = p.ws + (int64_t)slot_index * balanced_slot_floats(D);
  const int out_tid = thread_for_output();
#pragma unroll
  for (int e = 0; e < DecodeOut<D>::kPerThread; ++e) {
    const int idx = out_tid + e * kThreads;
    const int row = idx / D, d = idx % D;
    const int g = rb * 16 + row;
    if (idx < 16 * D && g < G) {
      const float val = res.row_sum[e] == 0.f ? 0.f : res.o[e] / res.row_sum[e];
      if (whole) {
        ((T*)p.out)[(int64_t)seq * p.o_ss + (int64_t)(hk * G + g) * p.o_sh + d] = (T)val;
      } else {
        slot[row * D + d] = val;
        if (d == 0) {
          slot[16 * D + row] = res.row_max[e] * max_scale;
          slot[16 * D + 16 + row] = res.row_sum[e];
        }
      }
    }
  }
}

// The second launch of a balanced call (paged.hip): merges the pairs that were cut.
int run_balanced_reduce(const PagedParams& p, hipStream_t stream);

}  // namespace fa
