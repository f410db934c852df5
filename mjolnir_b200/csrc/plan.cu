// Host-side split-KV planner and the runner handle of the C ABI.
//
// mj_plan_split_kv is the planner of mjolnir_b200/plan.py in C++, for hosts
// that drive the library without Python: the reference's occupancy-pinned
// split (arch/thor/plan.py:140-197: one wave holds sm_count * ctas_per_sm /
// (h_k * n_q_tiles) work items; a batch smaller than a wave gets the smallest
// chunk whose items fit one wave; items longest first, padded with empty items
// for a fixed grid) plus the B200 rebalance (the cheapest of that chunk and
// every ceil(T / k), k = 1 .. max_splits, under a longest-first model of the
// persistent grid's rounds plus a per-item overhead). Both produce the same
// plans for the same inputs (checked against each other in the tests).
//
// mj_runner owns what a decode step needs besides the caller's tensors: the
// fixed-address work list and split counts (so a captured CUDA graph replays
// later plans), the split-KV partials, the device status word, and a pinned
// staging copy of the plan. It allocates only in mj_create.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <functional>
#include <set>
#include <vector>

#include "common.cuh"

namespace mj {
int set_last_error(int code, const char* msg);
}

namespace {

struct Item {
  int32_t seq, tb, te, split;
};

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Longest-first wave model of the decode time, in tile units.
double wave_cost(const std::vector<int>& tiles, int chunk, int slots, double item_overhead) {
  std::vector<int> lens;
  int kmax = 0;
  for (int t : tiles) {
    const int k = ceil_div(t, chunk);
    kmax = std::max(kmax, k);
    for (int j = 0; j + 1 < k; ++j) lens.push_back(chunk);
    lens.push_back(t - (k - 1) * chunk);
  }
  std::sort(lens.begin(), lens.end(), [](int a, int b) { return a > b; });
  double sum = 0.0;
  int waves = 0;
  for (size_t i = 0; i < lens.size(); i += (size_t)slots) {
    sum += lens[i];
    ++waves;
  }
  return sum + item_overhead * waves + (kmax > 1 ? 0.25 : 0.0);
}

}  // namespace

struct mj_runner {
  int device, h_q, h_k, head_size, page_size, max_num_seqs, max_q_len, kv_format, max_splits, ctas_per_sm, sm_count;
  int cap;  // work-list capacity (fixed-grid length)
  int32_t* work = nullptr;      // device (cap, 4)
  int32_t* n_splits = nullptr;  // device (max_num_seqs,)
  float* o_part = nullptr;      // device partials
  float* lse_part = nullptr;
  int32_t* status = nullptr;    // device status word
  int32_t* stage = nullptr;     // pinned host staging: work then n_splits
  cudaEvent_t staged = nullptr; // the last plan's copy out of the staging buffer
  // the last plan
  int num_seqs = 0, q_len = 0, num_work = 0, with_reduction = 0, chunk_tiles = 0;
};

extern "C" {

int mj_plan_split_kv(const int32_t* seq_lens, int num_seqs, int h_k, int n_q_tiles, int sm_count, int ctas_per_sm,
                     int max_splits, int pad_to, int rebalance, float item_overhead, int32_t* work_out,
                     int work_capacity, int32_t* n_splits_out, int* num_work_out, int* chunk_tiles_out) {
  if (!seq_lens || num_seqs <= 0 || h_k <= 0 || n_q_tiles <= 0 || sm_count <= 0 || ctas_per_sm <= 0 || max_splits <= 0 ||
      !work_out || !n_splits_out || !num_work_out)
    return mj::set_last_error(MJ_ERR_INVALID, "mj_plan_split_kv: invalid argument");
  std::vector<int> tiles(num_seqs);
  int T = 1;
  for (int b = 0; b < num_seqs; ++b) {
    tiles[b] = std::max(1, ceil_div(std::max(seq_lens[b], 0), mj::kTileRows));
    T = std::max(T, tiles[b]);
  }
  const int slots = std::max(1, (sm_count * ctas_per_sm) / (h_k * n_q_tiles));
  const int shortest = std::max(1, ceil_div(T, max_splits));  // cap chunks per sequence
  int chunk = T;
  if (max_splits > 1) {
    // the reference's chunk: none when the batch fills a round, else the
    // shortest chunk whose items fit in one round
    if (num_seqs < slots) {
      int lo = shortest, hi = T;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        int64_t items = 0;
        for (int t : tiles) items += ceil_div(t, mid);
        if (items <= slots) hi = mid;
        else lo = mid + 1;
      }
      chunk = lo;
    }
    if (rebalance) {  // the cheapest of it and every ceil(T / k) under the round model
      std::set<int> cset{chunk};
      for (int k = 1; k <= max_splits; ++k) cset.insert(std::max(shortest, ceil_div(T, k)));
      double best = 0.0;
      bool have = false;
      for (auto it = cset.rbegin(); it != cset.rend(); ++it) {  // longest chunk first: it keeps a tie
        const double cost = wave_cost(tiles, *it, slots, item_overhead);
        if (!have || cost < best - 1e-9) {
          best = cost;
          chunk = *it;
          have = true;
        }
      }
    }
  }
  std::vector<Item> work;
  for (int b = 0; b < num_seqs; ++b) {
    const int k = ceil_div(tiles[b], chunk);
    n_splits_out[b] = k;
    for (int j = 0; j < k; ++j) work.push_back({b, j * chunk, std::min((j + 1) * chunk, tiles[b]), j});
  }
  std::stable_sort(work.begin(), work.end(), [](const Item& x, const Item& y) { return (x.te - x.tb) > (y.te - y.tb); });
  const int n = (int)work.size();
  const int total = pad_to > 0 ? pad_to : n;
  if (pad_to > 0 && pad_to < n) return mj::set_last_error(MJ_ERR_INVALID, "mj_plan_split_kv: pad_to below the work items");
  if (total > work_capacity) return mj::set_last_error(MJ_ERR_INVALID, "mj_plan_split_kv: work_out too small");
  for (int i = 0; i < total; ++i) {
    const Item w = i < n ? work[i] : Item{0, 0, 0, 0};
    work_out[4 * i + 0] = w.seq;
    work_out[4 * i + 1] = w.tb;
    work_out[4 * i + 2] = w.te;
    work_out[4 * i + 3] = w.split;
  }
  *num_work_out = total;
  if (chunk_tiles_out) *chunk_tiles_out = chunk;
  return MJ_OK;
}

// ---- block attention -------------------------------------------------------

// Splitting: an equal share of the step's key tiles per SM bounds an item, but
// a piece keeps at least kMinPiece tiles (its prologue and epilogue cost about
// as much as two). Where the pieces would need more than max_slots partials,
// the bound doubles until they do not.
int mj_block_plan(const int32_t* query_lens, const int32_t* seq_lens, int num_seqs, int h_q, int h_k, int head_size,
                  int causal, int sm_count, int max_slots, int32_t* work_out, int work_capacity, int32_t* merges_out,
                  int merges_capacity, int* num_work, int* num_merges, int* num_slots) {
  if (num_seqs < 0 || h_k <= 0 || h_q <= 0 || h_q % h_k || (head_size != 128 && head_size != 256) || sm_count <= 0 ||
      max_slots < 0 || (num_seqs && (!query_lens || !seq_lens)) || !num_work || !num_merges || !num_slots)
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_plan: invalid argument");
  constexpr int kMinPiece = 8;
  const int h_r = h_q / h_k, rows = MJ_BLOCK_ROWS(head_size), keys = MJ_BLOCK_KEYS;
  struct Block {
    int32_t seq, row0, tiles;
  };
  try {
    std::vector<Block> blocks;
    int64_t total = 0;
    for (int s = 0; s < num_seqs; ++s) {
      const int64_t n = query_lens[s], L = seq_lens[s], all = n * h_r;
      if (n < 0 || L < 0 || all > INT32_MAX) return mj::set_last_error(MJ_ERR_INVALID, "mj_block_plan: a length");
      for (int64_t r = 0; r < all; r += rows) {
        const int64_t last = causal ? L - n + (std::min(r + rows, all) - 1) / h_r : L - 1;  // last key seen
        blocks.push_back({s, (int32_t)r, last < 0 ? 0 : (int32_t)(last / keys + 1)});
        total += blocks.back().tiles;
      }
    }
    std::stable_sort(blocks.begin(), blocks.end(), [](const Block& x, const Block& y) { return x.tiles > y.tiles; });
    int64_t bound = std::max<int64_t>(kMinPiece, ceil_div(total * h_k, sm_count));
    auto pieces = [&](const Block& b) { return b.tiles > bound ? ceil_div(b.tiles, bound) : 1; };
    for (;; bound *= 2) {
      int64_t slots = 0;
      for (const Block& b : blocks) slots += pieces(b) > 1 ? pieces(b) : 0;
      if (slots <= max_slots) break;
    }
    int64_t nw = 0, nm = 0, ns = 0;
    for (const Block& b : blocks) {
      const int k = pieces(b);
      if (nw + k > work_capacity || (k > 1 && nm >= merges_capacity) || !work_out || (k > 1 && !merges_out))
        return mj::set_last_error(MJ_ERR_UNSUPPORTED, "mj_block_plan: more items than the capacity");
      if (k > 1) {
        const int32_t m[4] = {b.seq, b.row0, (int32_t)ns, k};
        std::copy(m, m + 4, merges_out + 4 * nm++);
      }
      for (int i = 0; i < k; ++i) {  // pieces of equal length, to a tile
        const int32_t w[8] = {b.seq, b.row0, (int32_t)((int64_t)b.tiles * i / k), (int32_t)((int64_t)b.tiles * (i + 1) / k),
                              k > 1 ? (int32_t)ns++ : -1, 0, 0, 0};
        std::copy(w, w + 8, work_out + 8 * nw++);
      }
    }
    *num_work = (int)nw;
    *num_merges = (int)nm;
    *num_slots = (int)ns;
  } catch (const std::exception&) {
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_plan: out of memory");
  }
  return MJ_OK;
}

}  // extern "C"

// Rows of a sequence, or of a group, with the key tiles [t0, t1) that they see.
namespace {
struct SharedBlock {
  int32_t seq, row0, t0, t1, span;
  bool slotted;  // leaves partials even in one piece
  bool rest;     // P in two terms: rows that the decode kernel serves without the group
  int32_t group, pieces, slot;
};
constexpr int kMinPiece = 8;

int64_t pieces_of(const SharedBlock& b, int64_t bound) { return b.t1 - b.t0 > bound ? ceil_div(b.t1 - b.t0, bound) : 1; }

// What blocks cut in pieces of at most `bound` tiles take, in tiles of a CTA's
// time: CTAs (an item and KV head each, longest first, as many at once as there
// are SMs) a round its longest item and as much as 12 tiles for its beginning and
// end, a piece of the row that has most of them 0.3 in the join. Negative: more
// than max_slots partials.
double cost_of(const std::vector<SharedBlock>& blocks, int64_t bound, int h_k, int sm_count, int64_t max_slots,
               std::vector<int32_t>& lengths) {
  int64_t slots = 0, most = 0;
  lengths.clear();
  for (const SharedBlock& b : blocks) {
    const int64_t pieces = pieces_of(b, bound);
    slots += pieces > 1 || b.slotted ? pieces : 0;
    most = std::max(most, pieces);
    lengths.insert(lengths.end(), (size_t)pieces, ceil_div(b.t1 - b.t0, pieces));
  }
  if (slots > max_slots) return -1.0;
  std::sort(lengths.begin(), lengths.end(), std::greater<int32_t>());
  double cost = most > 1 ? 0.3 * most : 0.0;
  for (size_t first = 0; first < lengths.size() * h_k; first += sm_count) cost += lengths[first / h_k] + 12.0;
  return cost;
}

// The bound of the least cost among those that cut the longest block in 1, 2, ...
// pieces (0: none has so few partials). 64 sequences behind 16K tokens of 8 KV
// heads: 55 us with 19 pieces, two rounds on 148 SMs, 30 with 18.
int64_t best_bound(const std::vector<SharedBlock>& blocks, int h_k, int sm_count, int64_t max_slots, double* cost) {
  std::vector<int32_t> lengths;
  int64_t longest = 1, best = 0;
  for (const SharedBlock& b : blocks) longest = std::max<int64_t>(longest, b.t1 - b.t0);
  for (int64_t k = 1; k <= sm_count; ++k) {
    const int64_t bound = std::max<int64_t>(kMinPiece, ceil_div(longest, k));
    const double c = cost_of(blocks, bound, h_k, sm_count, max_slots, lengths);
    if (c < 0.0) break;  // more pieces would need no fewer
    if (!best || c < *cost) {
      best = bound;
      *cost = c;
    }
    if (bound <= kMinPiece) break;
  }
  return best;
}

// A step whose sequences share prefixes: blocks of the groups' rows first, then
// those of the sequences from decode_seqs on. Empty message: fine.
struct SharedStep {
  std::vector<SharedBlock> blocks;
  size_t of_groups = 0;
  std::vector<int32_t> group_of, start;  // of a sequence: its group or -1, its first query row
  std::vector<int64_t> place, group_rows;  // its first row's place among its group's, a group's rows
};

const char* shared_step(SharedStep& st, const int32_t* query_lens, const int32_t* seq_lens, int num_seqs, int decode_seqs,
                        const int32_t* groups, int num_groups, int h_r, int head_size, int causal) {
  const int rows = MJ_BLOCK_ROWS(head_size), keys = MJ_BLOCK_KEYS;
  st.group_of.assign(num_seqs, -1);
  st.start.assign(num_seqs + 1, 0);
  st.place.assign(num_seqs, 0);
  st.group_rows.assign(num_groups, 0);
  int64_t rows_before = 0;
  for (int s = 0; s < num_seqs; ++s) {
    if (query_lens[s] < 0 || seq_lens[s] < 0) return "a length";
    rows_before += query_lens[s];
    if (rows_before * h_r > INT32_MAX) return "a length";
    st.start[s + 1] = (int32_t)rows_before;
  }
  for (int g = 0, end = 0; g < num_groups; ++g) {
    const int32_t first = groups[3 * g], count = groups[3 * g + 1], tokens = groups[3 * g + 2];
    if (first < end || count < 1 || count > num_seqs - first || tokens <= 0 || tokens % 128) return "a group";
    end = first + count;
    for (int s = first; s < end; ++s) {
      if (query_lens[s] && (causal ? (int64_t)seq_lens[s] - query_lens[s] : seq_lens[s]) < tokens)
        return "a query before the end of its group's tokens";
      st.group_of[s] = g;
      st.place[s] = st.group_rows[g];
      st.group_rows[g] += (int64_t)query_lens[s] * h_r;
    }
    for (int64_t r = 0; r < st.group_rows[g]; r += rows) st.blocks.push_back({first, (int32_t)r, 0, tokens / keys, count, true, first < decode_seqs, g, 1, -1});
  }
  st.of_groups = st.blocks.size();
  for (int s = decode_seqs; s < num_seqs; ++s) {
    const int64_t n = query_lens[s], L = seq_lens[s], all = n * h_r;
    const int t0 = st.group_of[s] < 0 ? 0 : groups[3 * st.group_of[s] + 2] / keys;
    for (int64_t r = 0; r < all; r += rows) {
      const int64_t last = causal ? L - n + (std::min(r + rows, all) - 1) / h_r : L - 1;  // last key seen
      const int t1 = last < 0 ? 0 : (int32_t)(last / keys + 1);
      st.blocks.push_back({s, (int32_t)r, t0, std::max(t0, t1), 0, st.group_of[s] >= 0, false, -1, 1, -1});
    }
  }
  return nullptr;
}
}  // namespace

extern "C" {

int mj_block_shared_worth(const int32_t* query_lens, const int32_t* seq_lens, int num_seqs, int decode_seqs,
                          const int32_t* groups, int num_groups, int h_q, int h_k, int head_size, int causal,
                          int sm_count, int max_slots, int* worth) {
  if (num_seqs < 0 || decode_seqs < 0 || decode_seqs > num_seqs || num_groups < 0 || h_k <= 0 || h_q <= 0 || h_q % h_k ||
      (head_size != 128 && head_size != 256) || sm_count <= 0 || max_slots < 0 || (num_seqs && (!query_lens || !seq_lens)) ||
      (num_groups && !groups) || !worth)
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_shared_worth: invalid argument");
  *worth = 0;
  try {
    SharedStep with, without;
    for (int i = 0; i < 2; ++i)
      if (const char* why = shared_step(i ? with : without, query_lens, seq_lens, num_seqs, decode_seqs, groups, i ? num_groups : 0,
                                        h_q / h_k, head_size, causal)) {
        char msg[128];
        snprintf(msg, sizeof(msg), "mj_block_shared_worth: %s", why);
        return mj::set_last_error(MJ_ERR_INVALID, msg);
      }
    if (with.of_groups == 0) return MJ_OK;
    double a = 0.0, b = 0.0;
    if (!best_bound(with.blocks, h_k, sm_count, max_slots, &a)) return MJ_OK;
    int64_t total = 0;
    for (const SharedBlock& x : without.blocks) total += x.t1 - x.t0;
    std::vector<int32_t> lengths;
    if (total) b = cost_of(without.blocks, std::max<int64_t>(kMinPiece, ceil_div(total * h_k, sm_count)), h_k, sm_count, INT64_MAX, lengths);
    // In the time of a tile HBM moves 6.8 MB: of keys and values to the decode
    // kernel, of partials to and from the join, whose launch takes that of 6.
    const double row = (double)h_k * head_size / 6.8e6;
    for (int s = 0; s < decode_seqs; ++s) {
      const int g = with.group_of[s];
      b += 2 * row * seq_lens[s];
      a += 2 * row * (seq_lens[s] - (g >= 0 && query_lens[s] ? groups[3 * g + 2] : 0));
    }
    a += 6.0;
    for (int g = 0; g < num_groups; ++g) a += 2 * 4 * 2 * row * with.group_rows[g];
    *worth = a < b;
  } catch (const std::exception&) {
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_shared_worth: out of memory");
  }
  return MJ_OK;
}

int mj_block_shared_plan(const int32_t* query_lens, const int32_t* seq_lens, int num_seqs, int decode_seqs,
                         const int32_t* decode_pieces, const int32_t* groups, int num_groups, int h_q, int h_k,
                         int head_size, int causal, int sm_count, int max_slots, int32_t* work_out, int work_capacity,
                         int32_t* joins_out, int joins_capacity, int* num_work, int* num_joins, int* num_rows,
                         int* num_slots) {
  if (num_seqs < 0 || decode_seqs < 0 || decode_seqs > num_seqs || num_groups < 0 || h_k <= 0 || h_q <= 0 || h_q % h_k ||
      (head_size != 128 && head_size != 256) || sm_count <= 0 || max_slots < 0 || (num_seqs && (!query_lens || !seq_lens)) ||
      (decode_seqs && !decode_pieces) || (num_groups && !groups) || work_capacity < 0 || joins_capacity < 0 ||
      (work_capacity && !work_out) || (joins_capacity && !joins_out) || !num_work || !num_joins || !num_rows || !num_slots)
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_shared_plan: invalid argument");
  const int h_r = h_q / h_k, rows = MJ_BLOCK_ROWS(head_size);
  try {
    SharedStep st;
    if (const char* why = shared_step(st, query_lens, seq_lens, num_seqs, decode_seqs, groups, num_groups, h_r, head_size, causal)) {
      char msg[128];
      snprintf(msg, sizeof(msg), "mj_block_shared_plan: %s", why);
      return mj::set_last_error(MJ_ERR_INVALID, msg);
    }
    for (int s = 0; s < decode_seqs; ++s)
      if (decode_pieces[s] < 0) return mj::set_last_error(MJ_ERR_INVALID, "mj_block_shared_plan: decode_pieces");
    std::vector<SharedBlock>& blocks = st.blocks;
    double cost = 0.0;
    const int64_t bound = best_bound(blocks, h_k, sm_count, max_slots, &cost);
    if (!bound) return mj::set_last_error(MJ_ERR_UNSUPPORTED, "mj_block_shared_plan: more partials than max_slots");
    int64_t nw = 0, ns = 0;
    for (SharedBlock& b : blocks) {
      b.pieces = (int32_t)pieces_of(b, bound);
      nw += b.pieces;
      if (b.pieces > 1 || b.slotted) {
        b.slot = (int32_t)ns;
        ns += b.pieces;
      }
    }
    if (nw > work_capacity) return mj::set_last_error(MJ_ERR_UNSUPPORTED, "mj_block_shared_plan: more items than the capacity");
    // joins: every sequence with rows, by its own blocks
    std::vector<int32_t> shared_first(num_groups, -1), shared_pieces(num_groups, 0);
    for (size_t i = st.of_groups; i-- > 0;) {
      shared_first[blocks[i].group] = blocks[i].slot;
      shared_pieces[blocks[i].group] = blocks[i].pieces;
    }
    int64_t nj = 0, nr = 0;
    bool room = true;
    auto join = [&](int s, int64_t row0, int64_t count, int first, int pieces) {
      if (nj >= joins_capacity) {
        room = false;
        return;
      }
      const int g = st.group_of[s];
      const int32_t e[12] = {s, (int32_t)row0, (int32_t)count, (int32_t)nr, first, pieces, g < 0 ? -1 : shared_first[g],
                             g < 0 ? 0 : shared_pieces[g], g < 0 ? 0 : (int32_t)(st.place[s] + row0), st.start[s], query_lens[s], 0};
      std::copy(e, e + 12, joins_out + 12 * nj++);
      nr += count;
    };
    for (int s = 0; s < decode_seqs; ++s)
      if (query_lens[s]) join(s, 0, (int64_t)query_lens[s] * h_r, -1, decode_pieces[s]);
    for (size_t i = st.of_groups; i < blocks.size(); ++i) {
      const SharedBlock& b = blocks[i];
      if (b.slot >= 0) join(b.seq, b.row0, std::min<int64_t>(rows, (int64_t)query_lens[b.seq] * h_r - b.row0), b.slot, b.pieces);
    }
    if (!room) return mj::set_last_error(MJ_ERR_UNSUPPORTED, "mj_block_shared_plan: more joins than the capacity");
    std::stable_sort(blocks.begin(), blocks.end(), [](const SharedBlock& x, const SharedBlock& y) {
      return (int64_t)(x.t1 - x.t0) * y.pieces > (int64_t)(y.t1 - y.t0) * x.pieces;
    });
    int64_t at = 0;
    for (const SharedBlock& b : blocks)
      for (int i = 0; i < b.pieces; ++i) {  // pieces of equal length, to a tile
        const int64_t t = b.t1 - b.t0;
        const int32_t w[8] = {b.seq, b.row0, (int32_t)(b.t0 + t * i / b.pieces), (int32_t)(b.t0 + t * (i + 1) / b.pieces),
                              b.slot < 0 ? -1 : b.slot + i, b.span, b.rest, 0};
        std::copy(w, w + 8, work_out + 8 * at++);
      }
    *num_work = (int)nw;
    *num_joins = (int)nj;
    *num_rows = (int)nr;
    *num_slots = (int)ns;
  } catch (const std::exception&) {
    return mj::set_last_error(MJ_ERR_INVALID, "mj_block_shared_plan: out of memory");
  }
  return MJ_OK;
}

// ---- runner handle --------------------------------------------------------

// the tensor-core kernel's rows per job (48; 16 at head_size 256) and CTAs
// per SM (the configured count up to 16 rows at head_size 128; else one)
static int runner_n_tiles(const mj_runner* r, int q_len) {
  const int n_q = q_len * (r->h_q / r->h_k);
  const int rows = r->head_size == 256 ? 16 : 48;
  return n_q <= rows ? 1 : (n_q + rows - 1) / rows;
}
static int runner_ctas(const mj_runner* r, int q_len) {
  return q_len * (r->h_q / r->h_k) <= 16 && r->head_size == 128 ? r->ctas_per_sm : 1;
}

void mj_destroy(mj_runner* r) {
  if (!r) return;
  int prev = 0;
  cudaGetDevice(&prev);
  cudaSetDevice(r->device);
  if (r->staged) {
    cudaEventSynchronize(r->staged);
    cudaEventDestroy(r->staged);
  }
  cudaFree(r->work);
  cudaFree(r->n_splits);
  cudaFree(r->o_part);
  cudaFree(r->lse_part);
  cudaFree(r->status);
  cudaFreeHost(r->stage);
  cudaSetDevice(prev);
  delete r;
}

mj_runner* mj_create(int device, int h_q, int h_k, int head_size, int page_size, int max_num_seqs, int max_q_len,
                     int kv_format, int max_splits, int ctas_per_sm) {
  if (h_q <= 0 || h_k <= 0 || h_q % h_k || head_size <= 0 || page_size <= 0 || max_num_seqs <= 0 || max_q_len <= 0 ||
      max_splits <= 0 || ctas_per_sm <= 0 || mj_row_bytes(head_size, kv_format) < 0) {
    mj::set_last_error(MJ_ERR_INVALID, "mj_create: invalid shape or format");
    return nullptr;
  }
  if (max_q_len * (h_q / h_k) > 64) {
    mj::set_last_error(MJ_ERR_UNSUPPORTED, "mj_create: more than 64 query rows per KV head");
    return nullptr;
  }
  int prev = 0;
  cudaGetDevice(&prev);
  mj_runner* r = new mj_runner();
  r->device = device;
  r->h_q = h_q;
  r->h_k = h_k;
  r->head_size = head_size;
  r->page_size = page_size;
  r->max_num_seqs = max_num_seqs;
  r->max_q_len = max_q_len;
  r->kv_format = kv_format;
  r->max_splits = max_splits;
  r->ctas_per_sm = ctas_per_sm;
  cudaError_t e = cudaSetDevice(device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&r->sm_count, cudaDevAttrMultiProcessorCount, device);
  const int slots1 = std::max(1, (r->sm_count * runner_ctas(r, 1)) / (h_k * runner_n_tiles(r, 1)));
  r->cap = std::max(max_num_seqs * max_splits, slots1);
  const int64_t nq = (int64_t)max_q_len * (h_q / h_k);
  const int64_t rows = (int64_t)max_splits * max_num_seqs * h_k * nq;
  if (e == cudaSuccess) e = cudaMalloc(&r->work, (size_t)r->cap * 4 * sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMalloc(&r->n_splits, (size_t)max_num_seqs * sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMalloc(&r->o_part, (size_t)rows * head_size * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&r->lse_part, (size_t)rows * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&r->status, sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMemset(r->status, 0, sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMemset(r->work, 0, (size_t)r->cap * 4 * sizeof(int32_t));
  if (e == cudaSuccess) e = cudaMallocHost(&r->stage, ((size_t)r->cap * 4 + max_num_seqs) * sizeof(int32_t));
  if (e == cudaSuccess) e = cudaEventCreateWithFlags(&r->staged, cudaEventDisableTiming);
  cudaSetDevice(prev);
  if (e != cudaSuccess) {
    char msg[256];
    snprintf(msg, sizeof(msg), "mj_create: %s", cudaGetErrorString(e));
    mj::set_last_error(MJ_ERR_CUDA, msg);
    mj_destroy(r);
    return nullptr;
  }
  return r;
}

int mj_plan(mj_runner* r, const int32_t* seq_lens_host, int num_seqs, int q_len, int margin, int fixed_grid,
            void* stream) {
  if (!r || !seq_lens_host) return mj::set_last_error(MJ_ERR_INVALID, "mj_plan: null argument");
  if (num_seqs <= 0 || num_seqs > r->max_num_seqs || q_len < 1 || q_len > r->max_q_len || margin < 0)
    return mj::set_last_error(MJ_ERR_INVALID, "mj_plan: num_seqs / q_len beyond the runner's capacity");
  // the previous plan's copy must have left the staging buffer
  cudaError_t e = cudaEventSynchronize(r->staged);
  if (e != cudaSuccess) return mj::set_last_error(MJ_ERR_CUDA, cudaGetErrorString(e));
  std::vector<int32_t> lens(seq_lens_host, seq_lens_host + num_seqs);
  for (auto& L : lens) L += margin;
  int32_t* work_h = r->stage;
  int32_t* ns_h = r->stage + (size_t)r->cap * 4;
  int num_work = 0, chunk = 0;
  int rc = mj_plan_split_kv(lens.data(), num_seqs, r->h_k, runner_n_tiles(r, q_len), r->sm_count, runner_ctas(r, q_len),
                            r->max_splits, r->cap, 1, 2.0f, work_h, r->cap, ns_h, &num_work, &chunk);
  if (rc) return rc;
  int real = 0, most = 1;
  for (int i = 0; i < num_work; ++i) real += work_h[4 * i + 2] > work_h[4 * i + 1];
  for (int b = 0; b < num_seqs; ++b) most = std::max(most, (int)ns_h[b]);
  int prev = 0;
  cudaGetDevice(&prev);
  cudaSetDevice(r->device);
  cudaStream_t s = (cudaStream_t)stream;
  e = cudaMemcpyAsync(r->work, work_h, (size_t)r->cap * 4 * sizeof(int32_t), cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaMemcpyAsync(r->n_splits, ns_h, (size_t)num_seqs * sizeof(int32_t), cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaEventRecord(r->staged, s);
  cudaSetDevice(prev);
  if (e != cudaSuccess) return mj::set_last_error(MJ_ERR_CUDA, cudaGetErrorString(e));
  r->num_seqs = num_seqs;
  r->q_len = q_len;
  r->num_work = fixed_grid ? r->cap : real;
  r->with_reduction = (most > 1 || fixed_grid) ? 1 : 0;
  r->chunk_tiles = chunk;
  return MJ_OK;
}

int mj_runner_fill(const mj_runner* r, mj_decode_args* a) {
  if (!r || !a) return mj::set_last_error(MJ_ERR_INVALID, "mj_runner_fill: null argument");
  if (!r->num_seqs) return mj::set_last_error(MJ_ERR_INVALID, "mj_runner_fill: no plan yet (call mj_plan)");
  a->num_seqs = r->num_seqs;
  a->q_len = r->q_len;
  a->h_q = r->h_q;
  a->h_k = r->h_k;
  a->head_size = r->head_size;
  a->page_size = r->page_size;
  a->kv_format = r->kv_format;
  a->work = r->work;
  a->num_work = r->num_work;
  a->n_splits = r->n_splits;
  a->max_splits = r->max_splits;
  a->o_part = r->o_part;
  a->lse_part = r->lse_part;
  a->part_seqs = r->max_num_seqs;
  a->with_combine = r->with_reduction;
  a->status = r->status;
  return MJ_OK;
}

int mj_runner_status(mj_runner* r) {
  if (!r) return -mj::set_last_error(MJ_ERR_INVALID, "mj_runner_status: null runner");
  int32_t code = 0;
  int prev = 0;
  cudaGetDevice(&prev);
  cudaSetDevice(r->device);
  cudaError_t e = cudaMemcpy(&code, r->status, sizeof(int32_t), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && code) e = cudaMemset(r->status, 0, sizeof(int32_t));
  cudaSetDevice(prev);
  if (e != cudaSuccess) return -mj::set_last_error(MJ_ERR_CUDA, cudaGetErrorString(e));
  return code;
}

}  // extern "C"
