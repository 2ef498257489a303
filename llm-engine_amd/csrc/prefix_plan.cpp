// Packing of a step for shared-prefix attention: le_prefix_plan_step /
// le_prefix_plan_upload.
//
// Sequences whose block tables begin with the same ids (the scheduler's prefix
// cache hands one prompt's blocks to all of them) share those keys. The
// tables, each cut where its sequence's own rows begin, are sorted; runs with
// a common beginning form a tree (their longest common prefixes are nested),
// and the groups are the cut through it that saves the most block reads. A
// group's shared keys are attended by all rows of its sequences at once, in
// tiles of query columns (row, head); what follows them by each sequence's
// rows alone. Every tile's keys are cut into partitions, one work item each.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <new>
#include <unordered_map>
#include <vector>

#include "le_internal.h"
#include "llm_engine_amd.h"

namespace {

using le::PrefixItem;
using le::PrefixRow;

constexpr int kMinSharedKeys = 64;    // a shorter common beginning is not worth a pass of its own
constexpr int kMaxParts = 128;        // partitions of a tile
constexpr int kCus = 256;             // MI355X
constexpr int kWideCost = 2;          // time of a wide tile's keys, in narrow ones
constexpr int kShortOwn = 256;        // keys of a sequence that few columns attend in narrow tiles
constexpr int kSoloKeys = 32;         // keys of a narrow item up to which a wave takes it alone (twice: in a very full step)
constexpr int kExtra = 6;             // time of a 16-bit workgroup around its tiles, in LDS tiles
constexpr int kMinF32 = 4;            // LDS tiles of an fp32 item that is not narrow, at least
constexpr int kSmallF32 = 256;        // LDS tiles of wide fp32 items up to which narrow ones take their place

int64_t align256(int64_t x) { return (x + 255) & ~static_cast<int64_t>(255); }

// the number of ids, up to n, that two tables begin with alike
int common(const int32_t* a, const int32_t* b, int n) {
  constexpr int kRun = 64;
  int i = 0;
  while (i + kRun <= n && std::memcmp(a + i, b + i, kRun * sizeof(int32_t)) == 0) i += kRun;
  while (i < n && a[i] == b[i]) i++;
  return i;
}

struct Group {
  int first, count;  // among the sorted slices
  int blocks;        // shared blocks
};

// The groups of sorted tables with common beginnings lcp[i] (of i - 1 and i).
// One pass with a stack of open runs; a closed run is worth its shared blocks
// times the sequences that need not read them, or what its inner runs are.
std::vector<Group> best_groups(const std::vector<int>& lcp, int min_blocks) {
  struct Run {
    int v, first, last;
    int64_t best;
    bool whole;
    std::vector<int> inner;
  };
  const int n = static_cast<int>(lcp.size());
  std::vector<Run> runs;  // closed ones, inner before outer
  std::vector<Run> open{Run{0, 0, 0, 0, false, {}}};
  for (int i = 1; i <= n; i++) {
    const int v = i < n ? lcp[i] : 0;
    int first = i - 1, closed = -1;
    while (v < open.back().v) {
      Run r = std::move(open.back());
      open.pop_back();
      r.last = i - 1;
      int64_t inside = 0;
      for (int k : r.inner) inside += runs[k].best;
      const int64_t all = r.v >= min_blocks ? static_cast<int64_t>(r.v) * (r.last - r.first) : 0;
      r.whole = all > 0 && all >= inside;
      r.best = std::max(all, inside);
      first = r.first;
      closed = static_cast<int>(runs.size());
      runs.push_back(std::move(r));
      if (v <= open.back().v) {
        open.back().inner.push_back(closed);
        closed = -1;
      }
    }
    if (v > open.back().v) {
      Run r{v, first, 0, 0, false, {}};
      if (closed >= 0) r.inner.push_back(closed);
      open.push_back(std::move(r));
    }
  }
  std::vector<Group> groups;
  std::vector<int> todo = open.front().inner;
  while (!todo.empty()) {
    const Run& r = runs[todo.back()];
    todo.pop_back();
    if (r.whole) groups.push_back(Group{r.first, r.last - r.first + 1, r.v});
    else todo.insert(todo.end(), r.inner.begin(), r.inner.end());
  }
  return groups;
}

// The LDS tiles (64 keys) of a partition: the fewest with which tiles of
// lengths `len` make at most `slots` workgroups (whole ones where they are more
// anyway).
int64_t part_tiles(const std::vector<int64_t>& len, int kv_heads, int64_t slots) {
  int64_t work = 0, most = 1;
  for (int64_t n : len) {
    work += n * kv_heads;
    most = std::max(most, n);
  }
  if (static_cast<int64_t>(len.size()) * kv_heads >= slots) return most;
  int64_t t = std::max<int64_t>(1, work / slots);
  for (; t < most; t += std::max<int64_t>(1, t / 16)) {
    int64_t n = 0;
    for (int64_t x : len) n += (x + t - 1) / t * kv_heads;
    if (n <= slots) break;
  }
  return std::min(t, most);
}

// The same of tiles whose products count: the partition with which the rounds of
// `slots` workgroups, each as long as a partition and the time of `extra` LDS
// tiles around it, end first. (2 x 315 rows behind 10624 keys, 32/4 heads x 64:
// 100 us in three rounds, 164 in one that fills 160 of 256 places.)
int64_t round_tiles(const std::vector<int64_t>& len, int kv_heads, int64_t slots, int64_t extra) {
  int64_t work = 0, most = 1;
  for (int64_t n : len) {
    work += n * kv_heads;
    most = std::max(most, n);
  }
  int64_t best = most, least = INT64_MAX;
  for (int64_t t = std::max<int64_t>(1, work / (8 * slots));; t += std::max<int64_t>(1, t / 16)) {
    t = std::min(t, most);
    int64_t n = 0;
    for (int64_t x : len) n += (x + t - 1) / t * kv_heads;
    const int64_t time = (n + slots - 1) / slots * (t + extra);
    if (time <= least) {
      least = time;
      best = t;
    }
    if (t == most) return best;
  }
}

struct Tile {
  std::vector<int32_t> rows;
  int32_t ids_off;  // block id of key_begin
  int32_t key_begin, key_end;
  bool causal;
  int part_first;  // index of its first partition among those of its rows
  int parts;
};

int plan_step(const le_step_slice* slices, int n_slices, const le_plan_config* cfg_in, void* host_buf,
              int64_t host_cap, le_prefix_plan* plan) {
  if (!plan || !cfg_in || n_slices < 0 || (n_slices > 0 && !slices)) return LE_EINVAL;
  const le_plan_config& cfg = *cfg_in;
  const int shape = le::check_attention_shape(cfg.q_heads, cfg.kv_heads, cfg.head_dim, cfg.block_size);
  if (shape != LE_OK) return shape;
  if (cfg.kv_dtype != LE_F32 && cfg.kv_dtype != LE_BF16 && cfg.kv_dtype != LE_F16) return LE_EINVAL;
  if (cfg.partition_tokens < 0 || cfg.chunk_partition_tokens < 0 || cfg.flags != 0 || cfg.table_capacity != 0) return LE_EINVAL;
  if (cfg.chunk_q_tile != 0 && cfg.chunk_q_tile != le::kPrefixNarrow && cfg.chunk_q_tile != le::kPrefixCols)
    return LE_EINVAL;
  const int bs = cfg.block_size, G = cfg.q_heads / cfg.kv_heads;

  // ---- validation; a key's slices use its first one's table, as le_plan_step's do ----
  int64_t n_tok = 0;
  std::unordered_map<int64_t, int> seen;
  std::vector<const le_step_slice*> table(n_slices);
  for (int i = 0; i < n_slices; i++) {
    const le_step_slice& s = slices[i];
    if (s.len <= 0 || s.start < 0 || s.num_blocks < 0 || s.len > INT32_MAX - s.start) return LE_EINVAL;
    if (s.start + s.len > INT32_MAX - 4096) return LE_EUNSUPPORTED;  // a kernel counts on to the end of a tile
    if (s.num_blocks > 0 && !s.blocks) return LE_EINVAL;
    table[i] = &slices[seen.emplace(s.seq_key, i).first->second];
    if ((s.start + s.len - 1) / bs >= table[i]->num_blocks) return LE_EINVAL;  // a position without a block
    n_tok += s.len;
  }
  if (n_tok > INT32_MAX / 2) return LE_EUNSUPPORTED;
  std::vector<int32_t> first_row(n_slices);
  std::vector<int32_t> positions(static_cast<size_t>(n_tok));
  for (int i = 0, t = 0; i < n_slices; i++) {
    first_row[i] = t;
    for (int j = 0; j < slices[i].len; j++) positions[t++] = slices[i].start + j;
  }

  // ---- groups ----
  // whole blocks before a slice's first row: every key in them is visible to
  // all its rows, and at least one key is left behind them
  std::vector<int> cap(n_slices), order(n_slices);
  for (int i = 0; i < n_slices; i++) {
    cap[i] = slices[i].start / bs;
    order[i] = i;
  }
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
    const int m = std::min(cap[a], cap[b]), at = common(table[a]->blocks, table[b]->blocks, m);
    return at < m ? table[a]->blocks[at] < table[b]->blocks[at] : cap[a] < cap[b];
  });
  std::vector<int> lcp(n_slices, 0);
  for (int i = 1; i < n_slices; i++) {
    const int a = order[i - 1], b = order[i];
    lcp[i] = common(table[a]->blocks, table[b]->blocks, std::min(cap[a], cap[b]));
  }
  const std::vector<Group> groups = best_groups(lcp, std::max(1, (kMinSharedKeys + bs - 1) / bs));

  // ---- tiles: shared keys by a group's rows, then every slice's own keys ----
  std::vector<int32_t> ids;
  std::vector<Tile> tiles;
  std::vector<int> shared(n_slices, 0);       // keys of the slice that its group reads
  auto add_tiles = [&](const std::vector<int32_t>& rows, int32_t ids_off, int begin, bool causal, int end) {
    const int n = static_cast<int>(rows.size());
    // fp32 products take 3.6 us per 64 keys (head_dim 64) in a wide tile and
    // 0.9 in a narrow one: a step too small to fill the chip with wide ones is
    // cut into narrow ones (24 rows behind 1500 keys, 14/2 heads x 64: 11.3 us
    // against 25; 128 rows behind 4096: 59 against 31).
    const int64_t wide_tiles = static_cast<int64_t>((n * G + le::kPrefixCols - 1) / le::kPrefixCols) * cfg.kv_heads *
                               ((end - begin + le::kPrefixTileKeys - 1) / le::kPrefixTileKeys);
    const bool small_f32 = cfg.kv_dtype == LE_F32 && wide_tiles <= kSmallF32;
    // A sequence's 33 to 64 columns would leave half of a wide tile's waves
    // idle: over a few keys two narrow tiles are quicker (48 sequences of up to
    // 8 rows behind 2000 keys, 28/4 heads x 128, own keys 8 to 700: 31 us, 35
    // as wide ones; up to 1024 keys narrow, 33).
    const bool few = causal && n * G <= 2 * le::kPrefixNarrow && end - begin <= kShortOwn;
    const int tile_rows = (cfg.chunk_q_tile > 0 ? cfg.chunk_q_tile : small_f32 || few ? le::kPrefixNarrow : le::kPrefixCols) / G;
    const int count = (n + tile_rows - 1) / tile_rows;
    for (int k = 0; k < count; k++) {
      const int a = static_cast<int>(static_cast<int64_t>(k) * n / count);
      const int b = static_cast<int>(static_cast<int64_t>(k + 1) * n / count);
      // a causal tile's keys end with its last row's own
      const int e = causal ? positions[rows[b - 1]] + 1 : end;
      tiles.push_back(Tile{std::vector<int32_t>(rows.begin() + a, rows.begin() + b), ids_off, begin, e, causal, 0, 1});
    }
  };
  for (size_t g = 0; g < groups.size(); g++) {
    const Group& gr = groups[g];
    std::vector<int32_t> rows;
    for (int k = 0; k < gr.count; k++) {
      const int i = order[gr.first + k];
      shared[i] = gr.blocks * bs;
      for (int j = 0; j < slices[i].len; j++) rows.push_back(first_row[i] + j);
    }
    std::sort(rows.begin(), rows.end());
    const int32_t off = static_cast<int32_t>(ids.size());
    const int32_t* t = table[order[gr.first]]->blocks;
    ids.insert(ids.end(), t, t + gr.blocks);
    add_tiles(rows, off, 0, false, gr.blocks * bs);
  }
  for (int i = 0; i < n_slices; i++) {
    std::vector<int32_t> rows(slices[i].len);
    for (int j = 0; j < slices[i].len; j++) rows[j] = first_row[i] + j;
    const int32_t off = static_cast<int32_t>(ids.size());
    const int b0 = shared[i] / bs, b1 = (slices[i].start + slices[i].len - 1) / bs + 1;
    ids.insert(ids.end(), table[i]->blocks + b0, table[i]->blocks + b1);
    add_tiles(rows, off, shared[i], true, slices[i].start + slices[i].len);
  }
  if (ids.size() > INT32_MAX / 2) return LE_EUNSUPPORTED;

  // ---- partitions ----
  // Tiles of more than kPrefixNarrow columns are bound by their products and
  // the chain of a tile's steps, the others by their keys' bytes; a CU holds
  // two workgroups. So the wide ones are cut to one a CU, beside which the
  // narrow ones stream (256 rows behind 16384 keys, 32/8 heads x 128, and 64 to
  // 1024 keys of their own: 174 us, with two a CU 208), or to two where the
  // narrow ones are few (122 rows after 131072 keys: 327 us, with one a CU 431).
  // The narrow ones are cut to the places left (64 rows behind 4096 keys and 16
  // to 512 of their own, 14/2 heads x 64: 12.9 us, uncut 14.8), with
  // an fp32 cache, whose products count here too, to one a CU (24 rows behind
  // 1500 keys 11.3 us, in parts twice as long 14.0), but not where they fill the
  // chip as they are, up to 1024 keys (48 sequences of 5 to 700 keys, 8 kv
  // heads: 18.9 us, cut at 512 keys 22.8).
  // Wide fp32 tiles of head_dim 64, two a CU, hide each other's softmax (3 x 220
  // rows behind 5200 keys, 12 heads: 129 us, one a CU 145), from 256 keys on (30
  // rows behind 8192, 32/4 heads: 32 us, cut at 128 keys 37); of head_dim 128
  // one fits.
  const int quantum = std::max(le::kPrefixTileKeys, bs);
  const int64_t places = cfg.kv_dtype == LE_F32 && cfg.head_dim > 64 ? kCus : 2 * kCus;  // workgroups at once
  auto wide = [&](const Tile& t) { return static_cast<int>(t.rows.size()) * G > le::kPrefixNarrow; };
  // Narrow tiles of shared keys (kind 2) are few and long beside the sequences'
  // own ones, and cut apart from them (4 x 10 sequences of up to 4 rows behind
  // 1184 keys and 3 of their own, 12 heads x 64: 12 us, together 24).
  auto kind = [&](const Tile& t) { return wide(t) ? 1 : t.causal ? 0 : 2; };
  std::vector<int64_t> len[3];
  int64_t work[3] = {0, 0, 0};
  for (const Tile& t : tiles) {
    len[kind(t)].push_back((t.key_end - t.key_begin + le::kPrefixTileKeys - 1) / le::kPrefixTileKeys);
    work[kind(t)] += len[kind(t)].back();
  }
  const bool f32 = cfg.kv_dtype == LE_F32;
  int64_t part[3];
  auto workgroups = [&](int k) {
    int64_t n = 0;
    for (int64_t x : len[k]) n += (x + part[k] - 1) / part[k] * cfg.kv_heads;
    return n;
  };
  part[1] = round_tiles(len[1], cfg.kv_heads,
                        (work[0] + work[2]) * 8 < work[1] || (f32 && cfg.head_dim == 64) ? places : kCus,
                        f32 ? kExtra / 2 : kExtra);
  if (f32) part[1] = std::max<int64_t>(part[1], kMinF32);
  const int64_t own = static_cast<int64_t>(len[0].size()) * cfg.kv_heads;
  const int64_t left = f32 ? kCus - std::min<int64_t>(workgroups(1), kCus / 2)
                           : 2 * kCus - std::min<int64_t>(workgroups(1), kCus);
  part[2] = part_tiles(len[2], cfg.kv_heads, std::max(left - own, left / 2));
  part[0] = part_tiles(len[0], cfg.kv_heads, std::max<int64_t>(left - workgroups(2), 1));
  if (own >= kCus) part[0] = std::max<int64_t>(part[0], 16);
  for (int k = 0; k < 3; k++) {
    const int asked = k == 1 ? cfg.chunk_partition_tokens : cfg.partition_tokens;
    part[k] = asked > 0 ? asked : part[k] * le::kPrefixTileKeys;
    part[k] = (part[k] + quantum - 1) / quantum * quantum;
  }
  std::vector<int32_t> n_parts(static_cast<size_t>(n_tok), 0), part0(static_cast<size_t>(n_tok), 0);
  int64_t n_items = 0;
  for (Tile& t : tiles) {
    const int64_t units = (t.key_end - t.key_begin + quantum - 1) / quantum;
    t.parts = static_cast<int>(std::min<int64_t>(kMaxParts, (units * quantum + part[kind(t)] - 1) / part[kind(t)]));
    t.part_first = n_parts[t.rows[0]];
    for (int32_t r : t.rows) n_parts[r] += t.parts;
    n_items += t.parts;
  }
  int64_t n_records = 0;
  for (int64_t r = 0; r < n_tok; r++) {
    part0[r] = static_cast<int32_t>(n_records);
    if (n_parts[r] > 1) n_records += n_parts[r];
  }
  if (n_records > INT32_MAX / 2 || n_items * cfg.kv_heads > INT32_MAX) return LE_EUNSUPPORTED;

  // ---- items, the longest to run first ----
  struct Placed {
    PrefixItem item;
    const Tile* tile;
  };
  std::vector<Placed> items;
  items.reserve(static_cast<size_t>(n_items));
  int rows_stride = 1, ids_stride = 1;
  for (const Tile& t : tiles) {
    const int64_t units = (t.key_end - t.key_begin + quantum - 1) / quantum;
    const bool split = n_parts[t.rows[0]] > 1;
    rows_stride = std::max(rows_stride, static_cast<int>(t.rows.size()));
    for (int k = 0; k < t.parts; k++) {
      PrefixItem it{};
      it.n_rows = static_cast<int32_t>(t.rows.size());
      const int a = static_cast<int>(k * units / t.parts) * quantum, b = static_cast<int>((k + 1) * units / t.parts) * quantum;
      it.key_begin = t.key_begin + a;
      it.key_end = static_cast<int32_t>(std::min<int64_t>(static_cast<int64_t>(t.key_begin) + b, t.key_end));
      it.ids_off = t.ids_off + a / bs;
      it.part = split ? t.part_first + k : -1;
      it.causal = t.causal ? 1 : 0;
      ids_stride = std::max(ids_stride, std::min(le::kPrefixListIds, (it.key_end - it.key_begin + bs - 1) / bs));
      items.push_back(Placed{it, &t});
    }
  }
  auto cost = [&](const Placed& a) { return static_cast<int64_t>(a.item.key_end - a.item.key_begin) * (wide(*a.tile) ? kWideCost : 1); };
  std::stable_sort(items.begin(), items.end(), [&](const Placed& a, const Placed& b) { return cost(a) > cost(b); });
  // Where there are more workgroups than places, a sequence's item of a few keys
  // is given to one wave: alone it would keep four waves for the time of a few trips to
  // memory (256 rows behind 512 keys and 1 to 30 of their own, 32/8 heads x 128:
  // 23 us, 33 without; 234 rows behind 80 and 3, fp32, 32/4 x 64: 15, 21; where
  // they all fit it is slower: 4 rows behind 512 keys and 8 to 100, 10.0 us
  // against 7.9). From twice the places on items of up to 64 keys too (186 fp32
  // rows of 35 keys, 10 heads x 128: 22 us, 43; at 1.25 times, 4 x 32 rows with
  // up to 200, 13.2 us, 12.7).
  const int64_t load = n_items * cfg.kv_heads / places;
  const int solo_keys = load >= 2 ? 2 * kSoloKeys : n_items * cfg.kv_heads > places ? kSoloKeys : 0;
  auto solo = [&](const Placed& a) { return kind(*a.tile) == 0 && a.item.key_end - a.item.key_begin <= solo_keys; };
  const auto first_solo = std::stable_partition(items.begin(), items.end(), [&](const Placed& a) { return !solo(a); });

  // ---- layout and copy ----
  le_prefix_plan out{};
  out.cfg = cfg;
  out.n_tokens = static_cast<int32_t>(n_tok);
  out.n_slices = n_slices;
  out.n_groups = static_cast<int32_t>(groups.size());
  out.n_items = static_cast<int32_t>(n_items);
  out.n_parts = static_cast<int32_t>(n_records);
  for (const Group& g : groups) out.saved_keys += static_cast<int64_t>(g.blocks) * bs * (g.count - 1);
  int64_t at = 0;
  auto place = [&](int64_t& off, size_t bytes) {
    off = at;
    at = align256(at + static_cast<int64_t>(bytes));
  };
  out.rows_stride = rows_stride;
  out.ids_stride = ids_stride;
  out.n_solo = static_cast<int32_t>(items.end() - first_solo);
  const size_t n = items.size();
  place(out.off_items, n * sizeof(PrefixItem));
  place(out.off_rows, n * rows_stride * sizeof(PrefixRow));
  place(out.off_item_ids, n * ids_stride * 4);
  place(out.off_ids, ids.size() * 4);
  place(out.off_part0, part0.size() * 4);
  place(out.off_row_parts, n_parts.size() * 4);
  out.bytes = at;
  *plan = out;
  if (out.bytes == 0) return LE_OK;
  if (!host_buf || host_cap < out.bytes) return LE_ENOSPACE;
  char* dst = static_cast<char*>(host_buf);
  PrefixItem* to_items = reinterpret_cast<PrefixItem*>(dst + out.off_items);
  PrefixRow* to_rows = reinterpret_cast<PrefixRow*>(dst + out.off_rows);
  int32_t* to_ids = reinterpret_cast<int32_t*>(dst + out.off_item_ids);
  for (size_t i = 0; i < n; i++) {
    const PrefixItem& it = items[i].item;
    to_items[i] = it;
    const std::vector<int32_t>& r = items[i].tile->rows;
    for (int k = 0; k < rows_stride; k++) {
      const int32_t t = r[std::min<size_t>(k, r.size() - 1)];
      to_rows[i * rows_stride + k] = PrefixRow{t, positions[t], part0[t], 0};
    }
    const int last = (it.key_end - it.key_begin - 1) / bs;
    for (int k = 0; k < ids_stride; k++) to_ids[i * ids_stride + k] = ids[it.ids_off + std::min(k, last)];
  }
  auto put = [&](int64_t off, const std::vector<int32_t>& v) {
    if (!v.empty()) std::memcpy(dst + off, v.data(), v.size() * 4);
  };
  put(out.off_ids, ids);
  put(out.off_part0, part0);
  put(out.off_row_parts, n_parts);
  return LE_OK;
}

}  // namespace

extern "C" {

int le_prefix_plan_step(const le_step_slice* slices, int n_slices, const le_plan_config* cfg, void* host_buf,
                        int64_t host_cap, le_prefix_plan* plan) {
  try {
    return plan_step(slices, n_slices, cfg, host_buf, host_cap, plan);
  } catch (...) {  // out of host memory
    return LE_ENOSPACE;
  }
}

int le_prefix_plan_upload(le_prefix_plan* plan, const void* host_buf, void* dev_buf, hipStream_t stream) {
  if (!plan || plan->bytes < 0) return LE_EINVAL;
  if (plan->bytes > 0) {
    if (!host_buf || !dev_buf) return LE_EINVAL;
    const hipError_t e =
        hipMemcpyAsync(dev_buf, host_buf, static_cast<size_t>(plan->bytes), hipMemcpyHostToDevice, stream);
    if (e != hipSuccess) return static_cast<int>(e);
  }
  plan->dev = dev_buf;
  return LE_OK;
}

}  // extern "C"
