// The division of attention work over a paged K/V cache, shared by the plan and the kernels.
//
// Work is a list of segments: a row tile of queries (tokens x the G query heads of one kv head)
// against a range of 128-key tiles. A plan lists the row tiles (each stands for Hkv segments, one
// per kv head) with the cost that lies before each, and gives every CTA an equal share of the
// summed cost: CTA c takes the key tiles whose cost begins in [c, c + 1) * chunk. A CTA's share may
// begin and end inside a segment; the parts of a split segment leave partial results that a second
// kernel joins.
#pragma once

#include "common.cuh"

namespace lg {

constexpr int PA_D = 128;     // head dim
constexpr int PA_KEYS = 128;  // keys per tile
constexpr int PA_ROWS = 128;  // query rows (token, head) per row tile

enum { PA_PROMPT = 0, PA_PREFIX = 1, PA_OWN = 2 };
constexpr int PA_MISFIT = 10;  // beside the codes of waits, 1 to 9

struct PaTile {
  int row;      // table row
  int q0, nq;   // tokens [q0, q0 + nq) of q and out
  int pos0;     // PA_PROMPT: position of token q0
  int key0;     // first key, a multiple of the page rows
  int key_end;  // one past the last key that any row sees
  int ntile;    // key tiles: ceil((key_end - key0) / 128), at least 1
  int ntile0;   // pair: key tiles of the first row tile (at most ntile)
  int kind;
  int pair;  // 1: two row tiles (2 * tq tokens) share each key tile
  int duo;   // 1: the same tokens' row tiles of two neighbouring kv heads, each with its own key
             // tiles; neither (an odd number of kv heads): one row tile, its key tiles in halves
  int w;     // cost of a key tile (of both heads')
  long long before;  // cost of all segments before this tile's first
};

// Costs: a row tile on one key tile is 2, so a key tile of two row tiles is 4 (2.2 us). A stream's
// own key tile is 2 as well: its few rows leave most of the softmax out, its loads are HBM's (3: 80
// against 71 us on 128 streams with a 16,384-row prefix). Every segment costs PA_SEG more (Q load,
// first score, output; 8: 156 against 153 us on 16 ragged prompts, 2: 205).
constexpr int PA_W_TWO = 4, PA_W_ONE = 2, PA_W_OWN = 2, PA_SEG = 6;
constexpr int PA_MIN_CHUNK = 10;  // at least the largest PA_SEG + w: no CTA below the last is idle

__host__ __device__ inline long long pa_cost(int ntile, int w) {
  return PA_SEG + (long long)ntile * w;
}

// A row tile stands for Hkv segments, or Hkv / 2 of two heads; head: a segment's first.
__host__ __device__ inline int pa_segments(const PaTile& t, int Hkv) { return Hkv >> t.duo; }

struct PaStart {
  int tile, head, t;  // a CTA's first segment and key tile
  int pad;
  PaTile rec;  // that tile's record, so that a CTA has it with the first load
};

struct alignas(16) PaHead {
  long long total, chunk;
  int kind, B, T, Hq;  // two 16-byte loads, see pa_fits
  int Hkv, R, prefix, window;
  int ntiles;  // row tiles
  int err;     // a wait that ran out (its code), else 0: ends the others' waits
  int misfit;  // PA_MISFIT after a call of other sizes, which did nothing
};

// The parts of a plan buffer.
struct PaPlan {
  PaHead* head;
  PaStart* start;  // [ncta + 1]
  int* kv;         // [B] rows of each sequence
  int* off;        // [B + 1] first row tile of each sequence (prompts)
  PaTile* tiles;   // [max_tiles]
  // partial results: per slot, {m, l} of every row, then o as [32 column quads][rows][4]
  float* wide;  // slots of 2 * PA_ROWS rows (prompts, prefixes)
  float* own;   // slots of G rows (streams' own keys)
  int ncta, max_tiles;
  int nprefix;  // streams: row tiles kept for the prefix, before the streams' own
  size_t bytes;
};

constexpr int PA_WIDE_ROWS = 2 * PA_ROWS;

__host__ __device__ inline size_t pa_slot_floats(int rows) { return (size_t)rows * (2 + PA_D); }

// Rows of a slot for a stream's own keys: G, even, so that slots stay 16-byte aligned.
__host__ __device__ inline int pa_own_rows(int Hq, int Hkv) { return (Hq / Hkv + 1) & ~1; }

// The slot of a stream's own keys for one head in the part of CTA c: parts in order, segment + CTA,
// with two slots a part when its segments have two heads.
__host__ __device__ inline size_t pa_own_slot(int b, int head, int c, int Hkv) {
  return Hkv & 1 ? (size_t)b * Hkv + head + c
                 : ((size_t)b * (Hkv >> 1) + (head >> 1) + c) * 2 + (head & 1);
}

__host__ __device__ inline int pa_tq(int Hq, int Hkv) { return PA_ROWS / (Hq / Hkv); }

}  // namespace lg
