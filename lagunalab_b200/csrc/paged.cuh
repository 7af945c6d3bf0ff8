// The division of attention work over a paged K/V cache, shared by the plan and the kernels.
//
// Work is a list of segments: a row tile of queries (tokens x the G query heads of one kv head)
// against a range of 128-key tiles. A plan lists the row tiles (each stands for Hkv segments, one
// per kv head) with the cost that lies before each, and gives every CTA an equal share of the
// summed cost: CTA c takes the key tiles that start in [c, c + 1) * chunk. A CTA's share may begin
// and end inside a segment; the parts of a split segment leave partial results that a second
// kernel joins.
#pragma once

#include "common.cuh"

namespace lg {

constexpr int PA_D = 128;     // head dim
constexpr int PA_KEYS = 128;  // keys per tile
constexpr int PA_ROWS = 128;  // query rows (token, head) per row tile

enum { PA_PROMPT = 0, PA_PREFIX = 1, PA_OWN = 2 };

struct PaTile {
  int row;      // table row
  int q0, nq;   // tokens [q0, q0 + nq) of q and out
  int pos0;     // PA_PROMPT: position of token q0
  int key0;     // first key, a multiple of the page rows
  int key_end;  // one past the last key that any row sees
  int ntile;    // ceil((key_end - key0) / 128), at least 1
  int kind;
  int pair;     // 1: two row tiles (2 * tq tokens) share each key tile; 0: one row tile
  int cost;     // of one segment (one kv head)
  long long before;  // cost of all segments before this tile's first
};

struct PaStart {
  int tile, head, t;  // a CTA's first segment and key tile
};

struct PaHead {
  long long total, chunk;
  int ntile_rows, nprefix;  // row tiles, and how many of them are PA_PREFIX
  int kind, B, T, Hq, Hkv, R, prefix, window;
};

// The parts of a plan buffer.
struct PaPlan {
  PaHead* head;
  PaStart* start;  // [ncta + 1]
  int* kv;         // [B] rows of each sequence
  int* off;        // [B + 1] first row tile of each sequence (prompts)
  PaTile* tiles;   // [max_tiles]
  char* parts;     // partial results
  int ncta, max_tiles;
  size_t bytes;
};

__host__ __device__ inline int pa_tq(int Hq, int Hkv) { return PA_ROWS / (Hq / Hkv); }

}  // namespace lg
