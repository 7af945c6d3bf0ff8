// Page operations of a paged K/V cache: reserve, fork, free and compact.
//
// A cache of `planes` planes (a layer's K or V each) holds P pages per plane; page p of every
// plane belongs together, so one table row names a stream's pages for the whole model. State on
// the device: table int32 [S, M] (page ids from column 0 on, -1 past them), lens int32 [S] (rows
// held), refs int32 [P] (streams that name the page; 0: free).
//
// Each operation is a one-CTA kernel that checks its arguments and takes pages, and where rows
// move a grid-wide kernel that carries the moves out. An operation whose check fails changes
// nothing and says why in status[0]. Pages are always taken lowest id first, in the order of the
// call's list, so the result does not depend on timing.
//
// Bounds: the moves read and write each row once, 16 bytes a lane, so they run at the copy rate of
// HBM (118 pages of 80 planes moved: 192 us, 6.4 TB/s); the one-CTA kernels are latency (a scan of
// refs, of the call's list and of the sources' table rows: a fork of 3 streams 8.5 us with the free
// before it, 8.1 without a look at the sources' whole pages), and the moving kernel's launch passes
// under them. Times here are graph replays; calls in a row of 64 children take 57 us for 49.
//
// A fork's copies are written plane by plane in the order of their pages. Reading a page once for
// all its copies instead left the reads 26 MB of 228, but the writes jumped between pages: 62 us
// against 49 for 64 children of 80 planes (202 MB written, 40 us in the moving kernel).
#include <algorithm>

#include "common.cuh"

namespace lg {

enum { PG_OK = 0, PG_NO_PAGES = 1, PG_BAD_STREAM = 2, PG_TABLE_FULL = 3, PG_BAD_PAGE = 4 };

constexpr int PG_THREADS = 1024;
constexpr int PG_MAX_STREAMS = 65536;  // the duplicate check's bitmap: 8 KiB of shared memory

// The moves of one operation, in the caller's workspace: page from[i] -> to[i], rows[i] rows.
struct Moves {
  int* count;
  int* from;
  int* to;
  int* rows;
  int* of;  // fork: child i's move, -1 without one
};

inline Moves moves_of(void* ws, int n) {
  int* w = static_cast<int*>(ws);
  return {w, w + 64, w + 64 + n, w + 64 + 2 * n, w + 64 + 3 * n};
}

// Every id of the list in [0, S) and none twice (bitmap bm, S bits); the whole CTA calls it.
__device__ bool list_ok(const int* ids, int n, int S, unsigned* bm, int* bad) {
  for (int i = threadIdx.x; i < (S + 31) / 32; i += blockDim.x) bm[i] = 0;
  if (threadIdx.x == 0) *bad = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = ids[i];
    if (s < 0 || s >= S || (atomicOr(&bm[s >> 5], 1u << (s & 31)) >> (s & 31) & 1)) *bad = 1;
  }
  __syncthreads();
  const bool ok = *bad == 0;
  __syncthreads();
  return ok;
}

// The first `need` free pages in ascending order into out[]; returns how many there are (at most
// need, or the free count when less). The whole CTA calls it; need is CTA-uniform; ref0 is page
// threadIdx.x's count, which the caller fetched early.
__device__ int take_free(const int* refs, int P, int need, int ref0, int* out, int* wt, int* tot) {
  int have = 0;
  for (int p0 = 0; p0 < P && have < need; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int v = p < P && (p0 == 0 ? ref0 : refs[p]) == 0;
    const int r = have + block_excl_scan(v, wt, tot);
    if (v && r < need) out[r] = p;
    have += *tot;
    __syncthreads();
  }
  return have < need ? have : need;
}

__global__ void __launch_bounds__(PG_THREADS)
    pages_reserve_kernel(int* table, int* refs, int S, int M, int P, int R, const int* ids,
                         const int* rows, int n, int* list, int* status) {
  __shared__ unsigned bm[PG_MAX_STREAMS / 32];
  __shared__ int bad, wt[32], tot, code;
  __shared__ unsigned long long asked;  // pages in all: the sums in 32 bits hold only up to P
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* first = list + P;  // [n + 1]: where each stream's new pages start in the list
  int* have = first + n + 1;
  const int ref0 = threadIdx.x < P ? refs[threadIdx.x] : 1;
  const bool ok = list_ok(ids, n, S, bm, &bad);
  if (threadIdx.x == 0) code = ok ? PG_OK : PG_BAD_STREAM, asked = 0;
  __syncthreads();
  if (!ok) {
    if (threadIdx.x == 0) status[0] = PG_BAD_STREAM, status[1] = 0;
    return;
  }
  for (int i = warp; i < n; i += PG_THREADS / 32) {  // pages the stream has: its leading entries
    int h = 0;
    const int* row = table + (size_t)ids[i] * M;
    for (int m0 = 0; m0 < M; m0 += 32) {
      const unsigned b = __ballot_sync(0xffffffffu, m0 + lane < M && row[m0 + lane] >= 0);
      h += __popc(b);
      if (b != 0xffffffffu) break;
    }
    if (lane == 0) have[i] = h;
  }
  __syncthreads();
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      if (rows[i] < 0 || rows[i] > (long long)M * R) code = PG_TABLE_FULL;
      else need = max(0, rows[i] / R + (rows[i] % R > 0) - have[i]);
    }
    unsigned long long all = need;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0 && all) atomicAdd(&asked, all);
    const int at = total + block_excl_scan(need, wt, &tot);
    if (i < n) first[i] = at;
    total += tot;
    __syncthreads();
  }
  if (threadIdx.x == 0) first[n] = total;
  const bool fit = asked <= (unsigned long long)P;  // then total is the sum
  if (code == PG_OK && (total > 0 || !fit)) {  // code is CTA-uniform here: written before a barrier
    const int got = fit ? take_free(refs, P, total, ref0, list, wt, &tot) : 0;
    if ((!fit || got < total) && threadIdx.x == 0) code = PG_NO_PAGES;
  }
  __syncthreads();
  if (code == PG_OK)
    for (int k = threadIdx.x; k < total; k += blockDim.x) {
      int lo = 0, hi = n - 1;  // the last stream whose pages start at or before k
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= k) lo = mid;
        else hi = mid - 1;
      }
      table[(size_t)ids[lo] * M + have[lo] + k - first[lo]] = list[k];
      refs[list[k]] = 1;
    }
  if (threadIdx.x == 0) {
    status[0] = code;
    status[1] = code == PG_OK ? total : 0;
  }
}

__global__ void __launch_bounds__(PG_THREADS)
    pages_free_kernel(int* table, int* lens, int* refs, int S, int M, int P, const int* ids, int n,
                      int* status) {
  __shared__ unsigned bm[PG_MAX_STREAMS / 32];
  __shared__ int bad;
  // every CTA checks the list for itself, then takes its share of the entries
  if (!list_ok(ids, n, S, bm, &bad)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) status[0] = PG_BAD_STREAM, status[1] = 0;
    return;
  }
  const long long all = (long long)n * M;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < all;
       e += (long long)gridDim.x * blockDim.x) {
    int* at = table + (size_t)ids[e / M] * M + e % M;
    const int p = *at;
    if (p >= 0) {
      *at = -1;
      if (p < P) atomicSub(refs + p, 1);
    }
    if (e % M == 0) lens[ids[e / M]] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) status[0] = PG_OK, status[1] = n;
}

__global__ void __launch_bounds__(PG_THREADS)
    pages_fork_plan_kernel(const int* table, const int* lens, int* refs, int S, int M, int P, int R,
                           const int* src, const int* dst, int n, Moves mv, int* status) {
  __shared__ unsigned bm[PG_MAX_STREAMS / 32];
  __shared__ int bad, wt[32], tot;
  __shared__ int faults;  // a bit a code; the lowest is told, whichever thread saw its own first
  // this turn's sources whose pages are looked at, their whole and part-filled pages, and the most
  __shared__ int look[PG_THREADS], pages[PG_THREADS], nlook, most;
  pdl_trigger();  // the moving kernel waits for this one itself
  // What the first children's checks and the search for free pages read is fetched before the
  // list's check: this kernel's time is that of its loads one after the other.
  struct Child {
    int s, d, before, len, held, page0;
  };
  auto child = [&](int i) {
    Child c = {-1, -1, -1, -1, -1, -1};
    if (i < n) {
      c.s = src[i], c.d = dst[i], c.before = i ? src[i - 1] : -1;
      if (c.s >= 0 && c.s < S) c.len = lens[c.s];
      if (c.d >= 0 && c.d < S) c.held = lens[c.d], c.page0 = table[(size_t)c.d * M];
    }
    return c;
  };
  const Child c0 = child(threadIdx.x);
  const int ref0 = threadIdx.x < P ? refs[threadIdx.x] : 1;
  const bool ok = list_ok(dst, n, S, bm, &bad);
  if (threadIdx.x == 0) faults = ok ? 0 : 1 << PG_BAD_STREAM, nlook = most = 0;
  __syncthreads();
  int total = 0;
  if (ok) {
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
      const int i = i0 + threadIdx.x;
      const Child c = i0 == 0 ? c0 : child(i);
      int part = 0, page = -1;
      if (i < n) {
        // a source that is also a child, or a child that still holds pages
        if (c.s < 0 || c.s >= S || (bm[c.s >> 5] >> (c.s & 31) & 1) || c.held != 0 ||
            c.page0 >= 0) {
          atomicOr(&faults, 1 << PG_BAD_STREAM);
        } else if (c.len < 0 || c.len > (long long)M * R) {
          atomicOr(&faults, 1 << PG_TABLE_FULL);
        } else {
          if ((part = c.len % R) > 0) page = table[(size_t)c.s * M + c.len / R];
          if (c.len > 0 && c.s != c.before) {  // children of one source in a row: once
            const int k = atomicAdd(&nlook, 1), np = c.len / R + (part > 0);
            look[k] = c.s;
            pages[k] = np;
            atomicMax(&most, np);
          }
        }
      }
      const int at = total + block_excl_scan(part > 0, wt, &tot);
      if (i < n) mv.of[i] = part > 0 ? at : -1;
      if (part > 0) {
        mv.from[at] = page;
        mv.rows[at] = part;
      }
      total += tot;
      // every page below a source's length is there, 2^bits threads a source
      const int bits = most > 1 ? 32 - __clz(most - 1) : 0;
      const long long all = (long long)nlook << bits;
      bool gone = false;
#pragma unroll 4
      for (long long t = threadIdx.x; t < all; t += PG_THREADS) {
        const int k = (int)(t >> bits), m = (int)(t & ((1ll << bits) - 1));
        if (m < pages[k]) gone |= (unsigned)table[(size_t)look[k] * M + m] >= (unsigned)P;
      }
      if (gone) atomicOr(&faults, 1 << PG_BAD_PAGE);
      __syncthreads();
      if (threadIdx.x == 0) nlook = most = 0;
      __syncthreads();
    }
    if (!faults && total > 0) {
      const int got = total <= P ? take_free(refs, P, total, ref0, mv.to, wt, &tot) : 0;
      if (got < total && threadIdx.x == 0) faults = 1 << PG_NO_PAGES;
    }
    __syncthreads();
  }
  if (!faults)
    for (int k = threadIdx.x; k < total; k += blockDim.x) refs[mv.to[k]] = 1;
  if (threadIdx.x == 0) {
    *mv.count = faults ? -1 : total;
    status[0] = faults ? __ffs(faults) - 1 : PG_OK;
    status[1] = faults ? 0 : total;
  }
}

// Compaction: live pages with id >= n (n: how many are live) go, ascending, to the free ids
// below n, ascending. name[p]: page p's new id.
__global__ void __launch_bounds__(PG_THREADS)
    pages_compact_plan_kernel(int* refs, int P, int R, int* name, Moves mv, int* status) {
  __shared__ int wt[32], tot, bad;
  pdl_trigger();
  int live = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  for (int p0 = 0; p0 < P; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int r = p < P ? refs[p] : 0;
    if (r < 0) bad = 1;
    live += __syncthreads_count(r > 0);
  }
  if (bad) {
    if (threadIdx.x == 0) *mv.count = -1, status[0] = PG_BAD_PAGE, status[1] = 0;
    return;
  }
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < P; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int r = p < P ? refs[p] : 0;
    const int hole = p < live && r == 0, mover = p >= live && r > 0;
    const int a = holes + block_excl_scan(hole, wt, &tot);
    holes += tot;
    __syncthreads();
    const int b = movers + block_excl_scan(mover, wt, &tot);
    movers += tot;
    __syncthreads();
    if (hole) mv.to[a] = p;
    if (mover) mv.from[b] = p;
    if (p < P) name[p] = p;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += blockDim.x) {
    const int f = mv.from[k], t = mv.to[k];
    mv.rows[k] = R;
    name[f] = t;
    refs[t] = refs[f];
    refs[f] = 0;
  }
  if (threadIdx.x == 0) {
    *mv.count = movers;
    status[0] = PG_OK;
    status[1] = movers;
  }
}

// One warp's piece of the moves: up to 4 KiB of one head's rows of one page of one plane.
// CTAs per SM: a fork's pieces are half empty and go round a small grid (8: 49 us for 64 children of
// 80 planes; 32: 51, 4: 58). A compaction's are whole, and a larger grid's CTAs follow each other in
// the order of addresses (8: 199 us for 118 pages, 32: 192; with nothing to move 6 and 8 us).
constexpr int MV_PIECE = 4096, MV_THREADS = 256, MV_FORK_CTAS = 8, MV_COMPACT_CTAS = 32;

__device__ __forceinline__ void move_rows(char* pool, const Moves& mv, int count, int planes, int P,
                                          int H, int R, int row_bytes) {
  const long long page = (long long)H * R * row_bytes, plane = page * P;
  const int pieces = (R * row_bytes + MV_PIECE - 1) / MV_PIECE, lane = threadIdx.x & 31;
  const long long tasks = (long long)count * planes * H * pieces;
  const long long nw = (long long)gridDim.x * (MV_THREADS / 32);
  for (long long w = blockIdx.x * (MV_THREADS / 32) + (threadIdx.x >> 5); w < tasks; w += nw) {
    const int piece = (int)(w % pieces);
    long long u = w / pieces;
    const int h = (int)(u % H);
    u /= H;
    const int k = (int)(u % count), pl = (int)(u / count);
    const int f = mv.from[k], t = mv.to[k];
    const int end = min(mv.rows[k] * row_bytes, (piece + 1) * MV_PIECE);
    if (f < 0 || f >= P || t < 0 || t >= P) continue;
    const char* s = pool + pl * plane + f * page + (long long)h * R * row_bytes;
    char* d = pool + pl * plane + t * page + (long long)h * R * row_bytes;
    uint4 v[MV_PIECE / 512];
#pragma unroll
    for (int i = 0; i < MV_PIECE / 512; ++i) {
      const int at = piece * MV_PIECE + i * 512 + lane * 16;
      if (at < end) v[i] = *reinterpret_cast<const uint4*>(s + at);
    }
#pragma unroll
    for (int i = 0; i < MV_PIECE / 512; ++i) {
      const int at = piece * MV_PIECE + i * 512 + lane * 16;
      if (at < end)  // a copy is not read soon: 3 us less on a fork of 202 MB than plain stores
        __stcs(reinterpret_cast<uint4*>(d + at), v[i]);
    }
  }
}

// The fork's table rows, counts and part-filled pages. A child's row: its source's whole pages,
// then the copied page. Children are nobody's source, so rows read and rows written differ.
__global__ void __launch_bounds__(MV_THREADS)
    pages_fork_kernel(char* pool, int planes, int* table, int* lens, int* refs, int M, int P, int H,
                      int R, int row_bytes, const int* src, const int* dst, int n, Moves mv) {
  pdl_wait();
  const int count = *mv.count;
  if (count < 0) return;  // the check failed
  const long long all = (long long)n * M;
  for (long long e = (gridDim.x - 1 - blockIdx.x) * (long long)blockDim.x + threadIdx.x; e < all;
       e += (long long)gridDim.x * blockDim.x) {
    const int i = (int)(e / M), m = (int)(e % M), len = lens[src[i]];
    int p = -1;
    if (m < len / R) {
      p = table[(size_t)src[i] * M + m];
      if (p >= 0 && p < P) atomicAdd(refs + p, 1);
    } else if (m == len / R && mv.of[i] >= 0) {
      p = mv.to[mv.of[i]];  // the child's copy of the part-filled page
    }
    table[(size_t)dst[i] * M + m] = p;
    if (m == 0) lens[dst[i]] = len;
  }
  move_rows(pool, mv, count, planes, P, H, R, row_bytes);
}

__global__ void __launch_bounds__(MV_THREADS)
    pages_compact_kernel(char* pool, int planes, int* table, long long entries, int P, int H, int R,
                         int row_bytes, const int* name, Moves mv) {
  pdl_wait();
  const int count = *mv.count;
  if (count <= 0) return;
  for (long long e = blockIdx.x * (long long)blockDim.x + threadIdx.x; e < entries;
       e += (long long)gridDim.x * blockDim.x) {
    const int p = table[e];
    if (p >= 0 && p < P && name[p] != p) table[e] = name[p];
  }
  move_rows(pool, mv, count, planes, P, H, R, row_bytes);
}

// A kernel that starts while the one before it (which triggers it and was itself launched plainly)
// still runs; it waits for that one's end on the GPU.
template <typename... KArgs, typename... Args>
static cudaError_t launch_early(void (*kernel)(KArgs...), int grid, int block, cudaStream_t st,
                                Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

static int pages_check(const char* who, const void* table, const void* refs, int S, int M, int P) {
  LG_CHECK_ARG(table && refs, "%s: NULL pointer", who);
  LG_CHECK_ARG(S > 0 && S <= PG_MAX_STREAMS && M > 0 && P > 0 && P <= (1 << 24),
               "%s: %d streams of %d pages over %d pages", who, S, M, P);
  return LG_OK;
}

static int pool_check(const char* who, const void* pool, int planes, int H, int R, int row_bytes) {
  LG_CHECK_ARG(pool && aligned(pool, 16), "%s: the pool must be 16-byte aligned", who);
  LG_CHECK_ARG(planes > 0 && H > 0 && R > 0 && row_bytes > 0 && row_bytes % 16 == 0 &&
                   (long long)R * row_bytes <= (1 << 30),
               "%s: %d planes, %d heads, %d rows of %d bytes (a multiple of 16)", who, planes, H, R,
               row_bytes);
  return LG_OK;
}

}  // namespace lg

using namespace lg;

extern "C" size_t lg_pages_workspace_bytes(int P, int n) {
  if (P < 0 || n < 0) return 0;
  return ((size_t)64 + 4 * (size_t)P + 4 * (size_t)n + 64) * sizeof(int);
}

extern "C" int lg_pages_reserve(int32_t* table, int32_t* refs, int S, int M, int P, int R,
                                const int32_t* ids, const int32_t* rows, int n, int32_t* status,
                                void* ws, size_t ws_bytes, void* stream) {
  if (int rc = pages_check("pages_reserve", table, refs, S, M, P)) return rc;
  LG_CHECK_ARG(((ids && rows) || n == 0) && status && n >= 0 && n <= S && R > 0,
               "pages_reserve: %d streams of %d", n, S);
  if (!ws || ws_bytes < lg_pages_workspace_bytes(P, n))
    return fail(LG_ERR_WORKSPACE, "pages_reserve: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  pages_reserve_kernel<<<1, PG_THREADS, 0, st>>>(table, refs, S, M, P, R, ids, rows, n,
                                                 static_cast<int*>(ws), status);
  LG_LAUNCH_CHECK("pages_reserve");
  return LG_OK;
}

extern "C" int lg_pages_free(int32_t* table, int32_t* lens, int32_t* refs, int S, int M, int P,
                             const int32_t* ids, int n, int32_t* status, void* stream) {
  if (int rc = pages_check("pages_free", table, refs, S, M, P)) return rc;
  LG_CHECK_ARG(lens && (ids || n == 0) && status && n >= 0 && n <= S,
               "pages_free: %d streams of %d", n, S);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long all = (long long)n * M;
  const int grid = (int)std::min<long long>(64, all / (4 * PG_THREADS) + 1);
  pages_free_kernel<<<grid, PG_THREADS, 0, st>>>(table, lens, refs, S, M, P, ids, n, status);
  LG_LAUNCH_CHECK("pages_free");
  return LG_OK;
}

extern "C" int lg_pages_fork(void* pool, int planes, int H, int R, int row_bytes, int32_t* table,
                             int32_t* lens, int32_t* refs, int S, int M, int P, const int32_t* src,
                             const int32_t* dst, int n, int32_t* status, void* ws, size_t ws_bytes,
                             void* stream) {
  if (int rc = pages_check("pages_fork", table, refs, S, M, P)) return rc;
  if (int rc = pool_check("pages_fork", pool, planes, H, R, row_bytes)) return rc;
  LG_CHECK_ARG(lens && ((src && dst) || n == 0) && status && n >= 0 && n <= S,
               "pages_fork: %d children of %d", n, S);
  if (!ws || ws_bytes < lg_pages_workspace_bytes(P, n))
    return fail(LG_ERR_WORKSPACE, "pages_fork: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Moves mv = moves_of(ws, n);
  pages_fork_plan_kernel<<<1, PG_THREADS, 0, st>>>(table, lens, refs, S, M, P, R, src, dst, n, mv,
                                                   status);
  LG_LAUNCH_CHECK("pages_fork_plan");
  const long long pieces =
      (long long)n * planes * H * (((long long)R * row_bytes + MV_PIECE - 1) / MV_PIECE);
  const int grid =
      (int)std::min<long long>((long long)MV_FORK_CTAS * device_sm_count(),
                               pieces / (MV_THREADS / 32) + 1);
  LG_CUDA_TRY(launch_early(pages_fork_kernel, grid, MV_THREADS, st, static_cast<char*>(pool),
                           planes, table, lens, refs, M, P, H, R, row_bytes, src, dst, n, mv));
  LG_LAUNCH_CHECK("pages_fork");
  return LG_OK;
}

extern "C" int lg_pages_compact(void* pool, int planes, int H, int R, int row_bytes, int32_t* table,
                                int32_t* refs, int S, int M, int P, int32_t* status, void* ws,
                                size_t ws_bytes, void* stream) {
  if (int rc = pages_check("pages_compact", table, refs, S, M, P)) return rc;
  if (int rc = pool_check("pages_compact", pool, planes, H, R, row_bytes)) return rc;
  LG_CHECK_ARG(status, "pages_compact: NULL status");
  if (!ws || ws_bytes < lg_pages_workspace_bytes(P, 0))
    return fail(LG_ERR_WORKSPACE, "pages_compact: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Moves mv = moves_of(ws, P);
  int* name = mv.of;  // [P]
  pages_compact_plan_kernel<<<1, PG_THREADS, 0, st>>>(refs, P, R, name, mv, status);
  LG_LAUNCH_CHECK("pages_compact_plan");
  // at most half of the pages move
  const long long pieces =
      (long long)(P / 2) * planes * H * (((long long)R * row_bytes + MV_PIECE - 1) / MV_PIECE);
  const int grid = (int)std::min<long long>((long long)MV_COMPACT_CTAS * device_sm_count(),
                                            pieces / (MV_THREADS / 32) + 1);
  LG_CUDA_TRY(launch_early(pages_compact_kernel, grid, MV_THREADS, st, static_cast<char*>(pool),
                           planes, table, (long long)S * M, P, H, R, row_bytes, name, mv));
  LG_LAUNCH_CHECK("pages_compact");
  return LG_OK;
}
