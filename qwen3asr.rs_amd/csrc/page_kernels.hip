// Blocks of the paged cache shared between rows of a batch, copied and moved
// (gfx950): rows forked from others, given up again, and the blocks in use
// brought to the front of the pool. The state is the block allocator's
// (metadata_kernels.hip) with one more array, shared[b]: how many rows hold block
// b besides the first. It is 0 for a block with one holder or none, so the
// allocator's other operations, whose blocks are fresh, need not know of it.
//
// All of it is moved bytes and whole numbers: the copy is bound by HBM (two
// passes over the blocks: 165 MB in 112 buffers of 28 layers 29 us, 5.7 TB/s), the rest
// by the latency of a few dependent loads (96 forks 4.7 + 3.7 us, their release 13; the
// blocks of a pool of 1024 paired and renamed 6 + 4).

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kPageThreads = 1024;

// Exclusive prefix sum over the workgroup's 1024 lanes; *total gets the sum.
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t* s_tmp, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t incl = (uint32_t)wave_scan_i32((int)v);
  if (lane == 63) s_tmp[wave] = incl;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / 64; ++w) {
    const uint32_t t = s_tmp[w];
    before += w < wave ? t : 0u;
    all += t;
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

// Waits for this wave's memory operations, atomics among them (a barrier alone
// does not); then the workgroup's, which all go to one L2, are done for each other.
__device__ __forceinline__ void finish_and_sync() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Place `at` + `more` of the ring (32-bit: the capacity is below 2^31).
__device__ __forceinline__ uint32_t ring_at(const PageState& s, uint32_t at, uint32_t more) {
  return (at % (uint32_t)s.ring_cap + more) % (uint32_t)s.ring_cap;
}

// (past the L1 cache, which other compute units' atomics do not update)
__device__ __forceinline__ uint32_t load_fresh(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- copies ----------------------------------------------------------------

template <typename V>
__device__ __forceinline__ void copy_as(char* base, int64_t src, int64_t dst, uint32_t bytes) {
  const V* s = reinterpret_cast<const V*>(base + src);
  V* d = reinterpret_cast<V*>(base + dst);
  for (uint32_t i = threadIdx.x; i < bytes / sizeof(V); i += blockDim.x) d[i] = s[i];
}

// Items (pair, buffer), pairs slowest; every workgroup takes its share of them.
__global__ __launch_bounds__(256) void copy_blocks_kernel(const CopyBuffers b, int32_t num_buffers,
                                                          const uint32_t* __restrict__ src,
                                                          const uint32_t* __restrict__ dst,
                                                          const uint32_t* __restrict__ num_pairs,
                                                          uint32_t max_pairs, int64_t num_blocks) {
  const uint32_t pairs = num_pairs != nullptr ? min(*num_pairs, max_pairs) : max_pairs;
  const uint64_t items = (uint64_t)pairs * (uint32_t)num_buffers;
  for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const uint32_t pair = (uint32_t)(it / (uint32_t)num_buffers);
    const uint32_t k = (uint32_t)(it % (uint32_t)num_buffers);
    const uint32_t from = src[pair], to = dst[pair];
    if ((int64_t)from >= num_blocks || (int64_t)to >= num_blocks || from == to) continue;
    char* base = b.base[k];
    const int64_t stride = b.stride[k];
    const uint32_t bytes = b.bytes[k];
    const uint64_t mix = (uint64_t)(uintptr_t)base | (uint64_t)stride | bytes;
    if (mix % 16 == 0) {
      const uint4* s = reinterpret_cast<const uint4*>(base + from * stride);
      uint4* d = reinterpret_cast<uint4*>(base + to * stride);
      const uint32_t n = bytes / 16;
      uint32_t i = threadIdx.x;
      for (; i + 3 * 256 < n; i += 4 * 256) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = load_stream(s + i + u * 256);
#pragma unroll
        for (int u = 0; u < 4; ++u) d[i + u * 256] = v[u];
      }
      for (; i < n; i += 256) d[i] = load_stream(s + i);
    } else if (mix % 4 == 0) {
      copy_as<uint32_t>(base, from * stride, to * stride, bytes);
    } else {
      copy_as<uint8_t>(base, from * stride, to * stride, bytes);
    }
  }
}

// ---- forks -----------------------------------------------------------------

// Which forks there can be, the new rows' lengths and the blocks that are copied
// for them, by one workgroup with a lane per fork.
__global__ __launch_bounds__(kPageThreads) void fork_decide_kernel(
    const PageState s, const uint32_t* __restrict__ src_rows,
    const uint32_t* __restrict__ dst_rows, int32_t num_forks, uint8_t* __restrict__ ok,
    uint32_t* __restrict__ copy_src, uint32_t* __restrict__ copy_dst,
    uint32_t* __restrict__ copy_count) {
  __shared__ uint32_t s_tmp[kPageThreads / 64];
  __shared__ __align__(16) uint32_t s_dst[kMaxForks];
  const int f = threadIdx.x;
  const uint32_t head = s.ring_state[0], avail = s.ring_state[1];
  uint32_t src = 0xffffffffu, dst = 0xffffffffu, tokens = 0, last = 0;
  if (f < num_forks) {
    src = src_rows[f];
    dst = dst_rows[f];
  }
  s_dst[f] = dst;
  __syncthreads();
  bool can = f < num_forks && src < (uint32_t)s.num_rows && dst < (uint32_t)s.num_rows;
  if (can) {
    const uint32_t have = min(s.row_blocks[src], (uint32_t)s.cols);
    tokens = (uint32_t)min((uint64_t)s.positions[src], (uint64_t)have * (uint32_t)s.block_size);
    can = s.row_blocks[dst] == 0;
  }
  // an earlier fork of the same row? (four at a time, the reads not waiting on each other)
  bool claimed = false;
  const int before = (int)(threadIdx.x & ~63u) < num_forks ? min(f | 63, num_forks) : 0;
#pragma unroll 4
  for (int e = 0; e < before; e += 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(&s_dst[e]);
    claimed |= ((v.x == dst) & (e < f)) | ((v.y == dst) & (e + 1 < f)) |
               ((v.z == dst) & (e + 2 < f)) | ((v.w == dst) & (e + 3 < f));
  }
  can = can && !claimed;
  const uint32_t full = tokens / (uint32_t)s.block_size;
  const bool part = can && tokens % (uint32_t)s.block_size != 0;
  if (part) last = s.block_tables[(int64_t)src * s.cols + full];
  uint32_t total;
  const uint32_t rank = group_scan(part ? 1u : 0u, s_tmp, &total);
  if (part && rank >= avail) can = false;
  // (every lane's reads of the rows are done: the scan's barriers)
  if (f < num_forks) ok[f] = can ? 1 : 0;
  if (can) {
    s.positions[dst] = tokens;
    s.row_blocks[dst] = full + (part ? 1u : 0u);
    if (part) {
      const uint32_t id = s.ring[ring_at(s, head, rank)];
      s.block_tables[(int64_t)dst * s.cols + full] = id;
      copy_src[rank] = last;
      copy_dst[rank] = id;
    }
  }
  if (f == 0) {
    const uint32_t used = min(total, avail);
    *copy_count = used;
    s.ring_state[0] = ring_at(s, head, used);
    s.ring_state[1] = avail - used;
  }
}

// The whole blocks of each fork's source become its own too. (A row that holds
// blocks is no fork's target, so no table that is read here is written.)
__global__ __launch_bounds__(256) void fork_share_kernel(const PageState s,
                                                         const uint32_t* __restrict__ src_rows,
                                                         const uint32_t* __restrict__ dst_rows,
                                                         const uint8_t* __restrict__ ok) {
  const int f = blockIdx.x;
  if (!ok[f]) return;
  const uint32_t src = src_rows[f], dst = dst_rows[f];
  const uint32_t full = s.positions[dst] / (uint32_t)s.block_size;
  for (uint32_t i = threadIdx.x; i < full; i += 256) {
    const uint32_t id = s.block_tables[(int64_t)src * s.cols + i];
    s.block_tables[(int64_t)dst * s.cols + i] = id;
    if (id != 0 && (int64_t)id < s.num_blocks) atomicAdd(&s.shared[id], 1u);
  }
}

// ---- releases --------------------------------------------------------------

// Rows give back blocks keep_blocks[r] .. row_blocks[r] - 1. Taken one after the
// other, rows in order and each row's last block first, every block loses a
// holder, and goes to the ring with its last one. Done at once: first all holders
// are subtracted, which leaves -1 where none is left; there, the entry that comes
// last in that order is found by an atomic minimum over codes that fall with the
// order, in the same word; that entry gives the block back, at a place in the
// ring by a prefix sum. The entries are numbered in that order, so a lane takes
// four of any rows at a time: with a wave per row instead, 96 rows of 40 blocks
// took 28 us, each waiting for its own loads.
__global__ __launch_bounds__(kPageThreads) void release_shared_kernel(
    const PageState s, const uint32_t* __restrict__ keep_blocks) {
  __shared__ uint32_t s_tmp[kPageThreads / 64];
  __shared__ uint32_t s_rows[kPageThreads], s_first[kPageThreads], s_have[kPageThreads];
  constexpr int U = 4;
  const uint32_t head = s.ring_state[0], count = s.ring_state[1];
  // Of the rows base .. base + 1023 those that give something back, in order, and the
  // number of each one's first entry; every pass lists them again unless one list
  // holds them all.
  struct List {
    uint32_t rows, entries;
  };
  auto list_rows = [&](int base) {
    const int r = base + threadIdx.x;
    uint32_t have = 0, keep = 0;
    if (r < s.num_rows) {
      have = min(s.row_blocks[r], (uint32_t)s.cols);
      keep = min(keep_blocks[r], have);
    }
    List l;
    const uint32_t rank = group_scan(keep < have ? 1u : 0u, s_tmp, &l.rows);
    const uint32_t first = group_scan(have - keep, s_tmp, &l.entries);
    if (keep < have) {
      s_rows[rank] = (uint32_t)r;
      s_first[rank] = first;
      s_have[rank] = have;
    }
    __syncthreads();
    return l;
  };
  // The blocks of entries e .. e + U - 1 of the list, 0: none or not counted. Their rows
  // are the last ones whose entries begin at or before them (found together, so that no
  // search waits for another's reads).
  auto blocks_of = [&](const List& l, uint32_t e, uint32_t (&id)[U]) {
    uint32_t row[U] = {};
    for (uint32_t step = l.rows > 1 ? 1u << (31 - __builtin_clz(l.rows - 1)) : 0u; step != 0;
         step /= 2) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t next = row[u] + step;
        if (next < l.rows && s_first[next] <= e + u) row[u] = next;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = 0;
      if (e + u >= l.entries) continue;
      const uint32_t i = s_have[row[u]] - 1u - (e + u - s_first[row[u]]);
      id[u] = s.block_tables[(int64_t)s_rows[row[u]] * s.cols + i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = (int64_t)id[u] < s.num_blocks ? id[u] : 0u;
  };
  const bool one_list = s.num_rows <= kPageThreads;
  List l{};
  // few entries are looked up once
  uint32_t held[U] = {};
  bool few = false;
  // body(id[U], number of the first of these entries): consecutive entries of a lane
  auto pass = [&](auto&& body, auto&& done) {
    uint32_t before = 0;
    for (int base = 0; base < s.num_rows; base += kPageThreads) {
      if (!one_list) l = list_rows(base);
      for (uint32_t at = 0; at < l.entries; at += U * kPageThreads) {
        const uint32_t e = at + U * threadIdx.x;
        if (few) {
          body(held, before + e);
        } else {
          uint32_t id[U];
          blocks_of(l, e, id);
          body(id, before + e);
        }
      }
      before += l.entries;
      done();
    }
  };
  auto code_of = [](uint32_t e) { return 0xfffffffeu - e; };
  if (one_list) {
    l = list_rows(0);
    if (l.rows == 0) return;  // (uniform)
    few = l.entries <= U * kPageThreads;
    if (few) blocks_of(l, U * threadIdx.x, held);
  }
  pass(
      [&](const uint32_t(&id)[U], uint32_t) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (id[u] != 0) atomicSub(&s.shared[id[u]], 1u);
      },
      [] { finish_and_sync(); });
  pass(
      [&](const uint32_t(&id)[U], uint32_t e) {
        uint32_t left[U];
#pragma unroll
        for (int u = 0; u < U; ++u) left[u] = id[u] != 0 ? load_fresh(&s.shared[id[u]]) : 0u;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (left[u] >= 0x80000000u) atomicMin(&s.shared[id[u]], code_of(e + u));
      },
      [] { finish_and_sync(); });
  uint32_t added = 0;
  pass(
      [&](const uint32_t(&id)[U], uint32_t e) {
        uint32_t last[U], n = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) last[u] = id[u] != 0 ? load_fresh(&s.shared[id[u]]) : 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) n += last[u] == code_of(e + u) ? 1u : 0u;
        uint32_t total;
        uint32_t at = (uint32_t)(((uint64_t)head + count + added + group_scan(n, s_tmp, &total)) %
                                 (uint32_t)s.ring_cap);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (last[u] == code_of(e + u)) {
            s.ring[at] = id[u];
            at = ring_at(s, at, 1u);
            // (no other entry of this block compares equal, before or after)
            __hip_atomic_store(&s.shared[id[u]], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        added += total;
      },
      [&] {
        const uint32_t k = threadIdx.x;
        if (k < l.rows) {
          const uint32_t end = k + 1 < l.rows ? s_first[k + 1] : l.entries;
          s.row_blocks[s_rows[k]] = s_have[k] - (end - s_first[k]);
        }
        __syncthreads();
      });
  if (threadIdx.x == 0) s.ring_state[1] = count + added;
}

// ---- copies before a write --------------------------------------------------

// Rows, in order, replace each block that they would write to and that others hold too:
// the one that their next token falls into, whose contents are copied, and those they
// still hold behind it. Such rows are rare (a row cut back below the length it was
// forked at): found by all lanes, taken one by one.
__global__ __launch_bounds__(kPageThreads) void unshare_rows_kernel(
    const PageState s, uint8_t* __restrict__ ok, uint32_t* __restrict__ copy_src,
    uint32_t* __restrict__ copy_dst, uint32_t* __restrict__ copy_count) {
  __shared__ uint32_t s_tmp[kPageThreads / 64];
  __shared__ uint32_t s_rows[kPageThreads];
  uint32_t head = s.ring_state[0], avail = s.ring_state[1], copies = 0;
  auto shared_block = [&](uint32_t id) {
    return id != 0 && (int64_t)id < s.num_blocks && s.shared[id] != 0;
  };
  for (int base = 0; base < s.num_rows; base += kPageThreads) {
    const int r = base + threadIdx.x;
    bool want = false;
    if (r < s.num_rows) {
      const uint32_t have = min(s.row_blocks[r], (uint32_t)s.cols);
      for (uint32_t at = s.positions[r] / (uint32_t)s.block_size; at < have && !want; ++at)
        want = shared_block(s.block_tables[(int64_t)r * s.cols + at]);
      ok[r] = 1;
    }
    uint32_t total;
    const uint32_t rank = group_scan(want ? 1u : 0u, s_tmp, &total);
    if (want) s_rows[rank] = (uint32_t)r;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (uint32_t k = 0; k < total; ++k) {
        const uint32_t row = s_rows[k], pos = s.positions[row];
        const uint32_t first = pos / (uint32_t)s.block_size;
        const uint32_t have = min(s.row_blocks[row], (uint32_t)s.cols);
        for (uint32_t at = first; at < have; ++at) {
          uint32_t* entry = &s.block_tables[(int64_t)row * s.cols + at];
          const uint32_t id = *entry;
          if (!shared_block(id)) continue;  // (or the rows before it have all taken copies)
          if (avail == 0) {
            ok[row] = 0;
            break;
          }
          const uint32_t fresh = s.ring[head % (uint32_t)s.ring_cap];
          head = (head + 1) % (uint32_t)s.ring_cap;
          --avail;
          s.shared[id] -= 1;
          *entry = fresh;
          if (at == first && pos % (uint32_t)s.block_size != 0) {
            copy_src[copies] = id;
            copy_dst[copies] = fresh;
            ++copies;
          }
        }
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *copy_count = copies;
    s.ring_state[0] = head;
    s.ring_state[1] = avail;
  }
}

// ---- compaction --------------------------------------------------------------

// Workspace: a bit per block that is free (word 0, bit 0 is block 0, never free),
// the number of moved blocks before each word, and {front, free}.
struct CompactSpace {
  uint32_t* free_bits;
  uint32_t* moved_before;
  uint32_t* sizes;
  int32_t words;
};
CompactSpace compact_space(void* workspace, int64_t num_blocks) {
  const int32_t words = (int32_t)((num_blocks + 31) / 32);
  uint32_t* w = static_cast<uint32_t*>(workspace);
  return {w, w + words, w + 2 * (int64_t)words, words};
}

__global__ __launch_bounds__(256) void compact_clear_kernel(CompactSpace c) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < c.words; i += gridDim.x * 256)
    c.free_bits[i] = 0;
}

__global__ __launch_bounds__(256) void compact_mark_kernel(const PageState s, CompactSpace c) {
  const uint32_t head = s.ring_state[0], count = min(s.ring_state[1], (uint32_t)s.ring_cap);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) {
    const uint32_t id = s.ring[ring_at(s, head, i)];
    if (id != 0 && (int64_t)id < s.num_blocks) atomicOr(&c.free_bits[id / 32], 1u << (id % 32));
  }
}

// Pools of at most this many blocks have their free bits collected by the pairing
// workgroup itself, in LDS: three launches become one (a few us each). A larger
// pool's ring is read faster by many workgroups.
constexpr int kCompactOneGroup = 65536;

// The k-th block in use past the front takes the k-th free place in it; the front
// is as long as there are blocks in use, so there are as many of the one as of the
// other. One workgroup, a run of words per lane.
template <bool kMark>
__global__ __launch_bounds__(kPageThreads) void compact_pair_kernel(
    const PageState s, CompactSpace c, uint32_t* __restrict__ copy_src,
    uint32_t* __restrict__ copy_dst, uint32_t* __restrict__ copy_count) {
  __shared__ uint32_t s_tmp[kPageThreads / 64];
  __shared__ uint32_t s_bits[kMark ? kCompactOneGroup / 32 : 1];
  if constexpr (kMark) {
    for (int i = threadIdx.x; i < c.words; i += kPageThreads) s_bits[i] = 0;
    __syncthreads();
    const uint32_t head = s.ring_state[0], count = min(s.ring_state[1], (uint32_t)s.ring_cap);
    for (uint32_t i = threadIdx.x; i < count; i += kPageThreads) {
      const uint32_t id = s.ring[ring_at(s, head, i)];
      if (id != 0 && (int64_t)id < s.num_blocks) atomicOr(&s_bits[id / 32], 1u << (id % 32));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < c.words; i += kPageThreads) c.free_bits[i] = s_bits[i];
  }
  const uint32_t* bits = kMark ? s_bits : c.free_bits;
  const int per = (c.words + kPageThreads - 1) / kPageThreads;
  const int a = min(threadIdx.x * per, (unsigned)c.words), b = min(a + per, c.words);
  uint32_t n = 0;
  for (int i = a; i < b; ++i) n += (uint32_t)__builtin_popcount(bits[i]);
  uint32_t free_blocks;
  group_scan(n, s_tmp, &free_blocks);
  const uint32_t nb = (uint32_t)s.num_blocks, front = nb - 1 - free_blocks;
  // bits of word i that are ids 1 .. front, and front + 1 .. nb - 1
  auto upto = [](uint32_t id, int i) {  // ids <= id
    const int64_t left = (int64_t)id + 1 - 32 * (int64_t)i;
    return left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
  };
  auto holes_of = [&](int i) { return bits[i] & upto(front, i); };
  auto moved_of = [&](int i) { return ~bits[i] & upto(nb - 1, i) & ~upto(front, i); };
  uint32_t holes = 0, moved = 0, total;
  for (int i = a; i < b; ++i) {
    holes += (uint32_t)__builtin_popcount(holes_of(i));
    moved += (uint32_t)__builtin_popcount(moved_of(i));
  }
  holes = group_scan(holes, s_tmp, &total);
  moved = group_scan(moved, s_tmp, &total);
  for (int i = a; i < b; ++i) {
    for (uint32_t m = holes_of(i); m != 0; m &= m - 1)
      copy_dst[holes++] = 32u * i + __builtin_ctz(m);
    c.moved_before[i] = moved;
    for (uint32_t m = moved_of(i); m != 0; m &= m - 1)
      copy_src[moved++] = 32u * i + __builtin_ctz(m);
  }
  if (threadIdx.x == 0) {
    *copy_count = total;
    c.sizes[0] = front;
    c.sizes[1] = free_blocks;
  }
}

// Tables, counts of holders and the ring follow.
__global__ __launch_bounds__(256) void compact_apply_kernel(
    const PageState s, CompactSpace c, const uint32_t* __restrict__ copy_src,
    const uint32_t* __restrict__ copy_dst, const uint32_t* __restrict__ copy_count) {
  const uint32_t front = c.sizes[0], free_blocks = c.sizes[1], moves = *copy_count;
  const int64_t start = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t e = start; e < (int64_t)s.num_rows * s.cols; e += step) {
    const int64_t r = e / s.cols;
    if ((uint32_t)(e - r * s.cols) >= s.row_blocks[r]) continue;
    const uint32_t id = s.block_tables[e];
    if (id <= front || (int64_t)id >= s.num_blocks) continue;
    const uint32_t bit = id % 32, word = c.free_bits[id / 32];
    if ((word >> bit) & 1u) continue;  // (a table that names a free block: left alone)
    // blocks in use past the front, in this word, before id
    const int64_t low = (int64_t)front + 1 - 32 * (int64_t)(id / 32);
    const uint32_t past = low <= 0 ? 0xffffffffu : 0xffffffffu << low;
    const uint32_t k = c.moved_before[id / 32] +
                       (uint32_t)__builtin_popcount(~word & past & ((1u << bit) - 1u));
    s.block_tables[e] = copy_dst[k];
  }
  for (int64_t k = start; s.shared != nullptr && k < moves; k += step) {
    s.shared[copy_dst[k]] = s.shared[copy_src[k]];
    s.shared[copy_src[k]] = 0;
  }
  for (int64_t i = start; i < free_blocks && i < s.ring_cap; i += step)
    s.ring[i] = front + 1 + (uint32_t)i;
  if (start == 0) {
    s.ring_state[0] = 0;
    s.ring_state[1] = free_blocks;
  }
}

unsigned grid_of(int64_t lanes) {
  const int64_t n = (lanes + 255) / 256;
  return (unsigned)(n < 1 ? 1 : n > 4096 ? 4096 : n);
}

}  // namespace

hipError_t launch_copy_blocks(const CopyBuffers& b, int32_t num_buffers, const uint32_t* src,
                              const uint32_t* dst, const uint32_t* num_pairs, int32_t max_pairs,
                              int64_t num_blocks, hipStream_t stream) {
  const int64_t items = (int64_t)max_pairs * num_buffers;
  hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)(items < 4096 ? items : 4096)), dim3(256),
                     0, stream, b, num_buffers, src, dst, num_pairs, (uint32_t)max_pairs,
                     num_blocks);
  return hipGetLastError();
}

hipError_t launch_fork_rows(const PageState& s, const uint32_t* src_rows, const uint32_t* dst_rows,
                            int32_t num_forks, uint8_t* ok, uint32_t* copy_src, uint32_t* copy_dst,
                            uint32_t* copy_count, hipStream_t stream) {
  hipLaunchKernelGGL(fork_decide_kernel, dim3(1), dim3(kPageThreads), 0, stream, s, src_rows,
                     dst_rows, num_forks, ok, copy_src, copy_dst, copy_count);
  if (num_forks == 0) return hipGetLastError();
  hipLaunchKernelGGL(fork_share_kernel, dim3((unsigned)num_forks), dim3(256), 0, stream, s,
                     src_rows, dst_rows, ok);
  return hipGetLastError();
}

hipError_t launch_release_shared(const PageState& s, const uint32_t* keep_blocks,
                                 hipStream_t stream) {
  hipLaunchKernelGGL(release_shared_kernel, dim3(1), dim3(kPageThreads), 0, stream, s, keep_blocks);
  return hipGetLastError();
}

hipError_t launch_unshare_rows(const PageState& s, uint8_t* ok, uint32_t* copy_src,
                               uint32_t* copy_dst, uint32_t* copy_count, hipStream_t stream) {
  hipLaunchKernelGGL(unshare_rows_kernel, dim3(1), dim3(kPageThreads), 0, stream, s, ok, copy_src,
                     copy_dst, copy_count);
  return hipGetLastError();
}

size_t compact_workspace_bytes(int64_t num_blocks) {
  return 8 * (size_t)((num_blocks + 31) / 32) + 8;
}

hipError_t launch_compact(const PageState& s, uint32_t* copy_src, uint32_t* copy_dst,
                          uint32_t* copy_count, void* workspace, hipStream_t stream) {
  const CompactSpace c = compact_space(workspace, s.num_blocks);
  if (s.num_blocks <= kCompactOneGroup) {
    hipLaunchKernelGGL((compact_pair_kernel<true>), dim3(1), dim3(kPageThreads), 0, stream, s, c,
                       copy_src, copy_dst, copy_count);
  } else {
    hipLaunchKernelGGL(compact_clear_kernel, dim3(grid_of(c.words)), dim3(256), 0, stream, c);
    hipLaunchKernelGGL(compact_mark_kernel, dim3(grid_of(s.num_blocks)), dim3(256), 0, stream, s,
                       c);
    hipLaunchKernelGGL((compact_pair_kernel<false>), dim3(1), dim3(kPageThreads), 0, stream, s, c,
                       copy_src, copy_dst, copy_count);
  }
  int64_t lanes = (int64_t)s.num_rows * s.cols;
  if (lanes < s.num_blocks) lanes = s.num_blocks;
  hipLaunchKernelGGL(compact_apply_kernel, dim3(grid_of(lanes)), dim3(256), 0, stream, s, c,
                     copy_src, copy_dst, copy_count);
  return hipGetLastError();
}

}  // namespace vpa
