// What the tree attention kernels share: the call's parameters and which keys a node sees.
//
// The key of node i < n of sequence b is row past_b + i of the cache.  Node i sees the rows below
// past_b, which every node sees, and of the tree's own rows its ancestors' and its own: one bit a
// node, made by walking up the parents.  Only the last tiles, those with rows from past_b on,
// look at the bits.  Nodes from n on see what a root sees; their results are put to zero at the end.
// Lengths come from device memory and are clamped to the buffers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "score_common.cuh"

namespace fpk {
namespace tree {

using score::ex2_approx;
using score::grid_wait;
using score::launch_dependent;
using score::OptIn;

constexpr int kMaxNodes = FPK_TREE_MAX_NODES;
constexpr int kWords = kMaxNodes / 32;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  int* status;
  const void *q, *k, *v;
  void* o;
  const float *ks, *vs;      // scales of an 8-bit cache, or null
  const int32_t* parents;
  const int32_t* past;       // [batch]
  const int32_t* lens;       // [batch] or null
  float* part_o;             // [CTA][2][block's rows][D] unnormalised partial results
  float2* part_ml;           // [CTA][2][block's rows] (running maximum of base 2, sum)
  const int64_t* before;     // [batch + 1] units of the sequences before each (of one block each), or null: few sequences
  int64_t parents_st;
  int64_t q_st[3], k_st[3], v_st[3], o_st[3], ks_st[3], vs_st[3];
  int32_t batch, heads, kv_heads, group, nodes, room;
  int32_t block_rows, mblocks;  // rows (heads of a group x nodes) a block, blocks a key/value head
  int32_t per;                  // blocks a sequence: kv_heads * mblocks
  int32_t ctas;
  int32_t by_rows;              // tensor cores: the two warpgroups take two row tiles, not every other key tile
  float scale, scale_log2;
};

struct Seq {
  int n;     // nodes
  int past;  // row of node 0: -kMaxNodes .. room
  int all;   // rows that every node sees
  int len;   // rows that some node sees
};
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  s.n = p.lens ? min(max(__ldg(p.lens + b), 0), p.nodes) : p.nodes;
  s.past = min(max(__ldg(p.past + b), -kMaxNodes), p.room);
  s.all = max(s.past, 0);
  s.len = min(max(s.past + s.n, 0), p.room);
  return s;
}

// parents of the sequence's nodes, -1 for a root, into shared memory by the whole block
__device__ __forceinline__ void load_parents(const Params& p, const Seq& s, int b, int* parent, int threads) {
  for (int i = threadIdx.x; i < s.n; i += threads) {
    const int x = __ldg(p.parents + b * p.parents_st + i);
    parent[i] = x >= 0 && x < i ? x : -1;
  }
}
// the node's own bit and its ancestors'; none for a node from n on.  A parent comes before its
// child, so that the walk ends, and a word is written once.
__device__ __forceinline__ void walk_up(const Seq& s, const int* parent, int node, uint32_t* bits) {
  int x = node < s.n ? node : -1;
#pragma unroll 1
  for (int w = kWords - 1; w >= 0; --w) {
    uint32_t u = 0u;
    while (x >= 32 * w) {
      u |= 1u << (x & 31);
      x = parent[x];
      if (x < 0) break;
    }
    bits[w] = u;
  }
}
// the row of key j is one that the node of these bits sees (a tree may end behind the cache)
__device__ __forceinline__ bool sees(const Seq& s, const uint32_t* bits, int j) {
  const int a = j - s.past;
  return j < s.all || (a >= 0 && j < s.len && ((bits[a >> 5] >> (a & 31)) & 1u));
}

// The work is cut into equal parts whatever the lengths: the units of 128 keys of all blocks (sequence,
// key/value head, row block) in one line, of which CTA c takes [total c / ctas, total (c + 1) / ctas)
// (CTAs beyond the units have nothing to do: each of the others has one at least).
// A part begins and ends inside a block or at its border; the rows of a block that several CTAs share
// go to the workspace, at most two such a CTA (its first and its last), and tree_combine_kernel
// joins them.
constexpr int kUnit = 128;

__device__ __forceinline__ int units_of(const Seq& s) { return max(1, (s.len + kUnit - 1) / kUnit); }

// by a converged warp
__device__ __forceinline__ int64_t total_units(const Params& p) {
  if (p.before) return p.before[p.batch] * p.per;
  int64_t n = 0;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) n += units_of(seq_of(p, b));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
  return n * p.per;
}
struct Where {
  int b;
  int64_t base;  // the sequence's first unit
};
// the sequence that unit u < total belongs to; by a converged warp
__device__ __forceinline__ Where where_is(const Params& p, int64_t u) {
  const int lane = threadIdx.x & 31;
  if (p.before) {  // the last sequence that begins at u or before it
    int low = 0, high = p.batch;
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (p.before[mid] * p.per <= u) low = mid;
      else high = mid;
    }
    return Where{low, p.before[low] * p.per};
  }
  int64_t run = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int64_t mine = b0 + lane < p.batch ? static_cast<int64_t>(units_of(seq_of(p, b0 + lane))) * p.per : 0;
    int64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, run + upto > u);
    if (hit) {
      const int l = __ffs(hit) - 1;
      return Where{b0 + l, run + __shfl_sync(0xffffffffu, upto - mine, l)};
    }
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Where{p.batch - 1, run};
}
__device__ __forceinline__ int ctas_of(const Params& p, int64_t total) {
  return static_cast<int>(total < p.ctas ? total : p.ctas);
}
// (in 32 bits where they do: a division in 64 is some 100 instructions; ctas is below 1024)
__device__ __forceinline__ int64_t first_unit(int64_t total, int cta, int ctas) {
  if (total < (1 << 22)) return static_cast<uint32_t>(total) * static_cast<uint32_t>(cta) / static_cast<uint32_t>(ctas);
  return total * cta / ctas;
}
__device__ __forceinline__ int cta_of(int64_t total, int64_t u, int ctas) {
  if (total < (1 << 22))
    return static_cast<int>(((static_cast<uint32_t>(u) + 1u) * static_cast<uint32_t>(ctas) - 1u) / static_cast<uint32_t>(total));
  return static_cast<int>(((u + 1) * ctas - 1) / total);
}

// A CTA's part, block after block
struct Walk {
  int64_t u, end, base;
  int b, slot;
  __device__ __forceinline__ Walk(const Params& p, int cta) {
    const int64_t total = total_units(p);
    const int ctas = ctas_of(p, total);
    u = first_unit(total, cta, ctas);
    end = cta < ctas ? first_unit(total, cta + 1, ctas) : u;
    slot = 0;
    b = 0;
    base = 0;
    if (u < end) {
      const Where w = where_is(p, u);
      b = w.b;
      base = w.base;
    }
  }
  __device__ __forceinline__ bool more() const { return u < end; }
};
struct Block {
  Seq sq;
  int b, kvh, mb;
  int t0, t1;   // units
  bool whole;   // all of the block's
  int slot;     // of the workspace, where not
};
__device__ __forceinline__ Block next_block(const Params& p, Walk& w) {
  Block k;
  k.b = w.b;
  k.sq = seq_of(p, w.b);
  const int units = units_of(k.sq);
  const int64_t at = w.u - w.base;
  int item;
  if (at < (1LL << 31)) {
    item = static_cast<int>(at) / units;
    k.t0 = static_cast<int>(at) % units;
  } else {
    item = static_cast<int>(at / units);
    k.t0 = static_cast<int>(at % units);
  }
  const int64_t left = w.end - w.u;
  k.t1 = left < units - k.t0 ? k.t0 + static_cast<int>(left) : units;
  k.kvh = item / p.mblocks;
  k.mb = item % p.mblocks;
  k.whole = k.t0 == 0 && k.t1 == units;
  k.slot = w.slot;
  w.slot = 1;
  w.u += k.t1 - k.t0;
  if (k.t1 == units && item + 1 == p.per) {
    w.base += static_cast<int64_t>(units) * p.per;
    ++w.b;
  }
  return k;
}
// where row r of a block that this CTA shares goes in the workspace
__device__ __forceinline__ int64_t part_row(const Params& p, int cta, int slot, int r) {
  return (static_cast<int64_t>(cta) * 2 + slot) * p.block_rows + r;
}

// The scale s of an 8-bit value in the weight.  In bf16 the weight exp2(x - m) s has f32's range, and
// f = s.  In f16 a weight times a small scale would leave the type's range, so s = 2^e f, 1 <= |f| < 2, and 2^e
// goes with the score: with y = x + e and m the largest y among the keys that the row sees,
//   sum_j exp2(x_j) s_j v_j = 2^m sum_j (exp2(y_j - m) f_j) v_j,   sum_j exp2(x_j) = 2^m sum_j exp2(y_j - m) 2^-e_j,
// where the largest rounded weight is 1 or more whatever the scales, and a key that the row does not see
// has no say.  (A power of two near the largest scale of a tile, the same for all rows, let a large value
// that a row did not see take the bits of that row's weights; us with it and so, heads 32 over 8, D 128: 24 ragged
// caches of 8192, one token 66.7 and 68.3; 16 of 4096, 16 nodes 82 and 78; 8 of 16384, 64 nodes 225 and 222.)
// e is held within kLow .. kHigh, so that a weight that is lost in f32 beside the largest, 2^-126 of it, is lost in the
// sum's 24 bits, too: kHigh - kLow + 24 <= 126.  Values with scales below 2^kLow are nothing in f16; a scale from
// 2^(kHigh + 7) on may give an infinity (a weight in f16 is up to 2^8 times 2^7 times the fraction).
// Where a mask may hide the key, a value's scale that is infinite or NaN makes the score NaN instead of the
// weight, and with it the rows that see the key; the mask comes after that.
constexpr int kLow = -60, kHigh = 40;
struct ValueScale {
  float rest, lift, lower;  // f, e, 2^-e
};
template <bool NORM>
__device__ __forceinline__ ValueScale value_scale(float s) {
  ValueScale x{s, 0.0f, 1.0f};
  if constexpr (NORM) {
    constexpr uint32_t low = static_cast<uint32_t>(127 + kLow) << 23, high = static_cast<uint32_t>(127 + kHigh) << 23;
    const uint32_t e = min(max(__float_as_uint(s) & 0x7f800000u, low), high);
    x.lift = __uint_as_float(0x4b000000u + (e >> 23)) - 8388735.0f;  // 2^23 + 127 + e, less 2^23 + 127
    x.lower = __uint_as_float((254u << 23) - e);
    x.rest = s * x.lower;
  }
  return x;
}

int launch_dec(const Params& p, int dtype, int D, cudaStream_t s);
int launch_f32(const Params& p, int D, bool few, cudaStream_t s);
int launch_tc_f16(const Params& p, int D, cudaStream_t s);
int launch_tc_bf16(const Params& p, int D, cudaStream_t s);

}  // namespace tree
}  // namespace fpk
