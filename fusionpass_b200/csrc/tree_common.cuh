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
  float* part_o;             // [rows][splits][D] unnormalised partial results
  float2* part_ml;           // [rows][splits] (running maximum of base 2, sum)
  int64_t parents_st;
  int64_t q_st[3], k_st[3], v_st[3], o_st[3], ks_st[3], vs_st[3];
  int32_t batch, heads, kv_heads, group, nodes, room;
  int32_t splits, items, mblocks;
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

int launch_dec(const Params& p, int dtype, int D, cudaStream_t s);
int launch_f32(const Params& p, int D, bool few, cudaStream_t s);

}  // namespace tree
}  // namespace fpk
