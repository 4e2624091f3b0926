// Drafted-token trees over the paged KV cache: step bookkeeping, attention
// and commit on device-side lengths and tables (include/tvara_kernels.h).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "common.hpp"

namespace tvara {

constexpr int kTreeMaxSeq = 8192;
constexpr int kTreeMaxNodes = 1024;

// Bits of the caller's status word (TVARA_TREE_* of the public header).
enum { kTreeBadBlock = 1, kTreeBadLengths = 2, kTreeNoBlocks = 4, kTreeBadParent = 8, kTreeTimeout = 16 };

struct TreePlan {
    int bt = 0, n_seq = 0, capacity = 0, max_nodes = 0, words = 0, max_blocks = 0, stride = 0, free_capacity = 0;
    const int* lengths = nullptr;
    const int* held = nullptr;
    const int* cu = nullptr;
    const int* parents = nullptr;
    const int* free_blocks = nullptr;
    const int* free_count = nullptr;
    int* tables = nullptr;
    long long* slots = nullptr;
    int* positions = nullptr;
    unsigned long long* ancestors = nullptr;
    int* held_out = nullptr;
    int* free_left = nullptr;
    int* status = nullptr;
};
void launch_tree_plan(const TreePlan& a, cudaStream_t s);

struct TreeAttn {
    int kv_kind = 0;  // 0 F32, 1 F16, 2 int8 with row scales
    int hq = 0, hkv = 0, group = 1, dim = 0, bt = 0;  // group = hq / hkv
    int n_seq = 0, capacity = 0, max_nodes = 0, words = 0, max_blocks = 0, stride = 0;
    unsigned long long bt_inverse = 0;  // 2^64 / bt rounded up, 0 for bt 1
    long long ldq = 0, ldo = 0;
    long long block_rows = 0, layer_rows = 0, kind_rows = 0;  // rows of dim elements: a block, to the layer, K to V
    int box_rows = 0;  // rows of a TMA box, 0: no TMA
    const float* q = nullptr;
    float* out = nullptr;
    const void* kv = nullptr;
    const float* scales = nullptr;
    const int* tables = nullptr;
    const int* lengths = nullptr;
    const int* cu = nullptr;
    const long long* slots = nullptr;
    const unsigned long long* ancestors = nullptr;
    int* status = nullptr;
};
std::size_t tree_attention_workspace(const TreeAttn& a);
void launch_tree_attention(const TreeAttn& a, void* workspace, cudaStream_t s);

struct TreeCommit {
    int elem = 4;  // bytes of a pool element
    int hkv = 0, dim = 0, bt = 0, layers = 0, n_seq = 0, capacity = 0, max_nodes = 0, max_blocks = 0;
    const int* lengths = nullptr;
    const int* cu = nullptr;
    const int* parents = nullptr;
    const unsigned* tokens = nullptr;
    const unsigned* choices = nullptr;
    const unsigned* first = nullptr;
    const long long* slots = nullptr;
    const long long* dest = nullptr;
    void* pool = nullptr;
    float* scales = nullptr;
    int* path = nullptr;
    int* accepted = nullptr;
    unsigned* next = nullptr;
    int* lengths_out = nullptr;
    int* status = nullptr;
};
void launch_tree_commit(const TreeCommit& a, cudaStream_t s);

}  // namespace tvara
