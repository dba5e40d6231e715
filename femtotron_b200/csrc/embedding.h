// Embedding lookup with a factor, and its gradient by sorted tokens.
//
//     out_t = scale w[id_t]  (0 where the id is not in this shard),   dw[v] = scale sum over id_t = v of dout_t
//
// The tokens are sorted by id (stable, so equal ids stay in the order of the batch), the sorted list is cut
// into pieces of 32, and each piece adds up its rows of dout run by run in registers.  A run inside one
// piece goes straight to dw; one that crosses pieces leaves a partial sum per piece, and a second kernel adds
// those up in order.  There are no atomics on values, and the sum's order depends on the ids alone.  The rows of
// a frequent word are added by as many blocks as it has pieces, its partial sums one after the other by one: 32768 tokens added to
// 128256 x 4096 take 251 us with words drawn evenly, 751 with one word in 90 % of the places, 783 with one in all (8192: 104, 169, 159;
// a scatter of atomics on values: 770, 2552, 2765; 198, 646, 697).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ft {
namespace emb {

enum Type : int { F32 = 0, BF16 = 1, F16 = 2 };

struct FwdArgs {
  const void* ids;
  const void* table;
  void* out;
  int64_t T, V, vstart;
  int H, type;
  bool ids64, vec;  // vec: 16-byte accesses
  float scale;
};
cudaError_t launch_fwd(const FwdArgs& a, cudaStream_t st);

// Up to SMALL_SORT tokens are sorted by one block in shared memory: 512 tokens in 7 us, 3001 in 9, 8192 in 28, where three
// kernels per digit take 24, 25 and 29 us and more launches.
constexpr int SMALL_SORT = 8192, SMALL_BITS = 9;
constexpr int SORT_CHUNK = 2048;   // tokens per block of a sorting pass over more tokens
constexpr int MAX_BINS = 1024;
constexpr int PIECE = 32;

struct SortArgs {
  const void* ids;
  bool ids64;
  int64_t vstart, V;
  int T, blocks, bits[4], passes;  // the digits of a key, lowest first
  uint32_t *key[2], *pos[2];       // [T] each, in turn
  uint32_t* counts;                // [bins][blocks]
};
cudaError_t launch_clear(void* x, int64_t bytes, bool beside_sort, cudaStream_t st);
// One launch for T <= SMALL_SORT: key[0] and pos[0] get the result.
cudaError_t launch_small_sort(const SortArgs& a, cudaStream_t st);
// The sorted keys (V for ids of other shards, last) and their places in the batch are in key[passes & 1].
cudaError_t launch_sort(const SortArgs& a, cudaStream_t st);

struct GradArgs {
  const uint32_t *key, *pos;
  const void* dout;     // [T, H]
  void* dw;             // [V, H]
  float* partial;       // [pieces][2][H]: sums of the run that a piece begins with, and of the one it ends with
  int T, H, V, pieces;
  int dout_type, dw_type;
  bool accumulate, vec;
  float scale;
};
cudaError_t launch_grad(const GradArgs& a, cudaStream_t st);

}  // namespace emb
}  // namespace ft
