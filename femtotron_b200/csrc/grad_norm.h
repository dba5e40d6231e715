// Global norm over many tensors and their scaling by one factor.
//
//     norm = sqrt(sum over all tensors of x^2),   clipped: y = x min(1, max_norm / (norm + 1e-6))
//
// The tensors' addresses travel in the kernel's parameters (a table of up to 1024 of them per launch): no copy
// to the device, nothing pinned, and a captured graph holds its own.  Every block takes one run of chunks in
// the order of the list, so the sum's order depends on the sizes alone; squares of eight values are summed in
// fp32 and go on in fp64, or in fp64 throughout where fp32 would over- or underflow.  The blocks that
// scale add the partial sums up by themselves, all in the same order: no launch in between, no counter.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ft {
namespace gn {

constexpr int MAX_TENSORS = 1024;  // 30 bytes of parameters each, of the 32764 that a launch has
constexpr int CHUNK = 8192;        // values
constexpr int MAX_SLOTS = 8;
enum Type : uint8_t { F32 = 0, BF16 = 1, F16 = 2 };

template <int N>
struct Table {
  const void* x[N];
  void* y[N];
  int64_t n[N];
  int chunk_end[N];    // chunks of this tensor and those before it
  uint8_t type[N], slot[N];
  int count, chunks;
};

// Partial sums [blocks][n_slots] of one table, and how many blocks a table of so many chunks is given.
int sumsq_blocks(int chunks);
template <int N>
cudaError_t launch_sumsq(const Table<N>& t, int n_slots, double* partial, cudaStream_t st);
cudaError_t launch_finish(const double* partial, int blocks, int n_slots, double* sums, cudaStream_t st);

struct Factor {
  const float* coef;       // the factor itself, or null:
  const double* partial;   // the partial sums of all tables (one slot),
  int blocks;
  float max_norm;          // from which it follows;
  float* norm;             // then the norm is written here
  bool in_place;           // a factor of 1 leaves everything as it is
};
static_assert(sizeof(Table<MAX_TENSORS>) + sizeof(Factor) <= 32764, "parameters of a launch");
template <int N>
cudaError_t launch_scale(const Table<N>& t, const Factor& f, cudaStream_t st);

}  // namespace gn
}  // namespace ft
