// Rows of many tensors reordered in place: of every group of B places, the row of place b becomes what the row of place
// parent[b] was, in every tensor.  (What the beams of a search keep, pages of keys and values that are being written and
// recurrent states, follows the beams that were chosen.)
//
// A thread holds one column of a row for all places of a group: it reads the columns of the rows that move, all of them, and only
// then writes.  No other thread touches its columns, so parents may be any permutation, with repeats, and no copy is made.
// Rows that stay are neither read nor written.
#include "common.h"

#define REORDER_TENSORS 96       // of a launch (the table is a kernel argument: nothing is uploaded, a recorded launch keeps it)
#define REORDER_MAX 64           // places of a group
#define REORDER_THREADS 256

struct ReorderTable {
  void* data[REORDER_TENSORS];
  int units[REORDER_TENSORS];    // of a row, 16, 4 or 2 bytes each
};

// NB: places that a thread has registers for; UNITS: columns of a thread
template <typename U, int NB, int UNITS>
__global__ void __launch_bounds__(REORDER_THREADS)
reorder_kernel(const ReorderTable table, const int* __restrict__ slots, const int* __restrict__ parents, int B, int pool) {
  // a place a lane: where its row comes from (-1: it stays) and where it is
  const int lane = threadIdx.x % DA_WAVE, at = (int)blockIdx.z * B + (lane < B ? lane : 0);
  const int parent = parents[at], slot = slots[at];
  const int units = table.units[blockIdx.y];
  int from = __shfl(slot, (unsigned)parent < (unsigned)B ? parent : lane, DA_WAVE);
  if (lane >= B || parent == lane || (unsigned)parent >= (unsigned)B || (unsigned)slot >= (unsigned)pool || (unsigned)from >= (unsigned)pool || from == slot) from = -1;
  if (__builtin_amdgcn_ballot_w64(from >= 0) == 0) return;
  U* data = (U*)table.data[blockIdx.y];
  const int c = blockIdx.x * (REORDER_THREADS * UNITS) + threadIdx.x;
  U v[NB][UNITS];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int f = __builtin_amdgcn_readlane(from, b);
    if (f < 0) continue;
    const U* row = data + (size_t)f * units;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      if (c + u * REORDER_THREADS < units) v[b][u] = row[c + u * REORDER_THREADS];
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (__builtin_amdgcn_readlane(from, b) < 0) continue;
    U* row = data + (size_t)__builtin_amdgcn_readlane(slot, b) * units;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      if (c + u * REORDER_THREADS < units) row[c + u * REORDER_THREADS] = v[b][u];
  }
}

// n tensors [layers, pool, row]; `data`, `row_bytes` (even) and `layers` are host arrays.
extern "C" int da_state_reorder(void* const* data, const long* row_bytes, const int* layers, int n, int pool, const int* slots,
                                const int* parents, int G, int B, void* stream) {
  DA_REQUIRE(n >= 0 && G >= 0 && G <= 65535 && B > 0 && B <= REORDER_MAX && pool >= 0,
             "state_reorder: bad sizes (tensors=%d rows=%d groups=%d places=%d; at most %d places)", n, pool, G, B, REORDER_MAX);
  for (int i = 0; i < n; ++i)
    DA_REQUIRE(row_bytes[i] > 0 && row_bytes[i] % 2 == 0 && row_bytes[i] < (1L << 31) && (uintptr_t)data[i] % 2 == 0 && layers[i] >= 0,
               "state_reorder: %d layers with a row of %ld bytes: not whole 2-byte units, or too long", layers[i], row_bytes[i]);
  if (n == 0 || G == 0 || B == 1 || pool == 0) return 0;
  auto unit_of = [&](int i) {
    const uintptr_t odd = (uintptr_t)data[i] | (uintptr_t)row_bytes[i];
    return B <= 16 && odd % 16 == 0 ? 16 : (odd % 4 == 0 ? 4 : 2);
  };
  for (int unit = 16; unit > 1; unit = unit == 16 ? 4 : unit - 2) {      // 16, 4, 2
    ReorderTable table;
    int count = 0, longest = 0;
    auto launch = [&]() {
      if (!count) return;
      hipStream_t s = (hipStream_t)stream;
      const dim3 block(REORDER_THREADS);
#define DA_REORDER(U, NB, UNITS) \
  hipLaunchKernelGGL((reorder_kernel<U, NB, UNITS>), dim3(da_ceil_div(longest, REORDER_THREADS * UNITS), count, G), block, 0, s, table, slots, parents, B, pool)
      if (unit == 16 && B <= 4) DA_REORDER(uint4, 4, 2);
      else if (unit == 16 && B <= 8) DA_REORDER(uint4, 8, 2);
      else if (unit == 16) DA_REORDER(uint4, 16, 1);
      else if (unit == 4 && B <= 16) DA_REORDER(uint32_t, 16, 2);
      else if (unit == 4) DA_REORDER(uint32_t, 64, 1);
      else DA_REORDER(uint16_t, 64, 1);
#undef DA_REORDER
      count = longest = 0;
    };
    for (int i = 0; i < n; ++i) {
      if (unit_of(i) != unit) continue;
      for (int layer = 0; layer < layers[i]; ++layer) {
        table.data[count] = (char*)data[i] + (long)layer * pool * row_bytes[i];
        table.units[count] = (int)(row_bytes[i] / unit);
        longest = table.units[count] > longest ? table.units[count] : longest;
        if (++count == REORDER_TENSORS) launch();
      }
    }
    launch();
    DA_CHECK_LAUNCH("state_reorder");
  }
  return 0;
}
