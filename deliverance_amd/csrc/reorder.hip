// Rows of many tensors reordered in place: of every group of B places, the row of place b becomes what the row of place
// parent[b] was, in every tensor.  (What the beams of a search keep, pages of keys and values that are being written and
// recurrent states, follows the beams that were chosen.)
//
// A thread holds one column of a row for all places of a group: it reads the columns of the rows that move, all of them, and only
// then writes.  No other thread touches its columns, so parents may be any permutation, with repeats, and no copy is made.
// Rows that stay are neither read nor written.
//
// Bound by memory: every row that moves is read and written once.  Loads and stores go past the caches: 8 x 8 beams' pages of 48
// layers of 25 heads, 315 MB, take 62.9 us (5.0 TB/s, a large copy 5.13) and 98 with ordinary ones, states of 543 MB 112 and
// 207; two columns a thread are behind (64.9, 117).  Above 16 places a column is 4 bytes, at the same rate (2 x 32 places of those pages 58.9 us, 1 x 64 60.9);
// rows of an odd number of 2-byte units go by those (8 x 8 places 421, 2 x 32 198).
#include "common.h"
#include <da_anew.h>

#define REORDER_TENSORS 96       // of a launch (the table is a kernel argument: nothing is uploaded, a recorded launch keeps it)
#define REORDER_MAX 64           // places of a group
#define REORDER_THREADS 256

// (The columns travel as structures: of vectors that are only sometimes loaded the compiler makes copies, and waits for each load: 101 us for 63.5.
// A row may begin on any 4 bytes.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename U> __device__ __forceinline__ U load_past(const U* p) { return __builtin_nontemporal_load(p); }
template <typename U> __device__ __forceinline__ void store_past(U* p, U v) { __builtin_nontemporal_store(v, p); }
template <> __device__ __forceinline__ uint4 load_past<uint4>(const uint4* p) {
  const u32x4 x = __builtin_nontemporal_load((const u32x4*)p);
  return make_uint4(x[0], x[1], x[2], x[3]);
}
template <> __device__ __forceinline__ void store_past<uint4>(uint4* p, uint4 v) {
  const u32x4 x = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(x, (u32x4*)p);
}
// (a use of what was loaded: the wait for the loads stands here, once, and not in front of every store, where it would wait for the stores too)
template <typename U> __device__ __forceinline__ void arrived(U& v) { v = (U)da_anew((uint32_t)v); }
template <> __device__ __forceinline__ void arrived<uint4>(uint4& v) { v.x = da_anew(v.x); }
// the words behind the last 16 bytes of a row, one a thread
template <typename U> __device__ __forceinline__ U load_word(const char*) { return U(); }
template <> __device__ __forceinline__ uint4 load_word<uint4>(const char* p) { return make_uint4(load_past((const uint32_t*)p), 0, 0, 0); }
template <typename U> __device__ __forceinline__ void store_word(char*, U) {}
template <> __device__ __forceinline__ void store_word<uint4>(char* p, uint4 v) { store_past((uint32_t*)p, v.x); }

struct ReorderTable {
  void* data[REORDER_TENSORS];
  int bytes[REORDER_TENSORS];    // of a row
};

// NB: places that a thread has registers for
template <typename U, int NB>
__global__ void __launch_bounds__(REORDER_THREADS)
reorder_kernel(const ReorderTable table, const int* __restrict__ slots, const int* __restrict__ parents, int B, int pool) {
  const int bytes = table.bytes[blockIdx.y], whole = bytes / (int)sizeof(U), units = whole + bytes % (int)sizeof(U) / 4;
  if (blockIdx.x * REORDER_THREADS >= (unsigned)units) return;
  // a place a lane: where its row comes from (-1: it stays) and where it is
  const int lane = threadIdx.x % DA_WAVE, at = (int)blockIdx.z * B + (lane < B ? lane : 0);
  const int parent = parents[at], slot = slots[at];
  int from = __shfl(slot, (unsigned)parent < (unsigned)B ? parent : lane, DA_WAVE);
  if (lane >= B || parent == lane || (unsigned)parent >= (unsigned)B || (unsigned)slot >= (unsigned)pool || (unsigned)from >= (unsigned)pool || from == slot) from = -1;
  if (__builtin_amdgcn_ballot_w64(from >= 0) == 0) return;
  const int c = blockIdx.x * REORDER_THREADS + threadIdx.x;
  const bool in = c < units, word = c >= whole;           // (all lanes stay: each is asked for its place)
  char* data = (char*)table.data[blockIdx.y] + (word ? (size_t)whole * sizeof(U) + (size_t)(c - whole) * 4 : (size_t)c * sizeof(U));
  U v[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int f = __builtin_amdgcn_readlane(from, b);
    if (f >= 0 && in) v[b] = word ? load_word<U>(data + (size_t)f * bytes) : load_past((const U*)(data + (size_t)f * bytes));
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) arrived(v[b]);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int f = __builtin_amdgcn_readlane(from, b), to = __builtin_amdgcn_readlane(slot, b);
    if (f >= 0 && in) {
      if (word) store_word(data + (size_t)to * bytes, v[b]);
      else store_past((U*)(data + (size_t)to * bytes), v[b]);
    }
  }
}

// n tensors [layers, pool, row]: a host array of three numbers each, their address, their row's bytes (even) and layers.
extern "C" int da_state_reorder(const long* tensors, int n, int pool, const int* slots, const int* parents, int G, int B, void* stream) {
  auto data = [&](int i) { return (char*)tensors[3 * i]; };
  auto row_bytes = [&](int i) { return tensors[3 * i + 1]; };
  auto layers = [&](int i) { return tensors[3 * i + 2]; };
  DA_REQUIRE(n >= 0 && G >= 0 && G <= 65535 && B > 0 && B <= REORDER_MAX && pool >= 0,
             "state_reorder: bad sizes (tensors=%d rows=%d groups=%d places=%d; at most %d places)", n, pool, G, B, REORDER_MAX);
  for (int i = 0; i < n; ++i)
    DA_REQUIRE(row_bytes(i) > 0 && row_bytes(i) % 2 == 0 && row_bytes(i) < (1L << 31) && (uintptr_t)data(i) % 2 == 0 && layers(i) >= 0,
               "state_reorder: %ld layers with a row of %ld bytes: not whole 2-byte units, or too long", layers(i), row_bytes(i));
  if (n == 0 || G == 0 || B == 1 || pool == 0) return 0;
  auto unit_of = [&](int i) {
    const uintptr_t odd = (uintptr_t)data(i) | (uintptr_t)row_bytes(i);
    return odd % 4 ? 2 : (B <= 16 ? 16 : 4);
  };
  for (int unit = 16; unit > 1; unit = unit == 16 ? 4 : unit - 2) {      // 16, 4, 2
    ReorderTable table;
    int count = 0, longest = 0;
    auto launch = [&]() {
      if (!count) return;
      hipStream_t s = (hipStream_t)stream;
      const dim3 block(REORDER_THREADS);
#define DA_REORDER(U, NB) \
  hipLaunchKernelGGL((reorder_kernel<U, NB>), dim3(da_ceil_div(longest, REORDER_THREADS), count, G), block, 0, s, table, slots, parents, B, pool)
      if (unit == 16 && B <= 4) DA_REORDER(uint4, 4);
      else if (unit == 16 && B <= 8) DA_REORDER(uint4, 8);
      else if (unit == 16) DA_REORDER(uint4, 16);
      else if (unit == 4) DA_REORDER(uint32_t, 64);
      else DA_REORDER(uint16_t, 64);
#undef DA_REORDER
      count = longest = 0;
    };
    for (int i = 0; i < n; ++i) {
      if (unit_of(i) != unit) continue;
      for (long layer = 0; layer < layers(i); ++layer) {
        table.data[count] = data(i) + layer * pool * row_bytes(i);
        table.bytes[count] = (int)row_bytes(i);
        const int units = (int)(row_bytes(i) / unit) + (unit == 16 ? (int)(row_bytes(i) % 16 / 4) : 0);
        longest = units > longest ? units : longest;
        if (++count == REORDER_TENSORS) launch();
      }
    }
    launch();
    DA_CHECK_LAUNCH("state_reorder");
  }
  return 0;
}
