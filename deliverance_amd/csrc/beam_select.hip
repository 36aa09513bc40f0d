// The choice of beam search, on the device: of every group of B beams the K pairs (beam, token) with the largest summed
// log-probability, in descending order, the lowest beam * V + token first among equals.
//
//   key(b, v) = score[b] + ((z[b, v] - max_b) - log sum_v exp(z[b, v] - max_b))
//
// A logit that is -inf or no number is never chosen and adds nothing to the sum; a score that is -inf or no number marks a
// place without a beam; where the largest logit is infinite, the entries that reach it share the probability.  Keys are 64-bit: a
// 32-bit sum of a score near -100 and a logit makes neighbouring logits equal.  The terms of the sum are 32-bit exponentials,
// summed in 64-bit.
//
// Two kernels.  beam_stats_kernel crosses the logits once: a wavefront takes 8 segments of 256 logits of a row and leaves each
// segment's largest logit and, for the 2,048 together, their maximum and sum.  beam_choose_kernel, one workgroup a group, works on
// what is left: the K best entries lie in the K segments with the best largest entries (among equal ones the first), so it
// chooses K segments and then K entries of those.
#include "common.h"

#define BEAM_MAX 64              // beams of a group
#define BEAM_MAX_KEEP 128        // candidates of a group
#define SEG 256                  // logits of a segment: 64 lanes, 4 each
#define SEGS_A_WAVE 8
#define PART (SEG * SEGS_A_WAVE)
#define STATS_WAVES 4
#define CHOOSE_THREADS 1024
#define CHOOSE_WAVES (CHOOSE_THREADS / DA_WAVE)
#define LIST 512                 // entries that may be ranked by counting

// a 64-bit number that orders like the key; 0 for one that is never chosen
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return !(v > -INFINITY) ? 0 : ((u >> 63) ? ~u : (u | 0x8000000000000000ull));
}
__device__ __forceinline__ double unordered64(uint64_t k) {
  return __builtin_bit_cast(double, (k >> 63) ? (k & 0x7fffffffffffffffull) : ~k);
}

__device__ __forceinline__ float clean(float z) { return z == z ? z : -INFINITY; }
// z - top, also where both are infinite
__device__ __forceinline__ float below(float z, float top) { return z == top ? 0.f : z - top; }

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));

__global__ void __launch_bounds__(STATS_WAVES * DA_WAVE)
beam_stats_kernel(const float* __restrict__ logits, long ldl, int V, int n_segs, int n_parts, float* __restrict__ seg_max,
                  float* __restrict__ part_max, double* __restrict__ part_sum) {
  const int lane = threadIdx.x % DA_WAVE, part = blockIdx.x * STATS_WAVES + threadIdx.x / DA_WAVE, row = blockIdx.y;
  if (part >= n_parts) return;
  const float* z = logits + (size_t)row * ldl;
  const int v0 = part * PART;
  float x[SEGS_A_WAVE][4];
#pragma unroll
  for (int s = 0; s < SEGS_A_WAVE; ++s) {
    const int v = v0 + s * SEG + 4 * lane;
    if (v + 4 <= V) {
      const float4_any f = *(const float4_any*)(z + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s][e] = clean(f[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s][e] = v + e < V ? clean(z[v + e]) : -INFINITY;
    }
  }
  float top = -INFINITY;
#pragma unroll
  for (int s = 0; s < SEGS_A_WAVE; ++s) {
    const float m = wave_max(fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3])));
    if (lane == 0 && v0 + s * SEG < V) seg_max[(size_t)row * n_segs + part * SEGS_A_WAVE + s] = m;
    top = fmaxf(top, m);
  }
  double sum = 0.0;
#pragma unroll
  for (int s = 0; s < SEGS_A_WAVE; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (x[s][e] > -INFINITY) sum += (double)expf(below(x[s][e], top));
  sum = wave_sum_d(sum);
  if (lane == 0) {
    part_max[(size_t)row * n_parts + part] = top;
    part_sum[(size_t)row * n_parts + part] = sum;
  }
}

struct Chosen {
  uint64_t key;
  int at;
};

// The workgroup's n entries (entry i has key(i), 0: none) cut down to a list in LDS that surely holds the `keep` best, the first
// among equals; returns the list's length.  `least`: a key that at least `keep` entries reach, or 1.
template <class Key>
__device__ int shortlist(int n, int keep, uint64_t least, Key key, Chosen* list, int* counts, int* length) {
  const int t = threadIdx.x, wave = t / DA_WAVE, lane = t % DA_WAVE;
  auto count = [&](auto pred) {
    int c = 0;
    for (int i = t; i < n; i += CHOOSE_THREADS) c += pred(key(i), i) ? 1 : 0;
    c = wave_sum_i(c);
    __syncthreads();
    if (lane == 0) counts[wave] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < CHOOSE_WAVES; ++w) c += counts[w];
    return c;
  };
  uint64_t lo = least;                                 // at least `keep` entries (or all there are) have lo <= key
  int last = n, c = count([&](uint64_t k, int) { return k >= lo; });
  if (c > LIST) {
    uint64_t hi = 0xffffffffffffffffull;               // fewer than `keep` have hi <= key
    while (c > LIST && hi - lo > 1) {
      const uint64_t mid = lo + (hi - lo) / 2;
      const int m = count([&](uint64_t k, int) { return k >= mid; });
      if (m >= keep) { lo = mid; c = m; }
      else hi = mid;
    }
    if (c > LIST) {                                    // many equal ones: the first of them
      int a = 0;                                       // entries equal to lo with a place of at most `last` are enough, with one below a not
      last = n - 1;
      while (a < last) {
        const int mid = a + (last - a) / 2;
        const int m = count([&](uint64_t k, int i) { return k > lo || (k == lo && i <= mid); });
        if (m >= keep) last = mid;
        else a = mid + 1;
      }
    }
  }
  if (t == 0) *length = 0;
  __syncthreads();
  for (int i = t; i < n; i += CHOOSE_THREADS) {
    const uint64_t k = key(i);
    if (k > lo || (k == lo && i <= last)) {
      const int at = atomicAdd(length, 1);
      list[at].key = k;
      list[at].at = i;
    }
  }
  __syncthreads();
  return *length;
}

// how many entries of the list stand before entry t
__device__ __forceinline__ int rank_of(const Chosen* list, int length, const Chosen& mine) {
  int r = 0;
  for (int j = 0; j < length; ++j) r += list[j].key > mine.key || (list[j].key == mine.key && list[j].at < mine.at);
  return r;
}

__global__ void __launch_bounds__(CHOOSE_THREADS)
beam_choose_kernel(const float* __restrict__ logits, long ldl, int V, int B, int K, const float* __restrict__ scores, int n_segs,
                   int n_parts, const float* __restrict__ seg_max, const float* __restrict__ part_max, const double* __restrict__ part_sum,
                   float* __restrict__ out_score, int* __restrict__ out_parent, int* __restrict__ out_token) {
  __shared__ double base[BEAM_MAX], logsum[BEAM_MAX];     // the score; the logarithm of the sum (-inf: no beam)
  __shared__ float top[BEAM_MAX];
  __shared__ Chosen list[LIST];
  __shared__ int counts[CHOOSE_WAVES], length[1], segs[BEAM_MAX_KEEP];
  __shared__ uint64_t least[1];
  const int g = blockIdx.x, t = threadIdx.x, wave = t / DA_WAVE, lane = t % DA_WAVE;
  const size_t row0 = (size_t)g * B;

  // ---- each row's maximum and the logarithm of its sum
  for (int b = wave; b < B; b += CHOOSE_WAVES) {
    const float* pm = part_max + (row0 + b) * n_parts;
    const double* ps = part_sum + (row0 + b) * n_parts;
    float m = -INFINITY;
    for (int i = lane; i < n_parts; i += DA_WAVE) m = fmaxf(m, pm[i]);
    m = wave_max(m);
    double s = 0.0;
    for (int i = lane; i < n_parts; i += DA_WAVE)
      if (pm[i] > -INFINITY) s += ps[i] * exp((double)below(pm[i], m));
    s = wave_sum_d(s);
    if (lane == 0) {
      const float sc = scores[row0 + b];
      top[b] = m;
      base[b] = (m > -INFINITY && sc == sc) ? (double)sc : -INFINITY;
      logsum[b] = s > 0.0 ? log(s) : 0.0;
    }
  }
  __syncthreads();
  auto key_of = [&](int b, float z) {
    const double x = z == top[b] ? 0.0 : (double)z - (double)top[b];
    return ordered64(base[b] + (x - logsum[b]));
  };

  // ---- K segments
  auto seg_key = [&](int i) { return key_of(i / n_segs, seg_max[row0 * n_segs + i]); };
  int n = shortlist(B * n_segs, K, 1, seg_key, list, counts, length);
  if (t == 0) *least = 1;
  __syncthreads();
  if (t < n) {
    const Chosen seg = list[t];
    const int r = rank_of(list, n, seg);
    if (r < K) segs[r] = seg.at;
    if (r == K - 1) *least = seg.key;                  // K entries of these segments reach it
  }
  __syncthreads();
  const int kept = n < K ? n : K;
  const uint64_t floor_key = *least;
  // in the order of their places, so that entry i + 1 of theirs stands behind entry i
  int mine = 0, behind = 0;
  if (t < kept) {
    mine = segs[t];
    for (int j = 0; j < kept; ++j) behind += segs[j] < mine;
  }
  __syncthreads();
  if (t < kept) segs[behind] = mine;

  // ---- K entries of them; a place is beam * V + token
  auto place_of = [&](int i) {
    const int at = segs[i / SEG], b = at / n_segs, v = (at - b * n_segs) * SEG + i % SEG;
    return v < V ? b * V + v : -1;
  };
  auto entry_key = [&](int i) -> uint64_t {
    const int p = place_of(i);
    if (p < 0) return 0;
    const int b = p / V;
    return key_of(b, clean(logits[(row0 + b) * ldl + (p - b * V)]));
  };
  __syncthreads();
  n = shortlist(kept * SEG, K, floor_key, entry_key, list, counts, length);
  if (t < n) {
    const Chosen entry = list[t];
    const int r = rank_of(list, n, entry), p = place_of(entry.at);
    if (r < K) {
      out_score[(size_t)g * K + r] = (float)unordered64(entry.key);
      out_parent[(size_t)g * K + r] = p / V;
      out_token[(size_t)g * K + r] = p % V;
    }
  }
  if (t >= n && t < K) {
    out_score[(size_t)g * K + t] = -INFINITY;
    out_parent[(size_t)g * K + t] = -1;
    out_token[(size_t)g * K + t] = -1;
  }
}

static long beam_parts(int V) { return ((long)V + PART - 1) / PART; }
static long beam_segs(int V) { return ((long)V + SEG - 1) / SEG; }

// Scratch of a call, in 32-bit words: the parts' sums (64-bit) and maxima, and the segments' maxima.
extern "C" int da_beam_select_words(int rows, int V) {
  if (rows < 0 || V <= 0) return -1;
  const long words = (long)rows * (3 * beam_parts(V) + beam_segs(V));
  return words > 0x7fffffffL ? -1 : (int)words;
}

extern "C" int da_beam_select(const float* logits, long ldl, int G, int B, int V, const float* scores, int K, float* out_score,
                              int* out_parent, int* out_token, float* scratch, long scratch_words, void* stream) {
  DA_REQUIRE(G >= 0 && B > 0 && B <= BEAM_MAX && V > 0 && ldl >= V && (long)B * V <= 0x7fffffffL,
             "beam_select: bad sizes (groups=%d beams=%d vocabulary=%d row length %ld; at most %d beams)", G, B, V, ldl, BEAM_MAX);
  DA_REQUIRE(K > 0 && K <= BEAM_MAX_KEEP, "beam_select: %d candidates (1 to %d)", K, BEAM_MAX_KEEP);
  if (G == 0) return 0;
  const int n_parts = (int)beam_parts(V), n_segs = (int)beam_segs(V);
  const long rows = (long)G * B, words = rows * (3L * n_parts + n_segs);
  DA_REQUIRE(rows <= 65535, "beam_select: %ld rows (at most 65,535)", rows);
  DA_REQUIRE(scratch && (uintptr_t)scratch % 8 == 0 && scratch_words >= words, "beam_select: %ld words of scratch on 8 bytes are needed, found %ld", words, scratch_words);
  double* part_sum = (double*)scratch;
  float* part_max = scratch + 2 * rows * n_parts;
  float* seg_max = part_max + rows * n_parts;
  hipLaunchKernelGGL(beam_stats_kernel, dim3(da_ceil_div(n_parts, STATS_WAVES), (unsigned)rows), dim3(STATS_WAVES * DA_WAVE), 0,
                     (hipStream_t)stream, logits, ldl, V, n_segs, n_parts, seg_max, part_max, part_sum);
  DA_CHECK_LAUNCH("beam_select (sums)");
  hipLaunchKernelGGL(beam_choose_kernel, dim3(G), dim3(CHOOSE_THREADS), 0, (hipStream_t)stream, logits, ldl, V, B, K, scores, n_segs, n_parts,
                     seg_max, part_max, part_sum, out_score, out_parent, out_token);
  DA_CHECK_LAUNCH("beam_select (choice)");
  return 0;
}
