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
// Two kernels.  beam_stats_kernel crosses the logits once: a wavefront takes 2 or 8 segments of 256 logits of a row and leaves each
// segment's largest logit and, for all of them, the maximum and the sum.  beam_choose_kernel, one workgroup a group, works on
// what is left.  It finds a key that K entries surely reach, the K-th best of the largest keys of 256 groups of segments (about K + K^2 / 512
// segments reach it, where their keys come in any order), reads the segments that reach it again, and puts the entries that reach it in order
// by counting, for each, those in front of it.  Where more reach it than the list holds (equal logits), the key is searched bit by bit, and
// among equal ones the place.
#include "common.h"

#define BEAM_MAX 64              // beams of a group
#define BEAM_MAX_KEEP 128        // candidates of a group
#define SEG 256                  // logits of a segment: 64 lanes, 4 each
#define SEGS_FEW 2               // segments of a wavefront: few logits, or many
#define SEGS_MANY 8
#define STATS_WAVES 4
#define CHOOSE_THREADS 1024
#define CHOOSE_WAVES (CHOOSE_THREADS / DA_WAVE)
#define GROUPS (CHOOSE_THREADS / 4)
#define HELD 2                   // segments whose keys a thread keeps
#define LIST 512                 // segments, and entries, that may be looked at one by one

// a 64-bit number that orders like the key; 0 for one that is never chosen
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return !(v > -INFINITY) ? 0 : ((u >> 63) ? ~u : (u | 0x8000000000000000ull));
}
__device__ __forceinline__ double unordered64(uint64_t k) {
  return __builtin_bit_cast(double, (k >> 63) ? (k & 0x7fffffffffffffffull) : ~k);
}

__device__ __forceinline__ float clean(float z) { return z == z ? z : -INFINITY; }

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));

// e^x of -200 <= x <= 0, a unit in the last place off: the product with log2 e in two parts
__device__ __forceinline__ float exp_near(float x) {
  const float hi = 1.44269502f, lo = 1.92596299e-8f;
  const float p = x * hi, rest = fmaf(x, lo, fmaf(x, hi, -p)), r = __builtin_amdgcn_exp2f(p);
  return fmaf(r, rest * 0.693147181f, r);
}

template <int SEGS>              // of a wavefront
__global__ void __launch_bounds__(STATS_WAVES * DA_WAVE)
beam_stats_kernel(const float* __restrict__ logits, long ldl, int V, int n_segs, int n_parts, float* __restrict__ seg_max,
                  float* __restrict__ part_max, double* __restrict__ part_sum) {
  const int lane = threadIdx.x % DA_WAVE, part = blockIdx.x * STATS_WAVES + threadIdx.x / DA_WAVE, row = blockIdx.y;
  if (part >= n_parts) return;
  const float* z = logits + (size_t)row * ldl;
  const int v0 = part * SEGS * SEG;
  float x[SEGS][4];
  if (v0 + SEGS * SEG <= V) {
#pragma unroll
    for (int s = 0; s < SEGS; ++s) {
      const float4_any f = *(const float4_any*)(z + v0 + s * SEG + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s][e] = f[e];
    }
  } else {
#pragma unroll
    for (int s = 0; s < SEGS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + s * SEG + 4 * lane + e;
        x[s][e] = v < V ? z[v] : -INFINITY;
      }
  }
  float top = -INFINITY, m[SEGS];
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {                        // (the maximum with a number drops what is none)
    m[s] = wave_max(fmaxf(fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3])), -INFINITY));
    top = fmaxf(top, m[s]);
  }
  float best = m[0];
#pragma unroll
  for (int s = 1; s < SEGS; ++s) best = lane == s ? m[s] : best;
  if (lane < SEGS && v0 + lane * SEG < V) seg_max[(size_t)row * n_segs + part * SEGS + lane] = best;
  double sum = 0.0;
  const bool infinite = top == INFINITY;
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {
    float e4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (what is no number, or -inf, or belongs to a part without entries: -200, whose exponential is 0)
      float d = infinite ? (x[s][e] == top ? 0.f : -200.f) : x[s][e] - top;
      e4[e] = exp_near(fmaxf(d, -200.f));
    }
    sum += (double)((e4[0] + e4[1]) + (e4[2] + e4[3]));
  }
  sum = wave_sum_d(sum);
  if (lane == 0) {
    part_max[(size_t)row * n_parts + part] = top;
    part_sum[(size_t)row * n_parts + part] = sum;
  }
}

struct Chosen {
  uint64_t key;
  int place;
};

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  const uint32_t lo = (uint32_t)dpp_move_i<CTRL, 0xF>((int)v, (int)v), hi = (uint32_t)dpp_move_i<CTRL, 0xF>((int)(v >> 32), (int)(v >> 32));
  return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ bool stands(uint64_t key, int place, uint64_t least, int last) { return key > least || (key == least && place <= last); }

// (least, last) moved up until at most LIST entries stand, and still `keep`: first by the key, then, where more are equal, by
// the place.  count(least, last): how many stand, the same in all threads.
template <class Count>
__device__ void narrow(uint64_t& least, int& last, int keep, Count count) {
  uint64_t hi = 0xffffffffffffffffull;                 // fewer than `keep` reach it
  int c = LIST + 1;
  while (c > LIST && hi - least > 1) {
    const uint64_t mid = least + (hi - least) / 2;
    const int m = count(mid, last);
    if (m >= keep) { least = mid; c = m; }
    else hi = mid;
  }
  if (c <= LIST) return;
  for (int a = 0; a < last;) {
    const int mid = a + (last - a) / 2;
    if (count(least, mid) >= keep) last = mid;
    else a = mid + 1;
  }
}

// magic: 2^32 / n_segs rounded up (0: divide), for fewer than 65,536 segments
__global__ void __launch_bounds__(CHOOSE_THREADS)
beam_choose_kernel(const float* __restrict__ logits, long ldl, int V, int B, int K, const float* __restrict__ scores, int n_segs,
                   int n_parts, const float* __restrict__ seg_max, const float* __restrict__ part_max, const double* __restrict__ part_sum,
                   float* __restrict__ out_score, int* __restrict__ out_parent, int* __restrict__ out_token, uint32_t magic) {
  __shared__ double base[BEAM_MAX], logsum[BEAM_MAX];     // the score (-inf: no beam); the logarithm of the sum
  __shared__ float top[BEAM_MAX];
  __shared__ __attribute__((aligned(16))) uint64_t group_best[GROUPS];
  __shared__ Chosen list[LIST];
  __shared__ int segs[LIST], counts[CHOOSE_WAVES], n_list[2];
  __shared__ uint64_t least_of[1];
  const int g = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / DA_WAVE), lane = t % DA_WAVE;
  const size_t row0 = (size_t)g * B;
  const int n = B * n_segs;

  // ---- asked for together: a thread's first segments, and the partial results of the wavefront's first row
  const float* sm = seg_max + row0 * n_segs;
  float zr[HELD];
#pragma unroll
  for (int e = 0; e < HELD; ++e) zr[e] = sm[min(t + e * CHOOSE_THREADS, n - 1)];
  for (int b = wave; b < B; b += CHOOSE_WAVES) {
    const float* pm = part_max + (row0 + b) * n_parts;
    const double* ps = part_sum + (row0 + b) * n_parts;
    const float sc = scores[row0 + b];
    // (a lane past the end takes the last part's maximum again, and no sum)
    const float p0 = pm[min(lane, n_parts - 1)], p1 = pm[min(lane + DA_WAVE, n_parts - 1)];
    const double s0 = ps[min(lane, n_parts - 1)], s1 = ps[min(lane + DA_WAVE, n_parts - 1)];
    float m = fmaxf(p0, p1);
    for (int i = lane + 2 * DA_WAVE; i < n_parts; i += DA_WAVE) m = fmaxf(m, pm[i]);
    m = wave_max(m);
    auto weighed = [&](float p, double s) { return s * (double)expf(p == m ? 0.f : p - m); };      // (a part without entries has the sum 0)
    double s = (lane < n_parts ? weighed(p0, s0) : 0.0) + (lane + DA_WAVE < n_parts ? weighed(p1, s1) : 0.0);
    for (int i = lane + 2 * DA_WAVE; i < n_parts; i += DA_WAVE) s += weighed(pm[i], ps[i]);
    s = wave_sum_d(m > -INFINITY ? s : 0.0);
    if (lane == 0) {
      top[b] = m;
      base[b] = (m > -INFINITY && sc == sc) ? (double)sc : -INFINITY;
      logsum[b] = s > 0.0 ? log(s) : 0.0;
    }
  }
  if (t < 2) n_list[t] = 0;
  if (t == 0) *least_of = 1;
  __syncthreads();
  auto key_of = [&](int b, float z) {
    const double x = z == top[b] ? 0.0 : (double)z - (double)top[b];
    return ordered64(base[b] + (x - logsum[b]));
  };
  auto total = [&](int c) {                               // over the workgroup
    c = wave_sum_i(c);
    __syncthreads();
    if (lane == 0) counts[wave] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < CHOOSE_WAVES; ++w) c += counts[w];
    return c;
  };
  auto row_of = [&](int i) { return magic ? (int)__umulhi((uint32_t)i, magic) : i / n_segs; };

  // ---- a key that K entries reach: the K-th best of the largest keys of GROUPS groups of segments
  uint64_t held[HELD], best = 0;
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    const int i = t + e * CHOOSE_THREADS;
    held[e] = i < n ? key_of(row_of(i), zr[e]) : 0;
    best = larger(best, held[e]);
  }
  for (int i = t + HELD * CHOOSE_THREADS; i < n; i += CHOOSE_THREADS) best = larger(best, key_of(row_of(i), sm[i]));
  auto each_seg = [&](auto f) {
#pragma unroll
    for (int e = 0; e < HELD; ++e) f(held[e], t + e * CHOOSE_THREADS);      // (one past the end has the key 0)
    for (int i = t + HELD * CHOOSE_THREADS; i < n; i += CHOOSE_THREADS) f(key_of(row_of(i), sm[i]), i);
  };
  best = larger(best, dpp_u64<0xB1>(best));               // 4 lanes
  best = larger(best, dpp_u64<0x4E>(best));
  if (lane % 4 == 0) group_best[t / 4] = best;
  __syncthreads();
  {
    // the four threads of a group count, a quarter each, the groups in front of it
    int before = 0;
#pragma unroll 8
    for (int k = 0; k < GROUPS / 4; ++k) {
      const int j = 4 * k + t % 4;
      const uint64_t other = group_best[j];
      before += other > best || (other == best && j < t / 4);
    }
    before += dpp_move_i<0xB1, 0xF>(before, before);
    before += dpp_move_i<0x4E, 0xF>(before, before);
    if (before == K - 1 && best > 1) *least_of = best;    // (the four write the same)
  }
  __syncthreads();
  uint64_t least = *least_of;

  // ---- the segments with an entry that reaches it
  int last = n;
  auto count_segs = [&](uint64_t lo, int at) {
    int c = 0;
    each_seg([&](uint64_t k, int i) { c += stands(k, i, lo, at); });
    return total(c);
  };
  auto list_segs = [&]() {
    each_seg([&](uint64_t k, int i) {
      if (stands(k, i, least, last)) {
        const int at = atomicAdd(&n_list[0], 1);
        if (at < LIST) segs[at] = i;
      }
    });
    __syncthreads();
    return n_list[0];
  };
  int n_found = list_segs();
  if (n_found > LIST) {
    narrow(least, last, K, count_segs);
    __syncthreads();
    if (t == 0) n_list[0] = 0;
    __syncthreads();
    n_found = list_segs();
  }

  // ---- their entries that reach it: a wavefront a segment
  int last_place = 0x7fffffff;
  auto each_entry = [&](auto f) {
    for (int j = wave; j < n_found; j += CHOOSE_WAVES) {
      const int i = __builtin_amdgcn_readfirstlane(segs[j]), b = i / n_segs, v = (i - b * n_segs) * SEG + 4 * lane;
      const float* z = logits + (row0 + b) * ldl + v;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v + e < V ? clean(z[e]) : -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) f(key_of(b, x[e]), b * V + v + e);
    }
  };
  auto list_entries = [&]() {
    each_entry([&](uint64_t k, int place) {
      if (stands(k, place, least, last_place)) {
        const int at = atomicAdd(&n_list[1], 1);
        if (at < LIST) list[at] = Chosen{k, place};
      }
    });
    __syncthreads();
    return n_list[1];
  };
  int n_entries = list_entries();
  if (n_entries > LIST) {
    narrow(least, last_place, K, [&](uint64_t lo, int at) {
      int c = 0;
      each_entry([&](uint64_t k, int place) { c += stands(k, place, lo, at); });
      return total(c);
    });
    __syncthreads();
    if (t == 0) n_list[1] = 0;
    __syncthreads();
    n_entries = list_entries();
  }

  // ---- in order
  if (t < n_entries) {
    const Chosen mine = list[t];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n_entries; ++j) r += list[j].key > mine.key || (list[j].key == mine.key && list[j].place < mine.place);
    if (r < K) {
      out_score[(size_t)g * K + r] = (float)unordered64(mine.key);
      out_parent[(size_t)g * K + r] = mine.place / V;
      out_token[(size_t)g * K + r] = mine.place % V;
    }
  }
  if (t >= n_entries && t < K) {
    out_score[(size_t)g * K + t] = -INFINITY;
    out_parent[(size_t)g * K + t] = -1;
    out_token[(size_t)g * K + t] = -1;
  }
}

static long beam_segs(int V) { return ((long)V + SEG - 1) / SEG; }
// Few logits: as many wavefronts as there can be; many: fewer partial results.
static int beam_segs_a_wave(long rows, int V) { return rows * beam_segs(V) < 8192 ? SEGS_FEW : SEGS_MANY; }
static long beam_parts(long rows, int V) {
  const int s = beam_segs_a_wave(rows, V);
  return (beam_segs(V) + s - 1) / s;
}

// Scratch of a call, in 32-bit words: the parts' sums (64-bit) and maxima, and the segments' maxima.
extern "C" int da_beam_select_words(int rows, int V) {
  if (rows < 0 || V <= 0) return -1;
  const long words = (long)rows * (3 * beam_parts(rows, V) + beam_segs(V));
  return words > 0x7fffffffL ? -1 : (int)words;
}

extern "C" int da_beam_select(const float* logits, long ldl, int G, int B, int V, const float* scores, int K, float* out_score,
                              int* out_parent, int* out_token, float* scratch, long scratch_words, void* stream) {
  DA_REQUIRE(G >= 0 && B > 0 && B <= BEAM_MAX && V > 0 && ldl >= V && (long)B * V <= 0x7fffffffL,
             "beam_select: bad sizes (groups=%d beams=%d vocabulary=%d row length %ld; at most %d beams)", G, B, V, ldl, BEAM_MAX);
  DA_REQUIRE(K > 0 && K <= BEAM_MAX_KEEP, "beam_select: %d candidates (1 to %d)", K, BEAM_MAX_KEEP);
  if (G == 0) return 0;
  const long rows = (long)G * B;
  const int n_parts = (int)beam_parts(rows, V), n_segs = (int)beam_segs(V);
  const long words = rows * (3L * n_parts + n_segs);
  DA_REQUIRE(rows <= 65535, "beam_select: %ld rows (at most 65,535)", rows);
  DA_REQUIRE(scratch && (uintptr_t)scratch % 8 == 0 && scratch_words >= words, "beam_select: %ld words of scratch on 8 bytes are needed, found %ld", words, scratch_words);
  double* part_sum = (double*)scratch;
  float* part_max = scratch + 2 * rows * n_parts;
  float* seg_max = part_max + rows * n_parts;
  const dim3 grid(da_ceil_div(n_parts, STATS_WAVES), (unsigned)rows), block(STATS_WAVES * DA_WAVE);
  if (beam_segs_a_wave(rows, V) == SEGS_FEW)
    hipLaunchKernelGGL((beam_stats_kernel<SEGS_FEW>), grid, block, 0, (hipStream_t)stream, logits, ldl, V, n_segs, n_parts, seg_max, part_max, part_sum);
  else
    hipLaunchKernelGGL((beam_stats_kernel<SEGS_MANY>), grid, block, 0, (hipStream_t)stream, logits, ldl, V, n_segs, n_parts, seg_max, part_max, part_sum);
  DA_CHECK_LAUNCH("beam_select (sums)");
  // i * magic / 2^32 is i / n_segs while i < 2^16 and n_segs < 2^16: the product's error, i * (magic * n_segs - 2^32) / n_segs / 2^32, is below i / 2^32
  const uint32_t magic = (long)B * n_segs < 65536 && n_segs > 1 ? (uint32_t)(((1ull << 32) + n_segs - 1) / n_segs) : 0;
  hipLaunchKernelGGL(beam_choose_kernel, dim3(G), dim3(CHOOSE_THREADS), 0, (hipStream_t)stream, logits, ldl, V, B, K, scores, n_segs, n_parts,
                     seg_max, part_max, part_sum, out_score, out_parent, out_token, magic);
  DA_CHECK_LAUNCH("beam_select (choice)");
  return 0;
}
