// Attention of one new token a beam over the paged cache, for groups of B sequences that begin with the same pages: the keys
// and values of those pages are read once a group.
//
//   o[r] = sum_j softmax_j(scale q[r] . k[j]) v[j]     over the positions lo_r <= j < len_r of row r's sequence
//
// The rows of a group that meet one key head (its B beams, Hq / Hkv query heads each) are the columns of the matrix products, 16 a
// workgroup: up to 16 rows for the bytes of one.  The positions are walked in chunks of 64: chunks that all rows share, then each
// beam's own ones, of which only that beam's columns take part.  The chunks are shared out over the wavefronts of a workgroup and
// over `splits` workgroups, by the launch's shape and the sequences' lengths; their partial results (weighted sums, maximum, sum of
// weights) are joined in LDS and by a second kernel, in a fixed order.
//
//   scores : S^T[key, row] = K[key, :] . q[row, :], 16 keys a product.  A lane receives 4 keys of one row.
//   softmax: a row's running maximum is the same in the four lanes that hold its keys, its sum is theirs alone until the end.
//   values : O^T[d, row] += V^T[d, key] P^T[key, row].  Values lie dimension by dimension, so the left operand is read as it lies;
//            which key stands in which row of the first product is chosen so that a lane's weights are the ones that the second
//            takes from it: nothing is exchanged.
// bfloat16: a 32-bit weight goes in as two bfloat16 parts (16 bits; one part alone would lose as much again as the result's own
// rounding).  32-bit: 16x16x4 products, nothing is rounded.
#include "gemm_common.h"
#include <da_lane_swap.h>

#define BEAMS_MAX 64             // beams of a group
#define BEAMS_MAX_D 256
#define CHUNK 64
#define ROWS 16                  // of a workgroup
#define BEAM_WAVES 4

struct Yes { static const bool value = true; };
struct No { static const bool value = false; };

// 2^x: scores carry log2 e in their scale
__device__ __forceinline__ float exp_of_2(float x) { return __builtin_amdgcn_exp2f(x); }

// Over the four lanes that hold a row's keys
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, DA_WAVE));
  return half_max(v);
}

// Over the wavefront, in every lane
template <class Op>
__device__ __forceinline__ int wave_join(int v, Op op) {
  v = op(v, dpp_move_i<0xB1, 0xF>(v, v));
  v = op(v, dpp_move_i<0x4E, 0xF>(v, v));
  v = op(v, dpp_move_i<0x141, 0xF>(v, v));
  v = op(v, dpp_move_i<0x140, 0xF>(v, v));
  v = op(v, dpp_move_i<0x142, 0xA>(v, v));
  v = op(v, dpp_move_i<0x143, 0xC>(v, v));
  return __builtin_amdgcn_readlane(v, DA_WAVE - 1);
}
// the sum of the lanes up to this one
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_move_i<0x111, 0xF>(0, v);
  v += dpp_move_i<0x112, 0xF>(0, v);
  v += dpp_move_i<0x114, 0xF>(0, v);
  v += dpp_move_i<0x118, 0xF>(0, v);
  v += dpp_move_i<0x142, 0xA>(0, v);
  v += dpp_move_i<0x143, 0xC>(0, v);
  return v;
}

// DK: head size in steps of 32, rounded up to a power of two.  STEP: keys whose loads are under way together.
template <typename T, int DK, int STEP>
__global__ void __launch_bounds__(BEAM_WAVES * DA_WAVE)
attn_beams_kernel(const T* __restrict__ q, int q_ld, const T* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                  const int* __restrict__ seq_lens, const int* __restrict__ shared, int B, int Hq, int Hkv, int D, int page, float scale,
                  int window, T* __restrict__ out, int out_ld, int splits, float* __restrict__ partial) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int DV = 2 * DK, DMAX = 32 * DK;            // value dimensions in steps of 16
  constexpr int QS = F32 ? 2 * DK : DK;                 // key loads a row: 16 dimensions (32-bit) or 32 (bfloat16) a step
  constexpr int KP = STEP / 16;                         // pieces of 16 keys
  constexpr int VP = F32 ? STEP / 16 : STEP / 32;       // value loads a dimension: 4 keys (32-bit) or 8 a lane
  constexpr int SPAN = F32 ? 4 : 8;                     // consecutive keys of a lane
  __shared__ float acc_lds[BEAM_WAVES][DMAX][ROWS + 1];
  __shared__ float m_lds[BEAM_WAVES][ROWS], l_lds[BEAM_WAVES][ROWS];

  const int t = threadIdx.x, lane = t % DA_WAVE, wave = __builtin_amdgcn_readfirstlane(t / DA_WAVE);
  const int col = lane % 16, quad = lane / 16;
  const int ratio = Hq / Hkv, R = B * ratio;
  const int hk = blockIdx.x % Hkv, rb = blockIdx.x / Hkv, g = blockIdx.y, z = blockIdx.z;
  const int r0 = rb * ROWS, s0 = g * B;
  const int b0 = r0 / ratio, b1 = (min(r0 + ROWS, R) - 1) / ratio;      // the beams of these rows
  const int lg = 31 - __builtin_clz(page), pmask = page - 1;
  const uint32_t page_elems = 2u * (uint32_t)(Hkv * page * D);
  const int cap = max_blocks * page;                    // (a longer length would lead out of the table)

  // a beam a lane: its length; then the query rows, the right operand (row r of the group is column r - r0)
  const int n_raw = seq_lens[s0 + (lane < B ? lane : 0)], shared_g = shared[g];
  const int r = r0 + col, rr = min(r, R - 1), beam = rr / ratio, head = hk * ratio + (rr - beam * ratio);
  uint4 qf[QS];
#pragma unroll
  for (int k = 0; k < QS; ++k) {
    const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
    qf[k] = make_uint4(0, 0, 0, 0);
    if (d < D && r < R) qf[k] = *(const uint4*)(q + (size_t)(s0 + beam) * q_ld + (size_t)head * D + d);
  }
  const int n_b = lane < B ? max(0, min(n_raw, cap)) : 0, lo_b = window > 0 ? max(0, n_b - window) : 0;
  const uint64_t alive = __builtin_amdgcn_ballot_w64(n_b > 0);
  const int first_live = alive ? __builtin_ctzll(alive) : 0;
  // shared chunks: those that all beams have in shared pages, and all see from their first position on
  const int common = min(shared_g, wave_join(n_b > 0 ? n_b : 0x7fffffff, [](int a, int b) { return min(a, b); }));
  const int shared0 = alive ? (wave_join(lo_b, [](int a, int b) { return max(a, b); }) + CHUNK - 1) / CHUNK : 0;
  const int shared1 = alive ? max(shared0, common / CHUNK) : 0;
  // a beam's own chunks: from its first one on to its last, without the shared ones
  const int own0 = lo_b / CHUNK, own = lane >= b0 && lane <= b1 && n_b > 0 ? (n_b + CHUNK - 1) / CHUNK - own0 - (shared1 - shared0) : 0;
  const int own_to = wave_scan(own);
  const int n_shared = shared1 - shared0, items = n_shared + __builtin_amdgcn_readlane(own_to, DA_WAVE - 1);
  const int per = (items + splits - 1) / splits;
  const int item0 = z * per, item1 = min(items, item0 + per);
  const int len_of_beam = __shfl(n_b, beam, DA_WAVE), lo = __shfl(lo_b, beam, DA_WAVE), len = r < R ? len_of_beam : 0;
  const float scale2 = scale * 1.4426950408889634f;

  floatx4 acc[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const T* const kbase = cache + (size_t)hk * page * D;
  const T* const vbase = cache + (size_t)(Hkv + hk) * page * D;

  for (int item = item0 + wave; item < item1; item += BEAM_WAVES) {
    // which chunk of whose table (own < 0: of all)
    int chunk = shared0 + item, mine = -1, src = first_live, first = 0, last = 0x7fffffff;
    if (item >= n_shared) {
      const int left = item - n_shared;
      mine = __builtin_popcountll(__builtin_amdgcn_ballot_w64(own_to <= left));
      mine = min(mine, b1);
      chunk = __builtin_amdgcn_readlane(own0, mine) + left - (__builtin_amdgcn_readlane(own_to, mine) - __builtin_amdgcn_readlane(own, mine));
      if (chunk >= shared0) chunk += n_shared;
      src = mine;
      first = max(chunk * CHUNK, __builtin_amdgcn_readlane(lo_b, mine));
      last = min(chunk * CHUNK + CHUNK, __builtin_amdgcn_readlane(n_b, mine)) - 1;
    } else {
      first = chunk * CHUNK;
      last = first + CHUNK - 1;
    }
    const int* bt = block_table + (size_t)(s0 + src) * max_blocks;
    const bool takes = mine < 0 || mine == beam;

    auto step = [&](int h0, auto cut_tag) {
      constexpr bool CUT = decltype(cut_tag)::value;
      // ---- every load of the step, then the arithmetic.  A lane's keys of the first product lie in one group of 8 (bfloat16), or are one
      // key a piece; keys and values that nobody sees are read from a place that somebody does.
      uint4 kf[KP][QS], vf[VP][DV];
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        const int key = h0 + (F32 ? 16 * j + col : 32 * (j / 2) + 8 * (col / 4) + 4 * (j % 2) + col % 4);
        const int seen = CUT ? max(first, min(last, key)) : key;
        const T* kp = kbase + (size_t)(uint32_t)max(bt[seen >> lg], 0) * page_elems + (size_t)(seen & pmask) * D;
#pragma unroll
        for (int k = 0; k < QS; ++k) {
          const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
          // (a step that can lie past D: zeros, not a neighbour's numbers, of which zero times an infinite one is no number)
          if (2 * k + 2 <= QS && QS > 1) kf[j][k] = *(const uint4*)(kp + d);
          else {
            kf[j][k] = make_uint4(0, 0, 0, 0);
            if (d < D) kf[j][k] = *(const uint4*)(kp + d);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        const int k0 = h0 + 4 * SPAN * j + SPAN * quad;  // the lane's first key
        const bool any = !CUT || (k0 <= last && k0 + SPAN - 1 >= first);
        const int at = any ? k0 : (first & ~(SPAN - 1));
        const T* vp = vbase + (size_t)(uint32_t)max(bt[at >> lg], 0) * page_elems + (size_t)col * page + (at & pmask);
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          vf[j][i] = *(const uint4*)vp;
          vp += 16 * (i + 1) < D ? 16 * page : 0;        // (a piece past D reads the last one again and is dropped)
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      floatx4 sc[KP];
#pragma unroll
      for (int j = 0; j < KP; ++j) sc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < QS; ++k)
#pragma unroll
        for (int j = 0; j < KP; ++j) {
          if (F32) {
            const uint32_t ka[4] = {kf[j][k].x, kf[j][k].y, kf[j][k].z, kf[j][k].w}, qa[4] = {qf[k].x, qf[k].y, qf[k].z, qf[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka[i]), __uint_as_float(qa[i]), sc[j], 0, 0, 0);
          } else {
            sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[j][k]), __builtin_bit_cast(bf16x8_t, qf[k]), sc[j], 0, 0, 0);
          }
        }
      // ---- the lane's keys: four a piece, of column col's row
      float e[KP][4], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < KP; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[j][i] = sc[j][i] * scale2;
          if (CUT) {
            const int key = h0 + (F32 ? 16 * j + 4 * quad + i : 32 * (j / 2) + 8 * quad + 4 * (j % 2) + i);
            e[j][i] = takes && key >= lo && key < len ? e[j][i] : -INFINITY;
          }
          top = fmaxf(top, e[j][i]);
        }
      const float m_new = fmaxf(m, quad_max(top)), m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp_of_2(m - m_use);
      m = m_new;
      float add = 0.f;
#pragma unroll
      for (int j = 0; j < KP; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[j][i] = exp_of_2(e[j][i] - m_use);
          add += e[j][i];
        }
      l = l * alpha + add;
      uint4 hi[VP], lw[VP];                             // bfloat16: the weights' two parts
      if (!F32) {
#pragma unroll
        for (int j = 0; j < VP; ++j) {
          uint32_t h4[4], l4[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float x = e[2 * j + w / 2][2 * (w % 2)], y = e[2 * j + w / 2][2 * (w % 2) + 1];
            h4[w] = pack2_bf16(x, y);
            l4[w] = pack2_bf16(x - __uint_as_float(h4[w] << 16), y - __uint_as_float(h4[w] & 0xffff0000u));
          }
          hi[j] = make_uint4(h4[0], h4[1], h4[2], h4[3]);
          lw[j] = make_uint4(l4[0], l4[1], l4[2], l4[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < DV; ++i) {
        floatx4 o;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = acc[i][x] * alpha;
#pragma unroll
        for (int j = 0; j < VP; ++j) {
          uint32_t v4[4] = {vf[j][i].x, vf[j][i].y, vf[j][i].z, vf[j][i].w};
          if (CUT) {                                    // positions that are not seen may hold anything
            const int k0 = h0 + 4 * SPAN * j + SPAN * quad;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if (F32) v4[w] = (k0 + w >= first && k0 + w <= last) ? v4[w] : 0u;
              else {
                const int ka = k0 + 2 * w;
                v4[w] &= ((ka >= first && ka <= last) ? 0x0000ffffu : 0u) | ((ka + 1 >= first && ka + 1 <= last) ? 0xffff0000u : 0u);
              }
            }
          }
          if (F32) {
#pragma unroll
            for (int x = 0; x < 4; ++x) o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v4[x]), e[j][x], o, 0, 0, 0);
          } else {
            const uint4 v = make_uint4(v4[0], v4[1], v4[2], v4[3]);
            o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, hi[j]), o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, lw[j]), o, 0, 0, 0);
          }
        }
        // (a column that takes no part keeps its sums: zero times another beam's infinite value is no number)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][x] = !CUT || takes ? o[x] : acc[i][x];
      }
    };
    if (mine < 0) {
#pragma unroll 1
      for (int h0 = first; h0 <= last; h0 += STEP) step(h0, No{});
    } else {
#pragma unroll 1
      for (int h0 = chunk * CHUNK + (first % CHUNK) / STEP * STEP; h0 <= last; h0 += STEP) step(h0, Yes{});
    }
  }

  // ---- the wavefronts' results joined
  l += __shfl_xor(l, 16, DA_WAVE);
  l += __shfl_xor(l, 32, DA_WAVE);
  if (len <= 0) l = 0.f;                                // (a place without a beam went along in the shared chunks)
  if (quad == 0) {
    m_lds[wave][col] = len > 0 ? m : -INFINITY;
    l_lds[wave][col] = l;
  }
#pragma unroll
  for (int i = 0; i < DV; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc_lds[wave][16 * i + 4 * quad + x][col] = len > 0 ? acc[i][x] : 0.f;
  __syncthreads();
  for (int i = t; i < ROWS * D; i += BEAM_WAVES * DA_WAVE) {
    const int row = i / D, d = i - row * D;
    if (r0 + row >= R) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < BEAM_WAVES; ++w) mm = fmaxf(mm, m_lds[w][row]);
    const float m_use = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < BEAM_WAVES; ++w) {
      const float a = exp_of_2(m_lds[w][row] - m_use);
      ll += a * l_lds[w][row];
      o += a * acc_lds[w][d][row];
    }
    const int bm = (r0 + row) / ratio, hd = hk * ratio + (r0 + row - bm * ratio);
    if (splits == 1) from_f32(out + (size_t)(s0 + bm) * out_ld + (size_t)hd * D + d, ll > 0.f || ll != ll ? o / ll : 0.f);
    else {
      float* p = partial + (((size_t)(s0 + bm) * Hq + hd) * splits + z) * (D + 2);
      p[d] = o;
      if (d == 0) {
        p[D] = mm;
        p[D + 1] = ll;
      }
    }
  }
}

// A wavefront a (sequence, head): a share a lane for the maxima and sums, then a dimension a lane.
#define MERGE_WAVES 4
template <typename T>
__global__ void __launch_bounds__(MERGE_WAVES * DA_WAVE)
attn_beams_merge_kernel(const float* __restrict__ partial, int splits, int pairs, int Hq, int D, T* __restrict__ out, int out_ld) {
  const int lane = threadIdx.x % DA_WAVE, pair = blockIdx.x * MERGE_WAVES + threadIdx.x / DA_WAVE;
  if (pair >= pairs) return;
  const int s = pair / Hq, h = pair - s * Hq;
  const float* p = partial + (size_t)pair * splits * (D + 2);
  const float* mine = p + (size_t)(lane < splits ? lane : 0) * (D + 2) + D;
  const float m = lane < splits ? mine[0] : -INFINITY, l = lane < splits ? mine[1] : 0.f;
  const float mm = wave_max(m), m_use = mm == -INFINITY ? 0.f : mm;
  const float w = lane < splits ? exp_of_2(m - m_use) : 0.f;
  const float ll = wave_sum(w * l), inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
  for (int d0 = 0; d0 < D; d0 += DA_WAVE) {
    const int d = d0 + lane;
    float o = 0.f;
    for (int z0 = 0; z0 < splits; z0 += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(size_t)min(z0 + u, splits - 1) * (D + 2) + (d < D ? d : 0)];
#pragma unroll
      for (int u = 0; u < 8; ++u) o += (z0 + u < splits ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), min(z0 + u, DA_WAVE - 1))) : 0.f) * v[u];
    }
    if (d < D) from_f32(out + (size_t)s * out_ld + (size_t)h * D + d, o * inv);
  }
}

extern "C" int da_attn_beams_takes(int D, int page) {
  return D % 16 == 0 && D >= 16 && D <= BEAMS_MAX_D && page >= 16 && (page & (page - 1)) == 0;
}

// How many workgroups share a group's positions: from the step's shape only.
extern "C" int da_attn_beams_splits(int G, int B, int Hq, int Hkv, int D, int max_blocks, int page) {
  if (G <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || max_blocks <= 0 || page <= 0) return 1;
  const long groups = (long)G * Hkv * da_ceil_div((long)B * (Hq / Hkv), ROWS);
  const long chunks = ((long)max_blocks * page + CHUNK - 1) / CHUNK;
  long n = 512 / groups;
  if (n > chunks / BEAM_WAVES) n = chunks / BEAM_WAVES;
  return n < 1 ? 1 : (n > 64 ? 64 : (int)n);
}

template <typename T, int DK, int STEP>
static void beams_launch(hipStream_t s, const void* q, int q_ld, const void* cache, const int* block_table, int max_blocks, const int* seq_lens,
                         const int* shared, int G, int B, int Hq, int Hkv, int D, int page, float scale, int window, void* out, int out_ld,
                         int splits, float* partial) {
  const int blocks = da_ceil_div((long)B * (Hq / Hkv), ROWS);
  hipLaunchKernelGGL((attn_beams_kernel<T, DK, STEP>), dim3(Hkv * blocks, G, splits), dim3(BEAM_WAVES * DA_WAVE), 0, s, (const T*)q, q_ld,
                     (const T*)cache, block_table, max_blocks, seq_lens, shared, B, Hq, Hkv, D, page, scale, window, (T*)out, out_ld, splits,
                     partial);
}

extern "C" int da_attn_beams(const void* q, int q_ld, const void* cache, int dtype, const int* block_table, int max_blocks, const int* seq_lens,
                             const int* shared, int G, int B, int Hq, int Hkv, int D, int page, float scale, int window, void* out, int out_ld,
                             int splits, float* workspace, long workspace_floats, void* stream) {
  DA_REQUIRE(G >= 0 && B > 0 && B <= BEAMS_MAX && (long)G * B <= 65535 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && max_blocks > 0 && window >= 0,
             "attention_beams: bad sizes (groups=%d beams=%d heads=%d/%d blocks=%d window=%d; at most %d beams)", G, B, Hq, Hkv, max_blocks, window, BEAMS_MAX);
  DA_REQUIRE(da_attn_beams_takes(D, page), "attention_beams: head size %d (multiples of 16 up to %d), page %d (powers of two from 16)", D, BEAMS_MAX_D, page);
  DA_REQUIRE(dtype == DA_F32 || dtype == DA_BF16, "attention_beams: dtype %d", dtype);
  const int el = dtype == DA_F32 ? 4 : 2;
  DA_REQUIRE((uintptr_t)q % 16 == 0 && (long)q_ld * el % 16 == 0 && (uintptr_t)cache % 16 == 0, "attention_beams: q and the cache must lie on 16 bytes");
  DA_REQUIRE((long)max_blocks * page <= 0x7fffff00L && 2L * Hkv * page * D <= 0x7fffffffL, "attention_beams: a page or a table is too large");
  DA_REQUIRE(splits >= 1 && splits <= DA_WAVE, "attention_beams: %d shares (1 to 64)", splits);
  const long need = splits > 1 ? (long)G * B * Hq * splits * (D + 2) : 0;
  DA_REQUIRE(need == 0 || (workspace && workspace_floats >= need), "attention_beams: %ld floats of workspace are needed, found %ld", need, workspace_floats);
  if (G == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
#define DA_BEAMS(T, DK, STEP) beams_launch<T, DK, STEP>(s, q, q_ld, cache, block_table, max_blocks, seq_lens, shared, G, B, Hq, Hkv, D, page, scale, window, out, out_ld, splits, workspace)
  if (dtype == DA_F32) {
    if (D <= 32) DA_BEAMS(float, 1, 32);
    else if (D <= 64) DA_BEAMS(float, 2, 32);
    else if (D <= 128) DA_BEAMS(float, 4, 32);
    else DA_BEAMS(float, 8, 16);
  } else {
    if (D <= 32) DA_BEAMS(bf16_t, 1, 64);
    else if (D <= 64) DA_BEAMS(bf16_t, 2, 64);
    else if (D <= 128) DA_BEAMS(bf16_t, 4, 32);
    else DA_BEAMS(bf16_t, 8, 32);
  }
#undef DA_BEAMS
  DA_CHECK_LAUNCH("attention_beams");
  if (splits > 1) {
    const int pairs = G * B * Hq;
    const dim3 grid(da_ceil_div(pairs, MERGE_WAVES)), block(MERGE_WAVES * DA_WAVE);
    if (dtype == DA_F32) hipLaunchKernelGGL((attn_beams_merge_kernel<float>), grid, block, 0, s, workspace, splits, pairs, Hq, D, (float*)out, out_ld);
    else hipLaunchKernelGGL((attn_beams_merge_kernel<bf16_t>), grid, block, 0, s, workspace, splits, pairs, Hq, D, (bf16_t*)out, out_ld);
    DA_CHECK_LAUNCH("attention_beams (merge)");
  }
  return 0;
}
