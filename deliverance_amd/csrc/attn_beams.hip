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

#define BEAMS_MAX 64             // beams of a group
#define BEAMS_MAX_D 256
#define CHUNK 64
#define ROWS 16                  // of a workgroup
#define BEAM_WAVES 4

__device__ __forceinline__ float beam_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// Row maximum over the four lanes that hold a row's keys
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, DA_WAVE));
  return fmaxf(v, __shfl_xor(v, 32, DA_WAVE));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16, DA_WAVE);
  return v + __shfl_xor(v, 32, DA_WAVE);
}

// DK: head size in steps of 32, rounded up to a power of two
template <typename T, int DK>
__global__ void __launch_bounds__(BEAM_WAVES * DA_WAVE)
attn_beams_kernel(const T* __restrict__ q, int q_ld, const T* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                  const int* __restrict__ seq_lens, const int* __restrict__ shared, int B, int Hq, int Hkv, int D, int page, float scale,
                  int window, T* __restrict__ out, int out_ld, int splits, float* __restrict__ partial) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int DV = 2 * DK, DMAX = 32 * DK;            // value dimensions in steps of 16
  constexpr int QS = F32 ? 2 * DK : DK;                 // key loads a row: 16 dimensions (32-bit) or 32 (bfloat16) a step
  __shared__ float acc_lds[BEAM_WAVES][DMAX][ROWS + 1];
  __shared__ float m_lds[BEAM_WAVES][ROWS], l_lds[BEAM_WAVES][ROWS];
  __shared__ int len_lds[BEAMS_MAX];

  const int t = threadIdx.x, lane = t % DA_WAVE, wave = __builtin_amdgcn_readfirstlane(t / DA_WAVE);
  const int col = lane % 16, quad = lane / 16;
  const int ratio = Hq / Hkv, R = B * ratio;
  const int hk = blockIdx.x % Hkv, rb = blockIdx.x / Hkv, g = blockIdx.y, z = blockIdx.z;
  const int r0 = rb * ROWS, r_last = min(r0 + ROWS, R) - 1;
  const int b0 = r0 / ratio, b1 = r_last / ratio;       // the beams of these rows
  const int s0 = g * B;
  const int lg = 31 - __builtin_clz(page), pmask = page - 1;
  const uint32_t page_elems = 2u * (uint32_t)(Hkv * page * D);

  // this lane's row
  const int r = r0 + col, beam = min(r, R - 1) / ratio, head = hk * ratio + (min(r, R - 1) - beam * ratio);
  const int cap = max_blocks * page;                    // (a longer length would lead out of the table)
  const int len = r < R ? min(seq_lens[s0 + beam], cap) : 0;
  const int lo = window > 0 && len - window > 0 ? len - window : 0;

  // the positions that every beam of the group has in shared pages, and from which on every row of this workgroup sees them
  int first_live = -1, common = cap, lo_max = 0;
  for (int b = 0; b < B; ++b) {
    const int n = min(seq_lens[s0 + b], cap);
    if (n <= 0) continue;
    if (first_live < 0) first_live = b;
    common = min(common, n);
    if (window > 0 && n - window > lo_max) lo_max = n - window;
  }
  common = first_live < 0 ? 0 : min(common, shared[g]);
  const int shared0 = (lo_max + CHUNK - 1) / CHUNK, shared1 = common / CHUNK > shared0 ? common / CHUNK : shared0;
  auto own_chunks = [&](int b, int& first, int& skip_at, int& skip_to) {      // number of the beam's own chunks
    const int n = min(seq_lens[s0 + b], cap);
    if (n <= 0) return 0;
    first = window > 0 && n - window > 0 ? (n - window) / CHUNK : 0;
    const int end = (n + CHUNK - 1) / CHUNK;
    skip_at = shared0;
    skip_to = shared1;
    // chunks first .. end - 1 without shared0 .. shared1 - 1
    return end - first - (shared1 - shared0);
  };
  int items = shared1 - shared0;
  for (int b = b0; b <= b1; ++b) {
    int f, a, e;
    items += own_chunks(b, f, a, e);
  }
  const int per = (items + splits - 1) / splits;
  const int item0 = z * per, item1 = min(items, item0 + per);

  // the query rows: the right operand
  uint4 qf[QS];
#pragma unroll
  for (int k = 0; k < QS; ++k) {
    const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
    qf[k] = make_uint4(0, 0, 0, 0);
    if (d < D && r < R) qf[k] = *(const uint4*)(q + (size_t)(s0 + beam) * q_ld + (size_t)head * D + d);
  }

  floatx4 acc[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  for (int item = item0 + wave; item < item1; item += BEAM_WAVES) {
    // which chunk of which table
    int chunk, mine = -1, src = first_live;
    if (item < shared1 - shared0) chunk = shared0 + item;
    else {
      int left = item - (shared1 - shared0), f = 0, a = 0, e = 0;
      for (mine = b0; mine < b1; ++mine) {
        const int n = own_chunks(mine, f, a, e);
        if (left < n) break;
        left -= n;
      }
      own_chunks(mine, f, a, e);
      chunk = f + left;
      if (e > a && chunk >= a) chunk += e - a;
      src = mine;
    }
    const int* bt = block_table + (size_t)(s0 + src) * max_blocks;
    const int n_src = min(seq_lens[s0 + src], cap), lo_src = window > 0 && n_src - window > 0 ? n_src - window : 0;
    const int c0 = chunk * CHUNK;
    const int first = mine < 0 ? c0 : max(c0, lo_src), last = mine < 0 ? c0 + CHUNK - 1 : min(c0 + CHUNK, n_src) - 1;
    const bool takes = mine < 0 || mine == beam;

#pragma unroll 1
    for (int h0 = c0; h0 < c0 + CHUNK; h0 += 32) {      // 32 keys at a time
      if (h0 > last || h0 + 31 < first) continue;
      floatx4 sc[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        const int key = h0 + (F32 ? 16 * j + col : 8 * (col / 4) + 4 * j + col % 4);
        const int seen = key < first ? first : (key > last ? last : key);
        const int pg = max(bt[seen >> lg], 0);
        const T* kp = cache + (size_t)pg * page_elems + ((size_t)hk * page + (seen & pmask)) * D;
#pragma unroll
        for (int k = 0; k < QS; ++k) {
          const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
          uint4 kf = make_uint4(0, 0, 0, 0);
          if (d < D) kf = *(const uint4*)(kp + d);
          if (F32) {
            const uint32_t ka[4] = {kf.x, kf.y, kf.z, kf.w}, qa[4] = {qf[k].x, qf[k].y, qf[k].z, qf[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka[i]), __uint_as_float(qa[i]), sc[j], 0, 0, 0);
          } else {
            sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf), __builtin_bit_cast(bf16x8_t, qf[k]), sc[j], 0, 0, 0);
          }
        }
      }
      // this lane's 8 keys: key_of(j, i)
      float s[2][4], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = h0 + (F32 ? 16 * j + 4 * quad + i : 8 * quad + 4 * j + i);
          const bool sees = takes && key >= first && key <= last && key >= lo && key < len;
          s[j][i] = sees ? sc[j][i] * scale : -INFINITY;
          top = fmaxf(top, s[j][i]);
        }
      const float m_new = fmaxf(m, quad_max(top)), m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = beam_exp(m - m_use);
      m = m_new;
      l *= alpha;
      float e[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[j][i] = beam_exp(s[j][i] - m_use);
          l += e[j][i];
        }
      uint4 hi = make_uint4(0, 0, 0, 0), lw = hi;       // bfloat16: the weights' two parts
      if (!F32) {
        uint32_t h4[4], l4[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float x = e[w / 2][2 * (w % 2)], y = e[w / 2][2 * (w % 2) + 1];
          h4[w] = pack2_bf16(x, y);
          l4[w] = pack2_bf16(x - __uint_as_float(h4[w] << 16), y - __uint_as_float(h4[w] & 0xffff0000u));
        }
        hi = make_uint4(h4[0], h4[1], h4[2], h4[3]);
        lw = make_uint4(l4[0], l4[1], l4[2], l4[3]);
      }
      const bool cut = h0 < first || h0 + 31 > last;
#pragma unroll
      for (int j = 0; j < (F32 ? 2 : 1); ++j) {
        const int k0 = h0 + (F32 ? 16 * j + 4 * quad : 8 * quad), span = F32 ? 4 : 8;      // the lane's keys of the left operand
        const bool any = k0 <= last && k0 + span - 1 >= first;
        const int at = any ? k0 : (first & ~(span - 1));
        const int pg = max(bt[at >> lg], 0);
        const T* vp = cache + (size_t)pg * page_elems + (size_t)(Hkv + hk) * page * D + (at & pmask);
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          const int d = 16 * i + col;
          uint4 vf = make_uint4(0, 0, 0, 0);
          if (16 * i < D) vf = *(const uint4*)(vp + (size_t)d * page);
          if (cut) {                                    // rows that are not seen may hold anything
            uint32_t v4[4] = {vf.x, vf.y, vf.z, vf.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if (F32) v4[w] = (k0 + w >= first && k0 + w <= last) ? v4[w] : 0u;
              else {
                const int ka = k0 + 2 * w;
                v4[w] &= ((ka >= first && ka <= last) ? 0x0000ffffu : 0u) | ((ka + 1 >= first && ka + 1 <= last) ? 0xffff0000u : 0u);
              }
            }
            vf = make_uint4(v4[0], v4[1], v4[2], v4[3]);
          }
          if (F32 ? j == 0 : true) {
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[i][x] *= alpha;
          }
          floatx4 o = acc[i];
          if (F32) {
            const uint32_t v4[4] = {vf.x, vf.y, vf.z, vf.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v4[x]), e[j][x], o, 0, 0, 0);
          } else {
            o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, hi), o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, lw), o, 0, 0, 0);
          }
          // (a column that takes no part keeps its sums: zero times another beam's infinite value is no number)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][x] = takes ? o[x] : acc[i][x];
        }
      }
    }
  }

  // ---- the wavefronts' results joined
  l = quad_sum(l);
  if (quad == 0) {
    m_lds[wave][col] = m;
    l_lds[wave][col] = l;
  }
#pragma unroll
  for (int i = 0; i < DV; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) acc_lds[wave][16 * i + 4 * quad + x][col] = acc[i][x];
  __syncthreads();
  for (int i = t; i < ROWS * D; i += BEAM_WAVES * DA_WAVE) {
    const int row = i / D, d = i - row * D;
    if (r0 + row >= R) break;
    float mm = -INFINITY;
    for (int w = 0; w < BEAM_WAVES; ++w) mm = fmaxf(mm, m_lds[w][row]);
    const float m_use = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, o = 0.f;
    for (int w = 0; w < BEAM_WAVES; ++w) {
      const float a = beam_exp(m_lds[w][row] - m_use);
      ll += a * l_lds[w][row];
      o += a * acc_lds[w][d][row];
    }
    const int bm = (r0 + row) / ratio, hd = hk * ratio + (r0 + row - bm * ratio);
    if (splits == 1) from_f32(out + (size_t)(s0 + bm) * out_ld + (size_t)hd * D + d, ll > 0.f || ll != ll ? o / ll : 0.f);
    else {
      float* p = partial + ((((size_t)(s0 + bm) * Hq + hd) * splits) + z) * (D + 2);
      p[d] = o;
      if (d == 0) {
        p[D] = mm;
        p[D + 1] = ll;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(BEAMS_MAX_D)
attn_beams_merge_kernel(const float* __restrict__ partial, int splits, int Hq, int D, T* __restrict__ out, int out_ld) {
  const int h = blockIdx.x, s = blockIdx.y, d = threadIdx.x;
  if (d >= D) return;
  const float* p = partial + ((size_t)s * Hq + h) * splits * (D + 2);
  float mm = -INFINITY;
  for (int z = 0; z < splits; ++z) mm = fmaxf(mm, p[(size_t)z * (D + 2) + D]);
  const float m_use = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, o = 0.f;
  for (int z = 0; z < splits; ++z) {
    const float* pz = p + (size_t)z * (D + 2);
    const float a = beam_exp(pz[D] - m_use);
    ll += a * pz[D + 1];
    o += a * pz[d];
  }
  from_f32(out + (size_t)s * out_ld + (size_t)h * D + d, ll > 0.f || ll != ll ? o / ll : 0.f);
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

template <typename T, int DK>
static void beams_launch(hipStream_t s, const void* q, int q_ld, const void* cache, const int* block_table, int max_blocks, const int* seq_lens,
                         const int* shared, int G, int B, int Hq, int Hkv, int D, int page, float scale, int window, void* out, int out_ld,
                         int splits, float* partial) {
  const int blocks = da_ceil_div((long)B * (Hq / Hkv), ROWS);
  hipLaunchKernelGGL((attn_beams_kernel<T, DK>), dim3(Hkv * blocks, G, splits), dim3(BEAM_WAVES * DA_WAVE), 0, s, (const T*)q, q_ld,
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
  DA_REQUIRE(splits >= 1 && splits <= 65535, "attention_beams: %d shares", splits);
  const long need = splits > 1 ? (long)G * B * Hq * splits * (D + 2) : 0;
  DA_REQUIRE(need == 0 || (workspace && workspace_floats >= need), "attention_beams: %ld floats of workspace are needed, found %ld", need, workspace_floats);
  if (G == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
#define DA_BEAMS(T, DK) beams_launch<T, DK>(s, q, q_ld, cache, block_table, max_blocks, seq_lens, shared, G, B, Hq, Hkv, D, page, scale, window, out, out_ld, splits, workspace)
  if (dtype == DA_F32) {
    if (D <= 32) DA_BEAMS(float, 1);
    else if (D <= 64) DA_BEAMS(float, 2);
    else if (D <= 128) DA_BEAMS(float, 4);
    else DA_BEAMS(float, 8);
  } else {
    if (D <= 32) DA_BEAMS(bf16_t, 1);
    else if (D <= 64) DA_BEAMS(bf16_t, 2);
    else if (D <= 128) DA_BEAMS(bf16_t, 4);
    else DA_BEAMS(bf16_t, 8);
  }
#undef DA_BEAMS
  DA_CHECK_LAUNCH("attention_beams");
  if (splits > 1) {
    const int threads = da_ceil_div(D, DA_WAVE) * DA_WAVE;
    if (dtype == DA_F32)
      hipLaunchKernelGGL((attn_beams_merge_kernel<float>), dim3(Hq, G * B), dim3(threads), 0, s, workspace, splits, Hq, D, (float*)out, out_ld);
    else
      hipLaunchKernelGGL((attn_beams_merge_kernel<bf16_t>), dim3(Hq, G * B), dim3(threads), 0, s, workspace, splits, Hq, D, (bf16_t*)out, out_ld);
    DA_CHECK_LAUNCH("attention_beams (merge)");
  }
  return 0;
}
