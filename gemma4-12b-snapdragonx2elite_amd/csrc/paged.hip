// A batch of sequences on a paged fp16 KV cache: the preparation of q, k and
// v with the append (q4_paged_prep), and attention over a prefix that every
// sequence shares and each one's own pages (q4_paged_attn).
//
// Cache: kc, vc [npages][nkv][page][hd]. Position j < P (P = *prefix_len, 0
// without a prefix) lives in page prefix_pages[j / page], row j % page; later
// positions in page table[s][(j - P) / page], row (j - P) % page, of their
// sequence s. A page number outside 0 .. npages - 1 names no page: nothing is
// written there, and its keys are left out.
#include "q4mi_common.h"

#include <cmath>

namespace q4 {

// An element of an int32 array at a wave-uniform index, through the scalar
// unit: nothing in these kernels writes the arrays, and a scalar load does not
// enter the count of vector loads that the tile loads' waits go by.
__device__ inline int uload(const int32_t* p, long i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>((uintptr_t)p)[i];
}

struct Pages {
  const int32_t* prefix_pages;  // [ceil(max_prefix / page)]
  const int32_t* prefix_len;    // [1]
  const int32_t* table;         // [nseq][ld]
  const int32_t* seq;           // [T]: sequence of each row, out of range = no row
  const int32_t* pos;           // [T]: its position
  int ld, nseq, npages, lg, max_prefix, max_own;
  // P, which divides the positions; attention visits its first max_prefix keys
  __device__ inline int prefix() const { return prefix_len ? max(uload(prefix_len, 0), 0) : 0; }
  __device__ inline int prefix_keys() const { return min(prefix(), max_prefix); }
};

// ---- q, k, v rows: norm, RoPE, append ---------------------------------------
// 8 consecutive elements of fp32 or fp16 data as fp32
template <int DT>
__device__ inline void pg_ld8(const void* p, long i, float (&v)[8]) {
  if constexpr (DT == Q4_DT_F16) {
    const v4u u = *reinterpret_cast<const v4u*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = h2f((uint16_t)(u[k] & 0xFFFFu));
      v[2 * k + 1] = h2f((uint16_t)(u[k] >> 16));
    }
  } else {
    const v4f a = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(p) + i);
    const v4f b = *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(p) + i + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = a[k];
      v[4 + k] = b[k];
    }
  }
}

// Sum over the LPH lanes of a head, the same bits in each of them.
template <int LPH>
__device__ inline float pg_head_sum(float v) {
  if constexpr (LPH == 8) return reduce8<false>(v);
  else if constexpr (LPH == 16) return reduce16<false>(v);
  else if constexpr (LPH == 32) return reduce32<false>(v);
  else return reduce64<false>(v);
}

// y = x inv(x) w, inv(v) = 1 / sqrt(mean(v^2) + 1e-6) of each head (v: no
// w), then RoPE(y)[i] = y[i] cos[i] -+ y[i +- HD / 2] sin[i] (v: none), rounded to
// fp16 into q or the cache. Row blockIdx.x (a token), HPG heads per group of
// LPH = HD / 8 lanes: heads 0 .. nH - 1 are q, then nkv of k, then nkv of v.
// A lane holds 8 elements, one 16-byte load of fp16 and one store; the RoPE
// partner is the same slot of lane ^ LPH / 2. Bound by memory for large
// batches (2048 rows of 16 + 2 heads of 512: 82 MB in 15.6 to 17.1 us, 4.8 to
// 5.3 TB/s, about the rate of a copy), else by the chain seq, pos -> RoPE row and page -> store
// (one row of 16 + 2 x 8 heads of 256 among others: 3.8 us).
template <int HD, int DT, int HPG>
__global__ void __launch_bounds__(256)
paged_prep_kernel(const void* __restrict__ qkv, int ld, int qoff, int koff, int voff, const float* __restrict__ qnw,
                  const float* __restrict__ knw, const float* __restrict__ cos_tab,
                  const float* __restrict__ sin_tab, int max_pos, uint16_t* __restrict__ q, int ldq,
                  uint16_t* __restrict__ kc, uint16_t* __restrict__ vc, int nH, int nkv, const Pages pg) {
  constexpr int LPH = HD / 8, G = 256 / LPH;
  const int t = blockIdx.x, lane = threadIdx.x % LPH, gi = threadIdx.x / LPH, i0 = 8 * lane;
  const int s = pg.seq[t], pos = pg.pos[t];
  if (s < 0 || s >= pg.nseq || pos < 0 || pos >= max_pos) return;  // (uniform) no row, or no RoPE row for it
  float c[8], sn[8];
  pg_ld8<Q4_DT_F32>(cos_tab, (long)pos * HD + i0, c);
  pg_ld8<Q4_DT_F32>(sin_tab, (long)pos * HD + i0, sn);
  // this token's cache row: -1 where it has none
  const int i = pos - pg.prefix(), pi = i >> pg.lg;
  int p = -1;
  if (i >= 0 && pi < pg.ld) p = pg.table[(long)s * pg.ld + pi];
  if (p >= pg.npages) p = -1;
  const int slot = i & ((1 << pg.lg) - 1);
#pragma unroll
  for (int k = 0; k < HPG; ++k) {
    const int hh = (blockIdx.y * HPG + k) * G + gi;
    if (hh >= nH + 2 * nkv) return;
    const bool isq = hh < nH, isv = hh >= nH + nkv;
    const int h = isq ? hh : isv ? hh - nH - nkv : hh - nH;
    float x[8], w[8];
    pg_ld8<DT>(qkv, (long)t * ld + (isq ? qoff : isv ? voff : koff) + (long)h * HD + i0, x);
    pg_ld8<Q4_DT_F32>(isq ? qnw : knw, i0, w);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    const float inv = inv_rms(pg_head_sum<LPH>(ss), HD);
    const bool lo = lane < LPH / 2;
    uint32_t r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = __fmul_rn(x[e], inv), y = __fmul_rn(n, w[e]);
      const float pr = __shfl_xor(y, LPH / 2);
      const float ro = __fadd_rn(__fmul_rn(y, c[e]), __fmul_rn(lo ? -pr : pr, sn[e]));
      r[e] = f2h_after_f32(isv ? n : ro);
    }
    const v4u out = {r[0] | r[1] << 16, r[2] | r[3] << 16, r[4] | r[5] << 16, r[6] | r[7] << 16};
    if (isq) *reinterpret_cast<v4u*>(q + (long)t * ldq + (long)h * HD + i0) = out;
    else if (p >= 0)
      *reinterpret_cast<v4u*>((isv ? vc : kc) + ((((long)p * nkv + h) << pg.lg) + slot) * HD + i0) = out;
  }
}

// ---- attention ---------------------------------------------------------------
// Scores S^T = K q^T and outputs O^T += V^T P^T on the f16 matrix cores, 16
// query rows as the columns of both products, so a lane (c, g) = (lane % 16,
// lane / 16) holds row c throughout: scores of keys 4g .. 4g + 3 of each
// 16-key subtile, the same keys' weights as the V product's B operand, and
// output elements 4g .. 4g + 3 of each 16-element tile. K and V tiles go from
// the cache straight into LDS (16 bytes per lane, no registers), row-major;
// the V product's A operand is read transposed from there (4 keys of one
// element per lane). Workgroups of 4 waves in two shapes share a launch:
//
//  * shared tiles, for a prefix with more than 16 query rows per KV head:
//    each wave holds 32 of 128 rows, or 16 of 64 (row = token * grp + head in
//    the group); all read the same tiles of KT keys, one tile ahead;
//  * streams, for a token's own pages (rows: the query heads of its KV head)
//    and a prefix with up to 16 rows: every wave holds all the rows and takes
//    every fourth tile of OKT keys by itself, K of its next tile loading
//    while this one's weights form and V of it while the next one's scores
//    do; the four waves join at the end.
//
// Each takes one split of the keys and leaves (reference exponent, sum,
// accumulator) per query row; a second kernel joins the parts (where a plan
// has only one part, the stream writes the output).
constexpr int PG_THREADS = 256, PG_WAVES = 4;
// MODE of a launch: no prefix, a prefix in shared tiles (of workgroups with 128 query rows, or with 64), or one as a
// stream.
enum { PG_OWN, PG_SHARED, PG_SHARED_FEW, PG_STREAM };
// Most rows of a prefix that streams: 16, a wave's MFMA columns. us with the merge behind 16384 (4096) keys, as streams
// and in shared tiles, each launch alone: 8 heads of 256, 2 rows 33.0 / 35.5 (17.5 / 17.6) and 16 rows 35.4 / 38.1
// (17.4 / 18.0); one of 512, 16 rows 24.0 / 23.4 (16.4 / 15.6); 8 of 128, 16 rows 20.4 / 21.1 (12.4 / 12.3).
constexpr int PG_STREAM_ROWS = 16;
// Most rows of a workgroup of 16 rows per wave, which leaves waves busy where 32 would leave them without rows; with
// more rows than it holds each tile would be loaded again. us with the merge behind 16384 keys with 16 and with 32 rows
// per wave: 8 heads of 256, 32 rows 42.7 / 43.6 and 64 rows 51.4 / 52.4; one of 512, 24.2 / 28.5 and 28.2 / 33.9; 8 of
// 128, 22.7 / 24.0 and 26.2 / 29.2.
constexpr int PG_FEW_ROWS = 64;
constexpr float PG_LOG2E = 1.4426950408889634f;
// A row's weights are 2^(score - ref): ref is set 6 below the row's largest
// score so far (in log2 units) and moves only when a score passes it by 14,
// so weights reach 2^14 < 65504 and the leading bits of those 2^20 below the
// largest are no fp16 subnormals; moving it rescales the accumulators, which
// is rare.
constexpr float PG_BELOW = 6.0f, PG_MOVE = 14.0f;

template <int HD>
struct PgTile {
  static constexpr int KT = HD >= 256 ? 32 : 64;             // keys of a shared tile
  static constexpr int OKT = HD >= 256 ? 16 : 32;            // keys of a stream's tile
  static constexpr int NCH = HD / 32, NDT = HD / 16;         // 32-element chunks, 16-element output tiles
  static constexpr int KPI = 512 / HD;                       // keys of one 1 KB load
  static constexpr int REGION = 2 * OKT * HD * 2;            // a stream's K and V tile
  static constexpr int STAGE = 2 * KT * HD * 2;              // a shared K and V tile
  static constexpr int DS = HD == 512 ? 2 : 1;               // waves that share the rows of one in shared tiles
  static constexpr int TILES = 2 * STAGE > PG_WAVES * REGION ? 2 * STAGE : PG_WAVES * REGION;
  static constexpr bool shared(int mode) { return mode == PG_SHARED || mode == PG_SHARED_FEW; }
  static constexpr int tiles(int mode) { return shared(mode) ? TILES : PG_WAVES * REGION; }
  // behind the tiles: statistics of the waves, or the scores that pairs of waves exchange (160 KB in all)
  static constexpr int lds(int mode) { return tiles(mode) + (shared(mode) && DS == 2 ? 2 * PG_WAVES * 4 * 1024 : 512); }
  static constexpr int threads(int mode) { return shared(mode) ? PG_THREADS * DS : PG_THREADS; }
  static constexpr int waves(int mode) { return HD == 512 ? (shared(mode) ? 2 : 1) : HD == 256 || mode != 0 ? 2 : 4; }
  static_assert(REGION >= 16 * HD * 4, "the waves' accumulators join in the tiles' place");
};

// LDS by 32-bit offset, so that constant parts fold into the instructions
__device__ inline uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)p; }
template <class T>
__device__ inline T lds_read(uint32_t at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) T*>((uintptr_t)at);
}
template <class T>
__device__ inline void lds_write(uint32_t at, T v) {
  *reinterpret_cast<__attribute__((address_space(3))) T*>((uintptr_t)at) = v;
}
typedef __fp16 v4hp __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
// two values rounded towards zero to fp16
__device__ inline v2h cvt_rtz(float a, float b) { return __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(a, b)); }
__device__ inline v8h join(v4h a, v4h b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// 4 fp16 of 16 consecutive row elements each, 4 rows per 16 lanes; the lane
// gets the element of its number from each of the 4 rows
__device__ inline v4h lds_read_tr(uint32_t at) {
  typedef __attribute__((address_space(3))) v4hp* lp;
  return __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lp)(uintptr_t)at));
}

// Where 16-byte chunk ch of key row `key` lies in a row of an LDS tile: an
// exclusive or with the key, so that the lanes of one access fall on distinct
// banks: the 16 keys of a K fragment (one chunk each), and the 8 keys of half
// a transposed V read (two chunks each). Rows of HD 64 are half a bank cycle.
template <int HD>
__device__ inline int k_swz(int key) { return HD >= 128 ? key & 15 : (key >> 1) & 7; }
template <int HD>
__device__ inline int v_swz(int key) { return HD >= 128 ? 2 * (key & 7) : 2 * ((key >> 1) & 3); }

__device__ const v4u pg_zero = {0, 0, 0, 0};  // what a lane without a key loads

// Four (two) 1 KB loads into consecutive LDS: the lane's 16 bytes at sbase +
// voff[i] + 1024 i into lds + 1024 i + 16 lane (the instruction's offset
// counts for both addresses).
__device__ inline void dma_block(const void* sbase, const uint32_t (&v)[4], uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\tglobal_load_lds_dwordx4 %1, %4 offset:%6\n\t"
      "global_load_lds_dwordx4 %2, %4 offset:%7\n\tglobal_load_lds_dwordx4 %3, %4 offset:%8" ::"v"(v[0]),
      "v"(v[1]), "v"(v[2]), "v"(v[3]), "s"(sbase), "s"(lds), "n"(1024), "n"(2 * 1024), "n"(3 * 1024)
      : "memory");
}
__device__ inline void dma_block(const void* sbase, const uint32_t (&v)[2], uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4" ::"v"(
          v[0]),
      "v"(v[1]), "s"(sbase), "s"(lds), "n"(1024)
      : "memory");
}

// A lane's byte offset of key row `row`, before the row's own: the key row of
// its group of lanes, and its chunk there under the swizzle of row0.
// The swizzles are linear over exclusive or where a key's bits do not
// overlap, so row r's offset is this ^ 16 swz(r): one register for all loads.
template <int HD, bool V>
__device__ inline uint32_t load_off(int row0) {
  constexpr int CPR = HD / 8;
  const int lane = threadIdx.x & 63, kk = lane / CPR, ch = lane % CPR;
  return kk * HD * 2 + 16 * (ch ^ (V ? v_swz<HD>(row0 + kk) : k_swz<HD>(row0 + kk)));
}

// Keys key0 .. key0 + NK - 1 of one page into rows row0 .. of an LDS tile.
// base: the cache at the page's row of key0 (uniform); off: load_off(row0);
// keys outside lo .. hi - 1, and those of no page, become zeros.
template <int HD, int NK, bool V>
__device__ __forceinline__ void load_rows(const uint16_t* base, uint32_t off, uint32_t tile, int row0, int key0, int lo,
                                          int hi, bool page) {
  constexpr int KPI = PgTile<HD>::KPI, N = NK / KPI, B = N % 4 == 0 ? 4 : 2;
  static_assert(N % B == 0, "whole blocks of loads");
  const uint32_t dst = __builtin_amdgcn_readfirstlane(tile + row0 * HD * 2);
  if (page && key0 >= lo && key0 + NK <= hi) {  // (uniform)
#pragma unroll
    for (int i = 0; i < N; i += B) {
      uint32_t v[B];
#pragma unroll
      for (int k = 0; k < B; ++k) v[k] = off ^ (16 * (V ? v_swz<HD>((i + k) * KPI) : k_swz<HD>((i + k) * KPI)));
      dma_block(reinterpret_cast<const char*>(base) + i * 1024, v, dst + i * 1024);
    }
  } else {
    pin(off);  // (nothing of this rare path is worth a register across the loop, nor code unrolled)
    const int kk = (threadIdx.x & 63) / (HD / 8);
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      const int key = key0 + i * KPI + kk;
      const uint32_t v = off ^ (16 * (V ? v_swz<HD>(i * KPI) : k_swz<HD>(i * KPI)));
      const void* p = reinterpret_cast<const char*>(base) + i * 1024 + v;
      dma16(page && key >= lo && key < hi ? p : (const void*)&pg_zero, reinterpret_cast<const void*>((uintptr_t)(dst + i * 1024)));
    }
  }
}

// A lane's LDS addresses of its K fragments and transposed V reads. Rows and
// tiles lie at multiples of 256 bytes (128 at HD 64), so that the exclusive
// or of a chunk's number is one of the address's bits: chunk 4 j + g of key c
// is at (ko ^ 64 (j % 4)) + 256 (j / 4), element tile d of keys 4 g ..
// 4 g + 3 at (vo ^ 32 (d % 8)) + 256 (d / 8), 16-key subtiles 32 HD apart.
template <int HD>
struct PgLane {
  static constexpr int NK = HD >= 128 ? 4 : 2, NV = HD >= 128 ? 8 : 4;
  uint32_t ko, vo;
  __device__ inline PgLane(uint32_t ktile, uint32_t vtile) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, key = 4 * g + (c >> 2);
    ko = ktile + c * HD * 2 + 16 * (g ^ k_swz<HD>(c));
    vo = vtile + key * HD * 2 + 16 * (((c & 3) >> 1) ^ v_swz<HD>(key)) + 8 * (c & 1);
  }
  __device__ inline void move(int by) { ko += by, vo += by; }  // to the other stage
  template <int ST, int J>
  __device__ inline v8h k() const { return lds_read<v8h>((ko ^ (64 * (J % NK))) + ST * 16 * HD * 2 + (J / NK) * 256); }
  template <int ST, int D>
  __device__ inline v4h v() const { return lds_read_tr((vo ^ (32 * (D % NV))) + ST * 16 * HD * 2 + (D / NV) * 256); }
};

// use(i, fragment i) for i < N with fragments read DEPTH ahead. The order is
// pinned: left to itself the compiler reads a fragment, waits ~100 cycles for
// it and goes on (tiles of head dim 512 took 9.6k cycles for 2k of MFMAs).
template <int N, int DEPTH, class T, class LD, class USE>
__device__ __forceinline__ void read_ahead(LD&& ld, USE&& use) {
  constexpr int A = DEPTH < N ? DEPTH : N;
  T f[A];
  static_for<0, A>([&](auto i) { f[i.value] = ld(i); });
  static_for<0, N>([&](auto i) {
    use(i, f[i.value % A]);
    if constexpr (i.value + A < N) f[i.value % A] = ld(std::integral_constant<int, i.value + A>{});
    __builtin_amdgcn_sched_barrier(0);
  });
}

// A query row as B operand: chunk j's elements 32 j + 8 g .. + 7
template <int N>
__device__ inline void load_q(const uint16_t* q, int g, v8h (&qf)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) qf[j] = *reinterpret_cast<const v8h*>(q + 32 * j + 8 * g);
}
// Its registers, zeros where there is no row. The compiler's wait for the
// loads stands here, behind the first tile's loads and before the tile loop,
// where it would wait for that loop's loads.
// An Inf becomes a NaN (q 0 + q, which leaves all finite values): the softmax
// over scores that hold one is NaN in either case, and so that all of them are
// NaN, not -inf as where a key is masked.
template <int N>
__device__ inline void settle(v8h (&qf)[N], bool live) {
  const v8h zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    qf[j] = live ? __builtin_elementwise_fma(qf[j], zero, qf[j]) : zero;
    pin(qf[j]);
  }
}

// Scores of NST subtiles of 16 keys for NR groups of 16 rows, over NCH chunks
template <int HD, int NST, int NR, int NCH, int DEPTH>
__device__ __forceinline__ void pg_scores(const PgLane<HD>& at, const v8h (&qf)[NR][NCH], v4f (&s)[NR][NST]) {
  constexpr int CH = NST * NR >= 4 || (NR == 2 && HD == 256) ? 1 : NST * NR == 2 ? 2 : 4;  // chains, so that MFMAs do
                                                                                      // not wait (a second one spills)
  v4f t[CH][NR][NST];
#pragma unroll
  for (int h = 0; h < CH; ++h)
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int st = 0; st < NST; ++st) t[h][r][st] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  read_ahead<NCH * NST, DEPTH, v8h>(
      [&](auto i) { return at.template k<i.value % NST, i.value / NST>(); },
      [&](auto i, v8h k) {
        constexpr int j = i.value / NST, st = i.value % NST;
#pragma unroll
        for (int r = 0; r < NR; ++r)
          t[j % CH][r][st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[r][j], t[j % CH][r][st], 0, 0, 0);
      });
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      s[r][st] = t[0][r][st];
      if constexpr (CH == 2) s[r][st] += t[1][r][st];
      if constexpr (CH == 4) s[r][st] = (s[r][st] + t[1][r][st]) + (t[2][r][st] + t[3][r][st]);
    }
}

// Weights of a lane's scores (NST subtiles of 4 keys; -inf where masked) as
// 2^(s log2e - ref), and the move of ref. A NaN passes the maximum by and ends
// in sum and acc. acc: NA accumulators to rescale; sum: of the lane's keys in
// fp32. A weight is the sum of two fp16 values, its leading bits and what they
// leave over, to 2^-20 of itself (rounded towards zero: two at a time in one
// instruction; 2^-30 of the row's largest where the second one is subnormal):
// the output is the mean of V rows under the weights that the sum holds, also
// where one key has nearly all of the weight.
// HL: lanes 8 .. 15 of a row's 16 hold the same rows as lanes 0 .. 7 and take
// the second values (w[0] of such a lane); else a lane has both.
template <bool HL>
constexpr int PG_PARTS = HL ? 1 : 2;
template <int NST, int NA, bool HL>
__device__ __forceinline__ void pg_weights(const v4f (&s)[NST], float& ref, v4f (&acc)[NA], float& sum,
                                           v4h (&w)[PG_PARTS<HL>][NST]) {
  float top = -INFINITY;
#pragma unroll
  for (int st = 0; st < NST; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, s[st][e]);
  top = slot_reduce<16, true>(top) * PG_LOG2E;
  const bool move = top > ref + PG_MOVE || (ref == -INFINITY && top > ref);
  if (__any(move)) {
    const float to = move ? top - PG_BELOW : ref;
    const float corr = move ? __builtin_amdgcn_exp2f(ref - to) : 1.0f;
    ref = to;
    sum *= corr;
#pragma unroll
    for (int d = 0; d < NA; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[d][e] *= corr;
  }
  const float r = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
  for (int st = 0; st < NST; ++st)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[st][e], PG_LOG2E, -r));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[st][e + 1], PG_LOG2E, -r));
      sum += p0;
      sum += p1;
      const v2h hi = cvt_rtz(p0, p1);
      const v2h lo = cvt_rtz(fmaf((float)hi[0], -1.0f, p0), fmaf((float)hi[1], -1.0f, p1));
      if constexpr (HL) {
        const bool low = threadIdx.x & 8;
        w[0][st][e] = low ? lo[0] : hi[0];
        w[0][st][e + 1] = low ? lo[1] : hi[1];
      } else {
        w[0][st][e] = hi[0], w[0][st][e + 1] = hi[1];
        w[1][st][e] = lo[0], w[1][st][e + 1] = lo[1];
      }
    }
}

// The reference that a row's part leaves, -inf where it has no keys. Where
// its sum is NaN +inf, so that the join takes it for the largest: the other
// parts' factors are then 0, this one's 2^(inf - inf) and the output are NaN.
__device__ inline float part_ref(float ref, float sum) { return sum == sum ? ref : INFINITY; }

// O^T += V^T P^T, for both parts of the weights
template <int HD, int NST, int NR, int NDT, int DEPTH, int PARTS>
__device__ __forceinline__ void pg_values(const PgLane<HD>& at, const v4h (&w)[NR][PARTS][NST], v4f (&acc)[NR][NDT]) {
  if constexpr (NST == 1) {  // both parts in one MFMA of 32 products, as 16 keys twice: the time of one of 16
    read_ahead<NDT, DEPTH, v4h>([&](auto i) { return at.template v<0, i.value>(); },
                                [&](auto i, v4h v) {
#pragma unroll
                                  for (int r = 0; r < NR; ++r)
                                    if constexpr (PARTS == 2)
                                      acc[r][i.value] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                          join(v, v), join(w[r][0][0], w[r][1][0]), acc[r][i.value], 0, 0, 0);
                                    else
                                      acc[r][i.value] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, w[r][0][0], acc[r][i.value], 0, 0, 0);
                                });
  } else {
    constexpr int NP = NST / 2;  // pairs of subtiles: 32 keys of one MFMA
    v8h wp[NR][PARTS][NP];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int k = 0; k < NP; ++k) wp[r][p][k] = join(w[r][p][2 * k], w[r][p][2 * k + 1]);
    read_ahead<NDT * NP, DEPTH, v8h>(
        [&](auto i) {
          constexpr int d = i.value / NP, k = i.value % NP;
          return join(at.template v<2 * k, d>(), at.template v<2 * k + 1, d>());
        },
        [&](auto i, v8h v) {
          constexpr int d = i.value / NP, k = i.value % NP;
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int r = 0; r < NR; ++r)
              acc[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wp[r][p][k], acc[r][d], 0, 0, 0);
        });
  }
}

struct PgArgs {
  const uint16_t *q, *kc, *vc;
  uint16_t* out;
  float* ws;        // accumulators [T nH][np][HD], then (ref, sum) [T nH][np][2]
  int ldq, ldo, T, nH, nkv, grp, window;
  int nsp, nso, np; // splits of the prefix and of the own keys, their sum
  int nrb, nhb;     // row blocks of the prefix, head blocks of a token's own pages
};
__device__ inline long pg_part(const PgArgs& a, int row, int part) { return (long)row * a.np + part; }
template <int HD>
__device__ inline float* pg_ml(const PgArgs& a, long part) { return a.ws + (long)a.T * a.nH * a.np * HD + 2 * part; }

// Token t's sequence, position and the first position that it attends.
template <bool UNIFORM>
__device__ inline bool pg_token(const Pages& pg, int t, int window, int& s, int& pos, int& lo) {
  s = UNIFORM ? uload(pg.seq, t) : pg.seq[t];
  pos = UNIFORM ? uload(pg.pos, t) : pg.pos[t];
  lo = window > 0 ? max(0, max(pos, 0) - window + 1) : 0;
  return s >= 0 && s < pg.nseq && pos >= 0;
}

// A lane's rows 16 r + c of the prefix rows from r0 on, and the span of their
// keys over the wave: first and last key of any row (blo, bhi), keys that
// every row has (wlo .. whi - 1). Loads NCH chunks of the rows from element e0.
template <int CTRL>
__device__ inline int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
template <bool MAX>
__device__ inline int row16_reduce(int v) {
  auto op = [](int a, int b) { return MAX ? max(a, b) : min(a, b); };
  v = op(v, dpp_i<DPP_XOR1>(v));
  v = op(v, dpp_i<DPP_XOR2>(v));
  v = op(v, dpp_i<DPP_MIRROR8>(v));
  return op(v, dpp_i<DPP_MIRROR16>(v));
}
template <int HD, int NR, int NCH>
struct PgRows {
  int pos[NR];  // -1: no row
  int blo, bhi, wlo, whi;
  bool any;
  static __device__ inline int row(const PgArgs& a, int kvh, int R) { return R / a.grp * a.nH + kvh * a.grp + R % a.grp; }
  // whether row r has key `key` < P
  __device__ inline bool has(int r, int key, int window) const {
    return key <= pos[r] && (window == 0 || key > pos[r] - window);
  }
  __device__ inline PgRows(const PgArgs& a, const Pages& pg, int kvh, int r0, int e0, int P, v8h (&qf)[NR][NCH]) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, nrows = a.T * a.grp;
    blo = 0x7FFFFFFF, bhi = 0, wlo = 0, whi = 0x7FFFFFFF;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int R = r0 + 16 * r + c, t = min(R, nrows - 1) / a.grp;
      load_q(a.q + (long)t * a.ldq + (long)(kvh * a.grp + min(R, nrows - 1) % a.grp) * HD + e0, g, qf[r]);
      int s, p, lo;
      const bool live = pg_token<false>(pg, t, a.window, s, p, lo) && R < nrows;
      const int hi = min(p, P - 1) + 1;
      pos[r] = live ? p : -1;
      if (live) {
        if (lo < hi) blo = min(blo, lo), bhi = max(bhi, hi);
        wlo = max(wlo, lo), whi = min(whi, hi);
      }
    }
    any = __any(pos[0] >= 0 || pos[NR - 1] >= 0);
    blo = __builtin_amdgcn_readfirstlane(row16_reduce<false>(blo));
    bhi = __builtin_amdgcn_readfirstlane(row16_reduce<true>(bhi));
    wlo = __builtin_amdgcn_readfirstlane(row16_reduce<true>(wlo));
    whi = __builtin_amdgcn_readfirstlane(row16_reduce<false>(whi));
  }
};

// NR groups of 16 rows per wave. Up to head dim 256 a wave holds its rows by
// itself; behind a long prefix the cache's bytes bound it (8 rows of 32 heads
// of 128 behind 32001 keys and 150 own: 134 MB in 32 us, 4.2 TB/s; its loads
// and barriers alone 24.3, and a start of ~3 us before the first tile); with
// many rows the weights' second parts show (64 rows there: 72 us, with weights
// of one fp16 value 61). Head dim 512 takes two waves per NR groups, each with
// half of the elements: of q for the scores, whose halves the pair adds
// through LDS, and of the outputs. So a wave's registers stay within 256 and
// two waves share a SIMD (one wave of 465 registers issued at most one
// instruction per 4 cycles, 840 a tile beside 2k cycles of MFMAs: with weights
// of one fp16 value 76 us per 23.8k keys for 64 rows of 16 heads, with pairs
// 68). What bounds it then (64 rows of 16 heads behind 32000 keys: 135 us, 3.3
// per 1000 keys; with weights of one value 113 and 2.7): softmax, score
// exchange and barriers beside the matrix products, with one workgroup's 160
// KB of LDS per CU nothing to run under them. Behind 8192 keys and up to 1000
// own (60 us, 18.2 GFLOP) it is the grid: the plan's 160 workgroups of the
// prefix take 58 us by themselves, on 160 of 256 CUs, where 8192 keys over all
// CUs would take 27; the own pages alone take 18.5.
template <int HD, int NR>
__device__ __forceinline__ void shared_role(const PgArgs& a, const Pages& pg, uint32_t lds, uint32_t xs, int bid) {
  using S = PgTile<HD>;
  constexpr int KT = S::KT, NST = KT / 16, DS = S::DS, NCH = S::NCH / DS, NDT = S::NDT / DS;
  constexpr int NW = PG_WAVES * DS, KW = KT / NW, HW = HD / DS;
  constexpr int DEPTH = DS == 2 ? 3 : 4;  // (a fourth spills in the tile loop; with three, one
                                          // register is saved before it and read back behind it)
  const int kvh = bid % a.nkv, split = bid / a.nkv % a.nsp, rb = bid / (a.nkv * a.nsp);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15,
            g = lane >> 4, dp = wave % DS;
  const int P = pg.prefix_keys(), r0 = (rb * PG_WAVES + wave / DS) * 16 * NR;
  v8h qf[NR][NCH];
  const PgRows<HD, NR, NCH> rows(a, pg, kvh, r0, dp * HW, P, qf);
  // the keys of all waves' rows: the whole prefix, which is known before the rows are, or the windows' part of it
  int blo = 0, bhi = P;
  if (a.window > 0) {
    if (lane == 0) {
      lds_write<int>(xs + 8 * wave, rows.blo);
      lds_write<int>(xs + 8 * wave + 4, rows.bhi);
    }
    __syncthreads();
    blo = 0x7FFFFFFF, bhi = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      blo = min(blo, __builtin_amdgcn_readfirstlane(lds_read<int>(xs + 8 * w)));
      bhi = max(bhi, __builtin_amdgcn_readfirstlane(lds_read<int>(xs + 8 * w + 4)));
    }
  }
  // this split's keys: whole tiles from the 16-key group of the first one on
  const int b16 = blo & ~15, per = KT * max(1, (int)ceil_div(max(0, bhi - b16), (long)KT * a.nsp));
  const int k0 = bhi > blo ? b16 + split * per : 0, k1 = bhi > blo ? min(k0 + per, bhi) : 0;

  float ref[NR], sum[NR];
  v4f acc[NR][NDT];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    ref[r] = -INFINITY;
    sum[r] = 0.0f;
#pragma unroll
    for (int d = 0; d < NDT; ++d) acc[r][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  PgLane<HD> at(lds + dp * HW * 2, lds + KT * HD * 2 + dp * HW * 2);
  const uint32_t koff = load_off<HD, false>(wave * KW), voff = load_off<HD, true>(wave * KW);
  const int mask = (1 << pg.lg) - 1;
  // pages of a tile's 16-key groups and of the wave's part of it, as they stand in the array (past the split's
  // last key: that key's page)
  auto page_of = [&](int key) { return uload(pg.prefix_pages, min(key, k1 - 1) >> pg.lg); };
  auto held = [&](int id) { return id >= 0 && id < pg.npages; };
  auto load = [&](int t0, int p, uint32_t tile) {
    const int key = t0 + wave * KW;
    const long o = ((((long)p * a.nkv + kvh) << pg.lg) + (key & mask)) * HD;
    load_rows<HD, KW, false>(a.kc + o, koff, tile, wave * KW, key, blo, k1, held(p));
    load_rows<HD, KW, true>(a.vc + o, voff, tile + KT * HD * 2, wave * KW, key, blo, k1, held(p));
  };
  int id[NST], nid[NST], mine = 0;  // pages of this tile and the next one, the wave's page of the next one
  if (k0 < k1) {
    load(k0, page_of(k0 + wave * KW), lds);
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      id[st] = page_of(k0 + 16 * st);
      nid[st] = page_of(k0 + KT + 16 * st);
    }
    mine = page_of(k0 + KT + wave * KW);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) settle(qf[r], rows.pos[r] >= 0);
  int by = S::STAGE;
  for (int t0 = k0; t0 < k1; t0 += KT, by = -by) {
    vmwait<0>();      // this wave's rows of the tile
    __syncthreads();  // every wave's; and every wave is done with the tile before
    if (t0 + KT < k1) {
      load(t0 + KT, mine, lds + (by > 0 ? S::STAGE : 0));
      mine = page_of(t0 + 2 * KT + wave * KW);
    }
    v4f s[NR][NST];
    if (DS == 2 || rows.any) pg_scores<HD, NST, NR, NCH, DEPTH>(at, qf, s);
    if constexpr (DS == 2) {  // add the pair's halves; both waves add the same two values
      const uint32_t x = xs + 16 * lane;
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int st = 0; st < NST; ++st) lds_write<v4f>(x + 1024 * (wave * NR * NST + r * NST + st), s[r][st]);
      lgkm0();
      __builtin_amdgcn_s_barrier();  // (not __syncthreads, which may wait for the tile loads)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int st = 0; st < NST; ++st) s[r][st] += lds_read<v4f>(x + 1024 * ((wave ^ 1) * NR * NST + r * NST + st));
    }
    if (DS == 2 || rows.any) {
      bool whole = t0 >= rows.wlo && t0 + KT <= rows.whi;
#pragma unroll
      for (int st = 0; st < NST; ++st) whole = whole && held(id[st]);
      if (!whole) {  // (uniform) some key is masked for some row
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int st = 0; st < NST; ++st)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = t0 + 16 * st + 4 * g + e;
              if (!(held(id[st]) && key < k1 && rows.has(r, key, a.window))) s[r][st][e] = -INFINITY;
            }
      }
      v4h w[NR][2][NST];
#pragma unroll
      for (int r = 0; r < NR; ++r) pg_weights<NST, NDT, false>(s[r], ref[r], acc[r], sum[r], w[r]);
      pg_values<HD, NST, NR, NDT, DEPTH>(at, w, acc);
    }
    at.move(by);
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      id[st] = nid[st];
      nid[st] = page_of(t0 + 2 * KT + 16 * st);
    }
  }
  // ---- this split's part of each row (a part without keys: its reference alone) ----
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float l = slot_reduce<16>(sum[r]);
    ref[r] = part_ref(ref[r], l);
    if (rows.pos[r] < 0) continue;
    const long part = pg_part(a, rows.row(a, kvh, r0 + 16 * r + c), split);
    if (g == 0 && dp == 0) {
      float* ml = pg_ml<HD>(a, part);
      ml[0] = ref[r];
      ml[1] = l;
    }
    if (ref[r] == -INFINITY) continue;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
      *reinterpret_cast<v4f*>(a.ws + part * HD + dp * HW + 16 * d + 4 * g) = acc[r][d];
  }
}

// OWN: item = (token, KV head, block of 16 heads, split) on the token's own
// pages; else (KV head, split) on the prefix for all rows.
template <int HD, bool HL, bool OWN>
__device__ __forceinline__ void stream_role(const PgArgs& a, const Pages& pg, uint32_t lds, float (*ml)[16][2], int item) {
  using S = PgTile<HD>;
  constexpr int OKT = S::OKT, NST = OKT / 16, NCH = S::NCH, NDT = S::NDT, NI = OKT / S::KPI, DEPTH = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15,
            g = lane >> 4;
  const int nsplit = OWN ? a.nso : a.nsp, nhb = OWN ? a.nhb : 1;
  const int kvh = OWN ? item / (nsplit * nhb) % a.nkv : item % a.nkv, split = OWN ? item % nsplit : item / a.nkv;
  const int hb = OWN ? item / nsplit % nhb : 0, t = OWN ? item / (nsplit * nhb * a.nkv) : 0;
  const int P = OWN ? pg.prefix() : pg.prefix_keys();

  // ---- rows, and the keys lo .. hi - 1 of them all (OWN: of the own pages) ----
  v8h qf[1][NCH];
  int lo, hi, wlo, whi, pos, heads = 16;  // pos: of the token, or of the lane's prefix row
  const int32_t* tab = pg.prefix_pages;
  if constexpr (OWN) {
    heads = min(a.grp - 16 * hb, 16);
    const int hc = HL ? c & 7 : c;
    load_q(a.q + (long)t * a.ldq + (long)(kvh * a.grp + 16 * hb + (hc < heads ? hc : 0)) * HD, g, qf[0]);
    int s;
    if (!pg_token<true>(pg, t, a.window, s, pos, lo)) return;  // (uniform) no row
    lo = max(0, lo - P);
    hi = min(pos - P, pg.max_own - 1) + 1;
    if (hi <= lo) lo = hi = 0;  // no keys (a position far past max_own: lo + split * per would pass 32 bits)
    tab = pg.table + (long)s * pg.ld;
    wlo = lo, whi = hi;
  } else {
    const PgRows<HD, 1, NCH> rows(a, pg, kvh, 0, 0, P, qf);
    lo = a.window > 0 ? rows.blo : 0, hi = a.window > 0 ? rows.bhi : P, wlo = rows.wlo, whi = rows.whi;
    if (hi <= lo) lo = hi = 0;
    pos = rows.pos[0];
  }
  // this split: groups of 4 tiles from the 16-key group of the first key on
  const int l16 = lo & ~15, per = 4 * OKT * max(1, (int)ceil_div(max(0, hi - l16), 4l * OKT * nsplit));
  const int k0 = l16 + split * per, k1 = min(k0 + per, hi);

  float ref = -INFINITY, sum = 0.0f;
  v4f acc[1][NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) acc[0][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t kt = lds + wave * S::REGION, vt = kt + OKT * HD * 2;
  const PgLane<HD> at(kt, vt);
  const uint32_t koff = load_off<HD, false>(0), voff = load_off<HD, true>(0);
  const int mask = (1 << pg.lg) - 1;
  auto page_of = [&](int key) { return uload(tab, min(key, k1 - 1) >> pg.lg); };
  auto held = [&](int id) { return id >= 0 && id < pg.npages; };
  auto load = [&](int t0, const int (&id)[NST], auto v) {
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      const int key = t0 + 16 * st;
      const long o = ((((long)id[st] * a.nkv + kvh) << pg.lg) + (key & mask)) * HD;
      load_rows<HD, 16, v.value>((v.value ? a.vc : a.kc) + o, v.value ? voff : koff, v.value ? vt : kt, 16 * st, key, lo,
                                 k1, held(id[st]));
    }
  };
  constexpr std::integral_constant<bool, false> KEYS;
  constexpr std::integral_constant<bool, true> VALUES;
  int id[NST], nid[NST];
  int t0 = k0 + OKT * wave;
  if (t0 < k1) {
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      id[st] = page_of(t0 + 16 * st);
      nid[st] = page_of(t0 + 4 * OKT + 16 * st);
    }
    load(t0, id, KEYS);
    load(t0, id, VALUES);
  }
  settle(qf[0], OWN ? (HL ? c & 7 : c) < heads : pos >= 0);
  for (; t0 < k1; t0 += 4 * OKT) {
    const bool more = t0 + 4 * OKT < k1;
    vmwait<NI>();  // the K rows; the V rows may be on their way
    v4f s[1][NST];
    pg_scores<HD, NST, 1, NCH, DEPTH>(at, qf, s);
    lgkm0();  // the K rows are read: the next tile's may land
    if (more) load(t0 + 4 * OKT, nid, KEYS);
    bool whole = t0 >= wlo && t0 + OKT <= min(whi, k1);
#pragma unroll
    for (int st = 0; st < NST; ++st) whole = whole && held(id[st]);
    if (!whole) {  // (uniform)
#pragma unroll
      for (int st = 0; st < NST; ++st)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = t0 + 16 * st + 4 * g + e;
          const bool in = OWN ? key >= lo : key <= pos && (a.window == 0 || key > pos - a.window);
          if (!(held(id[st]) && key < k1 && in)) s[0][st][e] = -INFINITY;
        }
    }
    v4h w[1][PG_PARTS<HL>][NST];
    pg_weights<NST, NDT, HL>(s[0], ref, acc[0], sum, w[0]);
    if (more) vmwait<NI>();
    else vmwait<0>();
    pg_values<HD, NST, 1, NDT, 4>(at, w, acc);
    lgkm0();
    if (more) load(t0 + 4 * OKT, nid, VALUES);
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      id[st] = nid[st];
      nid[st] = page_of(t0 + 8 * OKT + 16 * st);
    }
  }
  // ---- the waves join: a row's 16-byte pieces lie at (piece ^ row) in each wave's region ----
#pragma unroll
  for (int d = 0; d < NDT; ++d) lds_write<v4f>(kt + c * HD * 4 + 16 * ((4 * d + g) ^ c), acc[0][d]);
  const float l = slot_reduce<16>(sum);
  if (g == 0) {
    ml[wave][c][0] = part_ref(ref, l);
    ml[wave][c][1] = l;
  }
  __syncthreads();
  const int n = OWN ? heads : min(16, a.T * a.grp);
  for (int i = tid; i < n * (HD / 4); i += PG_THREADS) {
    const int h = i / (HD / 4), pc = i % (HD / 4);
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) top = fmaxf(top, ml[w][h][0]);
    float L = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {
      const float m = ml[w][h][0], e = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
      for (int k = 0; k < (HL ? 2 : 1); ++k) {  // with HL a row's leftover lies 8 rows on
        const int hh = h + 8 * k;
        const v4f v = lds_read<v4f>(lds + w * S::REGION + hh * HD * 4 + 16 * (pc ^ hh));
        if (k == 0) L = fmaf(ml[w][hh][1], e, L);
#pragma unroll
        for (int u = 0; u < 4; ++u) o[u] = fmaf(v[u], e, o[u]);
      }
    }
    const int row = OWN ? t * a.nH + kvh * a.grp + 16 * hb + h : PgRows<HD, 1, NCH>::row(a, kvh, h);
    if (OWN && a.np == 1) {
      const float inv = top == -INFINITY ? 0.0f : 1.0f / L;
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = f2h(o[k] * inv);
      *reinterpret_cast<v2u*>(a.out + (long)t * a.ldo + (long)(row - t * a.nH) * HD + 4 * pc) =
          v2u{b[0] | b[1] << 16, b[2] | b[3] << 16};
    } else {
      const long part = pg_part(a, row, (OWN ? a.nsp : 0) + split);
      if (pc == 0) {
        float* m = pg_ml<HD>(a, part);
        m[0] = top;
        m[1] = L;
      }
      if (top != -INFINITY) *reinterpret_cast<v4f*>(a.ws + part * HD + 4 * pc) = o;
    }
  }
}

// HL: up to 8 query heads per KV head, so that the idle lanes of the own
// pages' rows take the weights' second parts.
template <int HD, int MODE, bool HL>
__global__ void __launch_bounds__(PgTile<HD>::threads(MODE), PgTile<HD>::waves(MODE))
paged_attn_kernel(const PgArgs a, const Pages pg) {
  using S = PgTile<HD>;
  __shared__ __attribute__((aligned(256))) uint8_t tiles[S::lds(MODE)];
  const uint32_t lds = lds_addr(tiles);
  float(*ml)[16][2] = reinterpret_cast<float(*)[16][2]>(tiles + S::tiles(MODE));
  const int npre = MODE == PG_OWN ? 0 : a.nrb * a.nkv * a.nsp;
  if ((int)blockIdx.x >= npre) {
    if (S::threads(MODE) > PG_THREADS && threadIdx.x >= PG_THREADS) return;  // streams take 4 waves
    stream_role<HD, HL, true>(a, pg, lds, ml, blockIdx.x - npre);
  } else if constexpr (MODE == PG_SHARED) shared_role<HD, 2>(a, pg, lds, lds + S::tiles(MODE), blockIdx.x);
  else if constexpr (MODE == PG_SHARED_FEW) shared_role<HD, 1>(a, pg, lds, lds + S::tiles(MODE), blockIdx.x);
  else if constexpr (MODE == PG_STREAM) stream_role<HD, false, false>(a, pg, lds, ml, blockIdx.x);
}

// Output row blockIdx.x (token, head): sum_i e_i acc_i / sum_i e_i l_i over
// the row's parts, e_i = 2^(ref_i - largest ref), parts without keys left out.
// Groups of lanes take every NG-th part, 4 elements (8 at HD 512) per lane.
// Bound by the launch and one round trip of loads for few parts (3.5 - 5 us),
// by the parts' bytes for many (1024 rows of 512 in 24 parts: 10.4 us).
constexpr int PG_MAX_PARTS = 512;
template <int HD>
__global__ void __launch_bounds__(PG_THREADS) paged_merge_kernel(const PgArgs a, const Pages pg) {
  constexpr int EPL = HD == 512 ? 8 : 4, LPG = HD / EPL, NG = PG_THREADS / LPG;
  __shared__ float wt[PG_MAX_PARTS], red[2][PG_WAVES];
  __shared__ __attribute__((aligned(16))) float os[NG][HD];
  const int row = blockIdx.x, t = row / a.nH, h = row % a.nH, tid = threadIdx.x;
  const int s = pg.seq[t];
  if (s < 0 || s >= pg.nseq || pg.pos[t] < 0) return;  // (uniform) no row
  const float* ml = a.ws + (long)a.T * a.nH * a.np * HD + 2 * pg_part(a, row, 0);
  float top = -INFINITY;
  for (int i = tid; i < a.np; i += PG_THREADS) top = fmaxf(top, ml[2 * i]);
  top = reduce64<true>(top);
  if ((tid & 63) == 0) red[0][tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float L = 0.0f;
  for (int i = tid; i < a.np; i += PG_THREADS) {
    const float m = ml[2 * i], e = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    wt[i] = e;
    if (e != 0.0f) L = fmaf(ml[2 * i + 1], e, L);
  }
  L = reduce64<false>(L);
  if ((tid & 63) == 0) red[1][tid >> 6] = L;
  __syncthreads();
  L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int gi = tid / LPG, i0 = EPL * (tid % LPG);
  const float* w = a.ws + pg_part(a, row, 0) * HD + i0;
  v4f o[EPL / 4] = {};
  // PB parts at a time with all loads in flight (one at a time: 10 us for 113 parts of 64 rows of 512, now 5)
  constexpr int PB = 4;
  for (int i = gi; i < a.np; i += PB * NG) {
    v4f v[PB][EPL / 4];
    float e[PB];
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      const int part = min(i + j * NG, a.np - 1);
      e[j] = i + j * NG < a.np ? wt[part] : 0.0f;
#pragma unroll
      for (int k = 0; k < EPL / 4; ++k) v[j][k] = *reinterpret_cast<const v4f*>(w + (long)part * HD + 4 * k);
    }
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      if (e[j] == 0.0f) continue;  // (a part without keys was not written)
#pragma unroll
      for (int k = 0; k < EPL / 4; ++k)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[k][u] = fmaf(v[j][k][u], e[j], o[k][u]);
    }
  }
#pragma unroll
  for (int k = 0; k < EPL / 4; ++k) *reinterpret_cast<v4f*>(&os[gi][i0 + 4 * k]) = o[k];
  __syncthreads();
  const float inv = top == -INFINITY ? 0.0f : 1.0f / L;
  for (int i = tid; i < HD / 2; i += PG_THREADS) {
    float x = 0.0f, y = 0.0f;
#pragma unroll
    for (int gg = 0; gg < NG; ++gg) {
      x += os[gg][2 * i];
      y += os[gg][2 * i + 1];
    }
    reinterpret_cast<uint32_t*>(a.out + (long)t * a.ldo + (long)h * HD)[i] = (uint32_t)f2h(x * inv) | (uint32_t)f2h(y * inv) << 16;
  }
}

// Splits of the prefix and of the own keys, from the sizes and bounds alone,
// for about one workgroup of each shape per place on the chip (2 per CU up to
// hd 256, 1 at 512).
//  * prefix: more splits fill the chip, but each takes a part through memory,
//    8 hd bytes per row out and in. With a time per key and one per part the
//    sum is least at a square root of the keys per row; its factor is measured
//    (64 rows of 16 heads of 512 behind 8192 keys, with the merge: 25 85.0 us,
//    50 70.9, 100 80.6; 18 rows of 16 heads of 256 behind 2000: 17.0, 16.9,
//    16.5; 8 rows of 32 heads of 128 behind 32001: 37.8, 37.1, 37.3); at least
//    two tiles per split.
//  * own: up to 4 rounds of workgroups while a split keeps 8 tiles per wave, so
//    that ragged lengths even out.
struct PgPlan {
  int nsp, nso, nrb, nhb, mode;
};
static PgPlan pg_plan(int T, int nH, int nkv, int hd, int max_prefix, int max_own, int window) {
  const int grp = nH / nkv, per_cu = hd == 512 ? 1 : 2, places = 256 * per_cu;
  const int kt = hd >= 256 ? 32 : 64, okt = hd >= 256 ? 16 : 32;
  auto clamp = [](long v, long hi) { return (int)min(max(v, 1l), max(min(hi, PG_MAX_PARTS / 2l), 1l)); };
  PgPlan p{};
  const long rows = (long)T * grp;
  p.mode = !max_prefix ? PG_OWN : rows <= PG_STREAM_ROWS ? PG_STREAM : rows <= PG_FEW_ROWS ? PG_SHARED_FEW : PG_SHARED;
  p.nhb = ceil_div(grp, 16);
  if (max_prefix) {
    const int span = window > 0 ? min(window, max_prefix) : max_prefix;
    p.nrb = p.mode == PG_SHARED ? ceil_div(rows, 128) : 1;
    const long even = (long)sqrt(50.0 * per_cu * span / ((double)T * nH));
    p.nsp = clamp(min(places / ((long)p.nrb * nkv), even), ceil_div(span, 2 * kt));
  }
  const int span = window > 0 ? min(window, max_own) : max_own;
  const long items = (long)T * nkv * p.nhb;
  p.nso = clamp(min(4 * places / items, max(places / items, (long)ceil_div(span, 32 * okt))), ceil_div(span, 4 * okt));
  return p;
}

// A launch holds fewer than 2^32 threads: this many workgroups of 256, half as many of 512.
constexpr long PG_MAX_BLOCKS = 1l << 24;

// log2 of a page of 16 .. 4096 rows, -1 for any other size
static int page_lg(int page) {
  for (int lg = 4; lg <= 12; ++lg)
    if (page == 1 << lg) return lg;
  return -1;
}

}  // namespace q4

using namespace q4;

extern "C" {

int q4_paged_prep(const void* qkv, int dtype, int ld, int qoff, int koff, int voff, const float* qnw,
                  const float* knw, const float* cos_tab, const float* sin_tab, int max_pos, uint16_t* q, int ldq,
                  uint16_t* kc, uint16_t* vc, int npages, int page, const int32_t* table, int table_ld, int nseq,
                  const int32_t* prefix_len, const int32_t* seq, const int32_t* pos, int T, int nH, int nkv, int hd,
                  void* stream) {
  clear_error();
  Q4_ARG(qkv && qnw && knw && cos_tab && sin_tab && q && kc && vc && table && seq && pos, "null pointer");
  Q4_ARG(dtype == Q4_DT_F32 || dtype == Q4_DT_F16, "bad dtype");
  Q4_ARG(hd == 64 || hd == 128 || hd == 256 || hd == 512, "paged prep takes head dims 64/128/256/512 (got %d)", hd);
  Q4_ARG(T > 0 && nH > 0 && nkv > 0 && max_pos > 0 && npages > 0 && nseq > 0 && table_ld > 0, "bad sizes");
  const int lg = page_lg(page);
  Q4_ARG(lg > 0, "page=%d is not a power of two of 16..4096 rows", page);
  Q4_ARG(qoff >= 0 && koff >= 0 && voff >= 0 && (long)qoff + (long)nH * hd <= ld && (long)koff + (long)nkv * hd <= ld &&
             (long)voff + (long)nkv * hd <= ld,
         "q, k or v reach past the row stride %d", ld);
  Q4_ARG(ldq >= (long)nH * hd && ldq % 8 == 0, "row stride ldq=%d must be a multiple of 8 of at least nH * hd = %ld",
         ldq, (long)nH * hd);
  const int un = dtype == Q4_DT_F16 ? 8 : 4;
  Q4_ARG(ld % un == 0 && qoff % un == 0 && koff % un == 0 && voff % un == 0,
         "ld and the q, k, v offsets must be multiples of 16 bytes");
  for (const void* p : {qkv, (const void*)qnw, (const void*)knw, (const void*)cos_tab, (const void*)sin_tab,
                        (const void*)q, (const void*)kc, (const void*)vc})
    Q4_ARG(((uintptr_t)p & 15) == 0, "qkv, qnw, knw, the tables, q, kc and vc must be 16-byte aligned");
  Q4_ARG(T < PG_MAX_BLOCKS, "a batch of %d rows is too large", T);
  const size_t cache = (size_t)npages * nkv * page * hd * 2, nq = ((size_t)(T - 1) * ldq + (size_t)nH * hd) * 2;
  const size_t nx = ((size_t)(T - 1) * ld + max(qoff + nH * hd, max(koff, voff) + nkv * hd)) * (dtype == Q4_DT_F16 ? 2 : 4);
  Q4_ARG(!overlap(q, nq, qkv, nx), "q must not overlap qkv");
  Q4_ARG(!overlap(kc, cache, vc, cache), "kc and vc must not overlap");
  for (const void* c : {kc, vc})
    Q4_ARG(!overlap(c, cache, q, nq) && !overlap(c, cache, qkv, nx), "the cache must not overlap q or qkv");
  const Pages pg{nullptr, prefix_len, table, seq, pos, table_ld, nseq, npages, lg, 0, 0};
  const int groups = 256 / (hd / 8), heads = nH + 2 * nkv;
  hipStream_t st = as_stream(stream);
  // heads per group of lanes: few where the workgroups do not fill the chip (64 rows of 16 + 2 x 8 heads of 256: 4.8 us
  // with 4, 3.9 with 2 or 1; 976 rows 9.8, 9.6, 9.8), 4 share a row's RoPE loads where they do (1952 rows: 16.2, 16.8,
  // 17.4; 2048 rows of 16 + 2 heads of 512: 18.4, 19.7, 22.1; 1024 rows 10.6, 10.3, 10.9)
  const int hpg = (long)T * ceil_div(heads, groups) <= 6144 ? 2 : 4;
#define PG_PREP(HD, DT, HPG) \
  hipLaunchKernelGGL((paged_prep_kernel<HD, DT, HPG>), dim3(T, ceil_div(heads, HPG * groups)), dim3(256), 0, st, qkv, \
                     ld, qoff, koff, voff, qnw, knw, cos_tab, sin_tab, max_pos, q, ldq, kc, vc, nH, nkv, pg)
#define PG_PREP_DT(HD, DT)              \
  if (hpg == 2) PG_PREP(HD, DT, 2); \
  else PG_PREP(HD, DT, 4)
#define PG_PREP_HD(HD)                                 \
  if (dtype == Q4_DT_F16) { PG_PREP_DT(HD, Q4_DT_F16); } \
  else { PG_PREP_DT(HD, Q4_DT_F32); }
  switch (hd) {
    case 64: PG_PREP_HD(64); break;
    case 128: PG_PREP_HD(128); break;
    case 256: PG_PREP_HD(256); break;
    default: PG_PREP_HD(512); break;
  }
#undef PG_PREP_HD
#undef PG_PREP_DT
#undef PG_PREP
  Q4_LAUNCHED("paged_prep");
  return Q4_OK;
}

size_t q4_paged_attn_workspace_bytes(int T, int nH, int nkv, int hd, int max_prefix, int max_own, int window) {
  if (T <= 0 || nH <= 0 || nkv <= 0 || nH % nkv || hd <= 0 || max_prefix < 0 || max_own <= 0 || window < 0) return 0;
  const PgPlan p = pg_plan(T, nH, nkv, hd, max_prefix, max_own, window);
  const int np = p.nsp + p.nso;
  return np == 1 ? 0 : (size_t)T * nH * np * (hd + 2) * sizeof(float);
}

int q4_paged_attn(const uint16_t* q, int ldq, const uint16_t* kc, const uint16_t* vc, int npages, int page,
                  const int32_t* prefix_pages, int max_prefix, const int32_t* prefix_len, const int32_t* table,
                  int table_ld, int nseq, int max_own, const int32_t* seq, const int32_t* pos, uint16_t* out, int ldo,
                  int T, int nH, int nkv, int hd, int window, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  Q4_ARG(q && kc && vc && table && seq && pos && out, "null pointer");
  Q4_ARG(hd == 64 || hd == 128 || hd == 256 || hd == 512, "paged attention takes head dims 64/128/256/512 (got %d)",
         hd);
  Q4_ARG(nH > 0 && nkv > 0 && nH % nkv == 0, "nH=%d must be a multiple of nkv=%d", nH, nkv);
  Q4_ARG(T > 0 && npages > 0 && nseq > 0 && table_ld > 0 && window >= 0, "bad sizes");
  const int lg = page_lg(page);
  Q4_ARG(lg > 0, "page=%d is not a power of two of 16..4096 rows", page);
  Q4_ARG(max_prefix >= 0 && (max_prefix == 0 || (prefix_pages && prefix_len)),
         "max_prefix=%d needs prefix_pages and prefix_len", max_prefix);
  Q4_ARG(max_own > 0 && max_own <= (long)table_ld * page, "max_own=%d must be in 1..table_ld * page = %ld", max_own,
         (long)table_ld * page);
  Q4_ARG((long)max_prefix + max_own < (1l << 30), "a context of %ld keys is too long", (long)max_prefix + max_own);
  Q4_ARG(ldq >= (long)nH * hd && ldo >= (long)nH * hd && ldq % 8 == 0 && ldo % 8 == 0,
         "row strides ldq=%d, ldo=%d must be multiples of 8 of at least nH * hd = %ld", ldq, ldo, (long)nH * hd);
  for (const void* p : {(const void*)q, (const void*)kc, (const void*)vc, (const void*)out})
    Q4_ARG(((uintptr_t)p & 15) == 0, "q, kc, vc and out must be 16-byte aligned");
  const size_t cache = (size_t)npages * nkv * page * hd * 2, nq = ((size_t)(T - 1) * ldq + (size_t)nH * hd) * 2,
               no = ((size_t)(T - 1) * ldo + (size_t)nH * hd) * 2;
  Q4_ARG(!overlap(q, nq, out, no), "out must not overlap q");
  Q4_ARG(!overlap(kc, cache, out, no) && !overlap(vc, cache, out, no), "out must not overlap the cache");
  const size_t need = q4_paged_attn_workspace_bytes(T, nH, nkv, hd, max_prefix, max_own, window);
  Q4_ARG(ws_bytes >= need && (need == 0 || (ws && ((uintptr_t)ws & 15) == 0)),
         "paged attention needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, ws_bytes);
  Q4_ARG(need == 0 || (!overlap(ws, need, q, nq) && !overlap(ws, need, out, no) && !overlap(ws, need, kc, cache) &&
                       !overlap(ws, need, vc, cache)),
         "the workspace must not overlap q, out or the cache");
  const Pages pg{prefix_pages, max_prefix ? prefix_len : nullptr, table, seq, pos, table_ld, nseq, npages, lg,
                 max_prefix, max_own};
  const PgPlan p = pg_plan(T, nH, nkv, hd, max_prefix, max_own, window);
  const PgArgs a{q, kc, vc, out, reinterpret_cast<float*>(ws), ldq, ldo, T, nH, nkv, nH / nkv, window, p.nsp, p.nso,
                 p.nsp + p.nso, p.nrb, p.nhb};
  const long grid = (long)p.nrb * nkv * p.nsp + (long)T * nkv * p.nhb * p.nso;
  Q4_ARG(grid < PG_MAX_BLOCKS / 2 && (long)T * nH < PG_MAX_BLOCKS, "a batch of %d rows of %d heads is too large", T, nH);
  hipStream_t st = as_stream(stream);
  const bool hl = nH / nkv <= 8;  // a group's heads leave room in 16 rows for their weights' second parts
#define PG_LAUNCH(HD, MODE) \
  const dim3 threads(PgTile<HD>::threads(MODE));                                                                   \
  if (hl) hipLaunchKernelGGL((paged_attn_kernel<HD, MODE, true>), dim3((unsigned)grid), threads, 0, st, a, pg); \
  else hipLaunchKernelGGL((paged_attn_kernel<HD, MODE, false>), dim3((unsigned)grid), threads, 0, st, a, pg)
#define PG_ATTN(HD)                                  \
  if (p.mode == PG_OWN) { PG_LAUNCH(HD, PG_OWN); }                    \
  else if (p.mode == PG_SHARED) { PG_LAUNCH(HD, PG_SHARED); }         \
  else if (p.mode == PG_SHARED_FEW) { PG_LAUNCH(HD, PG_SHARED_FEW); } \
  else { PG_LAUNCH(HD, PG_STREAM); }
#define PG_MERGE(HD) hipLaunchKernelGGL(paged_merge_kernel<HD>, dim3(T * nH), dim3(PG_THREADS), 0, st, a, pg)
  switch (hd) {
    case 64: PG_ATTN(64); break;
    case 128: PG_ATTN(128); break;
    case 256: PG_ATTN(256); break;
    default: PG_ATTN(512); break;
  }
  Q4_LAUNCHED("paged_attn");
  if (a.np == 1) return Q4_OK;
  switch (hd) {
    case 64: PG_MERGE(64); break;
    case 128: PG_MERGE(128); break;
    case 256: PG_MERGE(256); break;
    default: PG_MERGE(512); break;
  }
#undef PG_ATTN
#undef PG_LAUNCH
#undef PG_MERGE
  Q4_LAUNCHED("paged_merge");
  return Q4_OK;
}

}  // extern "C"
