// Attention of a tree of drafted tokens over the 3-bit KV cache (speculative
// decoding).  The T <= 64 drafts of a sequence are its last T positions; draft
// i sees every earlier position (the prefix, P = len - T of them) and the
// drafts that its mask names:
//     x[i, s] = scale * q[i] . k[s]   for s < P, or s >= P and bit s - P of mask[i]
//     out[i]  = sum_s softmax(x[i])_s v[s],   0 for a draft that sees nothing,
// with k, v = min + code * (max - min) / 7 as stored, and the GQA head map of
// the single-token decode.  q and out are fp32 or bf16.
//
// Mathematics.  Rows of one kv head are its T * G queries (row = draft * G +
// head in group).  A code c = 0..7 becomes the fp16 1 + c/8 by two bit
// operations (the code is its leading mantissa bits) or, one subtraction later,
// (c - 3.5)/8, exactly either way:
//     k = (min - 8 st) + 8 st (1 + c/8) = (min + 3.5 st) + 8 st (c - 3.5)/8,
// st = (max - min)/7, so q . k is a multiple of sum(q) plus 8 st times a product
// of fp16 matrices.  q enters as fp16 hi + lo of q * 2^sh (sh puts the row's
// absmax in [2^14, 2^15)): hi alone holds a bf16 q exactly down to 2^-29 of the
// absmax, hi + lo hold 22 bits of an fp32 q or of a rotated one (mode T), which is
// no bf16 value.  p . v likewise: w = p st as fp16 hi + lo, 22 bits.  (hi alone, 11
// bits, took 532 us where 64 drafts over 8 x 32768 positions now take 616, but one
// bf16 output in twenty came out a step off.)  The centred form keeps the products'
// sums near zero, where the two parts of v do not cancel; the scores of a bf16 q do
// without it.  (As
// fp16 subnormals the codes would cost one operation less, but the tensor core
// aligns a product by the operands' exponents and drops the low bits: 2^-12 of
// the result were lost.)  Softmax statistics, the sum terms and the merge of the
// splits are fp32; the tensor core's sums are fp32 that it truncates, see below.
// With mma.sync instead (16 rows a warp, the codes unpacked by every warp) 16
// drafts over 32768 positions took 86 us where this takes 47 (32 q and 8 kv heads,
// bf16), and 64 drafts over 8 x 32768 positions 1868 us where it takes 616.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "ft_kv3.cuh"
#include "ft_tc.cuh"

namespace ft {
namespace {

constexpr int kMaxDraft = 64;       // bits of a mask word
constexpr int kTWarps = 4;          // 32-slot blocks per tile
constexpr int kTStageBytes = kTWarps * kRecBytes;
constexpr int kTPart = 2 + kD;      // partial record: M, l, numerator[128]

struct TreeParams {
  const void* q;  // [B][T][Hq][128], fp32 or bf16
  int q_bf16;
  int64_t Hq, Hkv;
  int G, T, rows, rgroups;  // rows = T * G per kv head, in tiles of 128
  const uint64_t* mask;     // [B][T], or null: draft i sees drafts 0..i
  int64_t nbc, head_off, head_blk, len;
  int64_t nlb;        // logical 32-slot blocks covering the longest sequence
  int64_t tiles_per;  // 128-slot tiles per split
  float qk_log2;      // softmax scale * log2(e)
  const uint32_t* blocks;
  const float* signs;  // mode T rotation signs, or null
  float* part;         // [B][Hkv][rows][nsplit][kTPart]
  int* err;
  const int32_t* table;  // paged pool, as the single-token decode
  const int32_t* seq_lens;
  int64_t tstride, n_pages;
  int nparts;  // splits
  uint8_t* qimg;  // prepared row tiles [B][Hkv][rgroups]
};

// Codes of bytes (0, 2) (h = 0) or (1, 3) (h = 1) of quad Q of a triple, as two
// fp16 values 1 + c/8: the field moves to mantissa bits 7..9.
template <int kLeft>
__device__ __forceinline__ uint32_t shifted(uint32_t w) {
  return kLeft >= 0 ? w << (kLeft < 0 ? 0 : kLeft) : w >> (kLeft < 0 ? -kLeft : 0);
}
template <int Q, int h>
__device__ __forceinline__ uint32_t quad_half2(uint32_t w0, uint32_t w1, uint32_t w2) {
  constexpr uint32_t kOne = 0x3C003C00u;
  if (Q < 6) {
    const uint32_t w = Q < 2 ? w0 : (Q < 4 ? w1 : w2);
    return (shifted<7 - 3 * (Q & 1) - 8 * h>(w) & 0x03800380u) | kOne;
  }
  // low two bits from bits 6, 7 of word 0 or 1, the high one from bit Q of word 2
  const uint32_t lo = (shifted<1 - 8 * h>(Q == 6 ? w0 : w1) & 0x01800180u) | kOne;
  return (shifted<9 - Q - 8 * h>(w2) & 0x02000200u) | lo;
}
// the same centred: (c - 3.5) / 8
__device__ __forceinline__ uint32_t sub_half2(uint32_t a, uint32_t b) {
  uint32_t v;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
  return v;
}
template <int Q, int h>
__device__ __forceinline__ uint32_t quad_centred(uint32_t w0, uint32_t w1, uint32_t w2) {
  return sub_half2(quad_half2<Q, h>(w0, w1, w2), 0x3DC03DC0u);
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {  // a in the low half
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

__device__ __forceinline__ float ex2(float x) {  // 2 ulp, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Draft tokens of row R (0 <= R < rows): the mask bits of its draft.
__device__ __forceinline__ uint64_t row_mask(const uint64_t* mask, int64_t b, int T, int t) {
  const uint64_t all = T == 64 ? ~0ull : (1ull << T) - 1ull;
  return (mask ? mask[b * T + t] : (2ull << t) - 1ull) & all;
}

// 128-point Walsh-Hadamard transform of the warp's vector, 4 elements a lane.
__device__ __forceinline__ void warp_fwht128(float (&v)[4], int lane) {
  float a = v[0] + v[1], b = v[0] - v[1], c = v[2] + v[3], d = v[2] - v[3];
  v[0] = a + c;
  v[1] = b + d;
  v[2] = a - c;
  v[3] = b - d;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float u = __shfl_xor_sync(0xffffffffu, v[j], o);
      v[j] = (lane & o) ? u - v[j] : u + v[j];
    }
}

// Four elements of query row R (lane's), as stored.
__device__ __forceinline__ uint4 load_q_raw(const TreeParams& p, int64_t b, int64_t kvh, int R,
                                            int lane) {
  const int t = R / p.G;
  const int64_t h = kvh * p.G + (R - t * p.G);
  const int64_t at = ((b * p.T + t) * p.Hq + h) * kD + 4 * lane;
  if (p.q_bf16) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + at);
    return make_uint4(w.x << 16, w.x & 0xffff0000u, w.y << 16, w.y & 0xffff0000u);
  }
  return *reinterpret_cast<const uint4*>(static_cast<const float*>(p.q) + at);
}

// The row's values, rotated in mode T, and its sh.
__device__ __forceinline__ void q_row(const TreeParams& p, const uint4& raw, int lane,
                                      float (&v)[4], int* sh) {
  v[0] = __uint_as_float(raw.x);
  v[1] = __uint_as_float(raw.y);
  v[2] = __uint_as_float(raw.z);
  v[3] = __uint_as_float(raw.w);
  if (p.signs) {
    const float4 sg = reinterpret_cast<const float4*>(p.signs)[lane];
    v[0] *= sg.x;
    v[1] *= sg.y;
    v[2] *= sg.z;
    v[3] *= sg.w;
    warp_fwht128(v, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= 0.08838834764831845f;  // 1 / sqrt(128)
  }
  float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // amax * 2^sh in [2^14, 2^15); a non-finite row stays as it is and ends NaN
  const int e = (int)((__float_as_uint(amax) >> 23) & 255u);
  *sh = e == 255 ? 0 : min(14 + 127 - e, 120);
}

// exponent e with v < 2^e for a finite v >= 0, held in [-85, 128]
__device__ __forceinline__ int bound_exp(float v) {
  const int e = (int)(__float_as_uint(v) >> 23) - 126;
  return min(max(e, -85), 128);
}

// e of a position's value factors: vs < 2^e and |vc| < 2^(e + 85), so that with
// x - M + e <= 15 the weights stay below 2^15 and the terms of the sums below 2^100;
// an infinity or NaN bounds nothing.
__device__ __forceinline__ int value_exp(float vs, float vc) {
  const float v = fmaxf(vs, fabsf(vc) * 0x1p-85f);
  return bound_exp(v < INFINITY ? v : 0.0f);
}

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// v * 2^(2 h): references are even and lie up to 2^200 apart, beyond one factor's range
__device__ __forceinline__ float scale2(float v, float half_pow) { return v * half_pow * half_pow; }

// The tile kernel takes V as V * 2^-16, so that with the largest ranges (e = 112) exp2(x - M)
// is at least 2^-107 for the heaviest position, 2^19 above the smallest normal float;
// the combine kernel scales back.  (Values below 2^-110 lose low bits to it: 2^-133.)
constexpr float kValueScale = 0x1p-16f;

// ---------------------------------------------------------------- tiles --
// S = Q K' (128 query rows x 128 positions a tile), then O += P V', on the
// 5th-generation tensor core, K' and V' being the tile's codes as fp16.
//
// One CTA per SM, 28 warps.  A producer warp streams the records of a tile (4 of
// 3584 bytes) into raw buffers; four warps write the operand K' (1 + c/8) and four
// V' ((c - 3.5)/8), one record each, in the swizzled K-major layout; two warps
// compute each position's factors; one thread issues the MMAs; two groups of eight
// softmax warps (16 rows each) take the even and the odd tiles, each with its own S
// and O in TMEM and its own running statistics, and merge at the end.  P overwrites S.
// The waits of the chain S -> P -> O poll, all others suspend the warp: 64 drafts over
// 8 x 32768 positions take 616 us, 625 when these suspend it too.
// The K index of the first product is dims in the order 32 (Q/2) + 8r + 4 (Q%2)
// + (0 2 1 3)[b] of dim 16Q + 4r + b; positions run as 32 w + 8 (s%4) + 4 (s/4%2)
// + (0 2 1 3)[s/8] of slot s of record w; both so that a converter lane writes the
// 16 bytes it holds, and eight lanes of a store meet eight banks.
// References: even integer M per row with x - M + e <= 15 for the e of each position
// (value_exp), so that neither the sum terms overflow, those of constant vectors among
// them, nor w: w = exp2(x - M)(max - min)/7 stays below 2^15 in fp16; the largest x - M + e
// starts in (5, 7] and M moves only when one passes 15, by a power of two that the sums,
// the P columns already written and O in TMEM are then scaled by.  So the largest w of
// a row has at least 2^4, and a w at 2^-k of it is off by 2^-25 or 2^(k - 29) of itself,
// whatever the largest p belongs to (a sink with values near 0) and whatever ranges
// positions of little weight have.  A record's scores are compared with 15 minus the
// e of its largest range first; only where one passes that does each position's own e
// count.
// kTerms 1: bf16 queries (mode R), q as one fp16; 2: fp32 or rotated queries, hi and lo.
// P's hi and lo of a record take the columns of its scores.  O is summed in TMEM over
// the whole split, where the tensor core truncates, 2^-25 of O a product on average:
// 2^-14 after 2048 products, against 2^-9 of the bf16 output; for fp32 a split has at
// most 8 tiles (64 products a group: 2^-19 expected, 1e-6 as measured), the splits being
// merged in fp32.
constexpr int kPreRows = 128;
constexpr int kPreWarps = 28;
constexpr int kPreRaw = 3;
constexpr int kOperand = 128 * 128 * 2;  // bytes of Q, K' or V' (two swizzled panels)
// one term of q: Q, two K', two V'; two terms: Q hi and lo, two K', one V'
__host__ __device__ constexpr int off_k(int terms) { return terms * kOperand; }
__host__ __device__ constexpr int off_v(int terms) { return (terms + 2) * kOperand; }
constexpr int kPreOffRaw = 5 * kOperand;
constexpr int kPreOffFac = kPreOffRaw + kPreRaw * kTStageBytes;
constexpr int kFacBytes = 64 * 32 + 16;  // per position pair {st, st, kc, kc} {vst, vst, vc, vc}; e per record
constexpr int kPreOffQinfo = kPreOffFac + 4 * kFacBytes;  // [128] sum term, [128] factor
constexpr int kPreOffMask = kPreOffQinfo + kPreRows * 8;  // [128] draft bits
constexpr int kPreOffBars = kPreOffMask + kPreRows * 8;
// what tree_query_kernel prepares for a row tile: the operand as it lies in shared
// memory, then the row sums, factors and draft bits
__host__ __device__ constexpr int q_image(int terms) { return terms * kOperand + kPreRows * 16; }
static_assert(kPreOffMask == kPreOffQinfo + kPreRows * 8, "one copy brings both");
constexpr int kPreBars = 2 * kPreRaw + 5 * 2 + 2 * 4 + 2;
constexpr int kPreSmem = kPreOffBars + kPreBars * 8 + 16 + 1024;  // 1024: alignment
static_assert(kPreSmem <= 227 * 1024, "one CTA per SM");
constexpr int kMergeStride = kD + 4;  // floats per row of a merge area (conflict-free float4)
constexpr int kMergeArea = kPreRows * kMergeStride;
static_assert(2 * kMergeArea * 4 <= kPreOffRaw, "the merge uses the operand buffers");
static_assert(2 * kPreRows * 12 <= kPreRaw * kTStageBytes, "row statistics use the raw buffers");

__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
// Registers of a warpgroup from here on.  The seven groups' shares add up to the
// 896 x 72 that the block is launched with: 4 x 88, 2 x 56, 40 (x 128 threads).
template <int kRegs>
__device__ __forceinline__ void more_regs() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void fewer_regs() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Lane (row of the MMA) of query row i of a tile: the first 64 rows take 16 lanes
// in each quarter of the SM, so that fewer rows still use all four.
__device__ __forceinline__ int row_lane(int i) {
  return 32 * ((i >> 4) & 3) + 16 * (i >> 6) + (i & 15);
}

// With at most 64 rows (kDup) the row tile holds each row twice, as i and i + 64: the
// first takes the first two records of each tile, the second the others, so that all
// softmax warps work and each for half as long.  Their weights are 0 in the records
// that the other takes, their sums are merged like those of the two groups.  (5 drafts
// over 517 positions, 2 kv heads: 18.6 -> 16.6 us; 16 over 32768, 8 kv heads: 47.7 ->
// 46.7.  Without the rows' second copies half the softmax warps have nothing to do.)
__host__ __device__ constexpr bool twice(int rows) { return rows <= kPreRows / 2; }

// The query operand of tree_tile_kernel, 32 rows a CTA, four a warp: fp16 in the
// swizzled K-major layout, the rows' sums, factors and draft bits.  A kernel of
// its own: every split of the positions needs the same operand, and its code,
// fetched anew by each launch, took longer in the big kernel than here.
constexpr int kQueryRows = 32;
template <int kTerms>
__global__ void __launch_bounds__(256) tree_query_kernel(const __grid_constant__ TreeParams p) {
  tc::pdl_launch_dependents();  // the tile kernel may start to load the cache
  const int64_t tile = blockIdx.x / (kPreRows / kQueryRows);  // (row, row tile)
  const int64_t row = tile / p.rgroups, b = row / p.Hkv, kvh = row % p.Hkv;
  const int R0 = (int)(tile % p.rgroups) * kPreRows;
  const int i0 = (blockIdx.x % (kPreRows / kQueryRows)) * kQueryRows + (threadIdx.x >> 5) * 4;
  const int lane = threadIdx.x & 31;
  uint8_t* img = p.qimg + tile * (int64_t)q_image(kTerms);
  const int from = R0 + (twice(p.rows) ? i0 & 63 : i0);
  uint4 raw[4];
#pragma unroll
  for (int y = 0; y < 4; ++y)
    raw[y] = from + y < p.rows ? load_q_raw(p, b, kvh, from + y, lane) : make_uint4(0, 0, 0, 0);
  uint64_t mask = 0;
  if (lane < 4 && from + lane < p.rows) mask = row_mask(p.mask, b, p.T, (from + lane) / p.G);
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int i = i0 + y;
    float v[4];
    int sh;
    q_row(p, raw[y], lane, v, &sh);
    const float mul = pow2i(sh);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= mul;
    const uint32_t h0 = pack_half2(v[0], v[2]), h1 = pack_half2(v[1], v[3]);
    const float2 f0 = unpack_half2(h0), f1 = unpack_half2(h1);
    float sum = (f0.x + f0.y) + (f1.x + f1.y);  // of the q that the products take
    const int Q = lane >> 2, c = 4 * ((Q >> 1) & 1) + (lane & 3), at = row_lane(i);
    uint8_t* to = img + (Q >> 2) * (kOperand / 2) + at * 128 + ((c ^ (at & 7)) << 4) + (Q & 1) * 8;
    *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1);
    if (kTerms == 2) {
      const uint32_t l0 = pack_half2(v[0] - f0.x, v[2] - f0.y);
      const uint32_t l1 = pack_half2(v[1] - f1.x, v[3] - f1.y);
      const float2 d0 = unpack_half2(l0), d1 = unpack_half2(l1);
      sum += (d0.x + d0.y) + (d1.x + d1.y);
      *reinterpret_cast<uint2*>(to + kOperand) = make_uint2(l0, l1);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == y) {
      float* info = reinterpret_cast<float*>(img + kTerms * kOperand);
      info[at] = sum * ldexpf(p.qk_log2, -sh);
      info[kPreRows + at] = ldexpf(p.qk_log2, 3 - sh);
      reinterpret_cast<uint64_t*>(info + 2 * kPreRows)[at] = mask;
    }
  }
}

template <bool kValue>
struct Masked {
  static constexpr bool value = kValue;
};

template <int kTerms, bool kDup>
__global__ void __launch_bounds__(kPreWarps * 32, 1)
    tree_tile_kernel(const __grid_constant__ TreeParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = tc::smem_u32(smem);
  const uint32_t bars = sbase + kPreOffBars;
  const uint32_t raw_full = bars, raw_empty = raw_full + 8 * kPreRaw;
  const uint32_t k_full = raw_empty + 8 * kPreRaw, v_full = k_full + 16;
  const uint32_t qk_done = v_full + 16, pv_done = qk_done + 16, p_full = pv_done + 16;
  const uint32_t fac_full = p_full + 16, fac_empty = fac_full + 32;
  const uint32_t q_full = fac_empty + 32, fin = q_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kPreOffBars + kPreBars * 8);

  const int split = blockIdx.x;
  const int64_t kvh = blockIdx.y / p.rgroups;
  const int R0 = (int)(blockIdx.y % p.rgroups) * kPreRows;
  const int64_t b = blockIdx.z, row = b * p.Hkv + kvh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, r = lane & 3;
  int64_t len_b = p.len, nlb_b = p.nlb;
  if (p.table) {
    len_b = p.seq_lens[b];
    if (len_b < 0 || len_b > p.len) {
      if (tid == 0) atomicCAS(p.err, 0, 1007);
      len_b = len_b < 0 ? 0 : p.len;
    }
    nlb_b = (len_b + kBlk - 1) / kBlk;
  }
  const int64_t t_all = (nlb_b + kTWarps - 1) / kTWarps, t_begin = (int64_t)split * p.tiles_per;
  const int64_t t_end = t_begin + p.tiles_per < t_all ? t_begin + p.tiles_per : t_all;
  const int n = t_end > t_begin ? (int)(t_end - t_begin) : 0;
  const int nrows = p.rows - R0 < kPreRows ? p.rows - R0 : kPreRows;
  float* part = p.part + ((row * p.rows + R0) * p.nparts + split) * kTPart;
  if (n == 0) {  // a shorter sequence of the batch: an empty partial
    for (int i = tid; i < nrows; i += blockDim.x) {
      part[(int64_t)i * p.nparts * kTPart] = -INFINITY;
      part[(int64_t)i * p.nparts * kTPart + 1] = 0.0f;
    }
    tc::pdl_wait();  // this grid never ends before the query kernel
    return;
  }

  if (tid == 0) {
    for (int s = 0; s < kPreRaw; ++s) {
      tc::mbar_init(raw_full + 8 * s, 1);
      tc::mbar_init(raw_empty + 8 * s, 10);  // K', V' and factor warps
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(k_full + 8 * s, 4);
      tc::mbar_init(v_full + 8 * s, 4);
      tc::mbar_init(qk_done + 8 * s, 1);
      tc::mbar_init(pv_done + 8 * s, 1);
      tc::mbar_init(p_full + 8 * s, 8);
    }
    for (int s = 0; s < 4; ++s) {
      tc::mbar_init(fac_full + 8 * s, 2);
      tc::mbar_init(fac_empty + 8 * s, 8);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(fin, 1);
    tc::fence_barrier_init();
  }
  if (warp == 25) tc::tmem_alloc(tc::smem_u32(tmem_slot), 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tO = tmem + 256;  // S (and P) 2 x 128 columns, O 2 x 128

  if (warp >= 24) {
    fewer_regs<40>();
    if (warp == 24) {
      // ---------------------------------------------------- producer warp --
      if (lane == 0) {
        bool ok = true;
        int issued = 0;
        int64_t pb = (p.head_blk + t_begin * kTWarps) % p.nbc;
        for (int j = 0; j < n && ok; ++j) {
          if (j == (n < kPreRaw ? n - 1 : kPreRaw - 1)) {
            // the first records are on their way; the queries come from the
            // kernel before this one
            tc::pdl_wait();
            const uint8_t* img =
                p.qimg + (row * p.rgroups + R0 / kPreRows) * (int64_t)q_image(kTerms);
            tc::mbar_arrive_expect_tx(q_full, q_image(kTerms));
            tc::bulk_g2s(sbase, img, kTerms * kOperand, q_full);
            tc::bulk_g2s(sbase + kPreOffQinfo, img + kTerms * kOperand, kPreRows * 16, q_full);
          }
          const int s = j % kPreRaw;
          if (j >= kPreRaw)
            ok = tc::mbar_wait_sleep(raw_empty + 8 * s, ((j / kPreRaw) - 1) & 1, p.err, 51);
          if (!ok) break;
          const int64_t jb = (t_begin + j) * kTWarps;
          const int nb = nlb_b - jb < kTWarps ? (int)(nlb_b - jb) : kTWarps;
          tc::mbar_arrive_expect_tx(raw_full + 8 * s, nb * kRecBytes);
          const uint32_t dst = sbase + kPreOffRaw + s * kTStageBytes;
          if (p.table) {
            for (int i = 0; i < nb; ++i) {  // a bad table entry reads page 0 and is reported
              const int64_t pg =
                  checked_page(p.table, b * p.tstride + jb + i, p.n_pages, p.err, 1008);
              tc::bulk_g2s(dst + i * kRecBytes,
                           p.blocks + ((pg < 0 ? 0 : pg) * p.Hkv + kvh) * kRecWords, kRecBytes,
                           raw_full + 8 * s);
            }
          } else {
            // nb consecutive records from physical block pb, wrapping at most once
            const int n1 = pb + nb <= p.nbc ? nb : (int)(p.nbc - pb);
            tc::bulk_g2s(dst, p.blocks + (row * p.nbc + pb) * kRecWords, n1 * kRecBytes,
                         raw_full + 8 * s);
            if (n1 < nb)
              tc::bulk_g2s(dst + n1 * kRecBytes, p.blocks + row * p.nbc * kRecWords,
                           (nb - n1) * kRecBytes, raw_full + 8 * s);
            pb += nb;
            if (pb >= p.nbc) pb -= p.nbc;
          }
          ++issued;
        }
        // the copies in flight must land before the CTA may exit
        for (int j = issued - kPreRaw < 0 ? 0 : issued - kPreRaw; j < issued; ++j)
          tc::mbar_wait_sleep(raw_full + 8 * (j % kPreRaw), (j / kPreRaw) & 1, p.err, 52);
        tc::mbar_wait_sleep(q_full, 0, p.err, 52);
      }
    } else if (warp == 25) {
      // --------------------------------------------------------- MMA warp --
      // the warp stays together; one elected lane issues
      constexpr uint32_t idesc = tc::idesc_f16(128, 128);
      uint32_t leader;
      bool ok = tc::mbar_wait_sleep(q_full, 0, p.err, 50);
      const uint64_t qd = tc::smem_desc_sw128(sbase);
      auto qk = [&](int j) {
        const int s = j & 1;
        ok = tc::mbar_wait(k_full + 8 * s, (j >> 1) & 1, p.err, 53);
        if (!ok) return;
        tc::tc_fence_after();
        const uint64_t kd = tc::smem_desc_sw128(sbase + off_k(kTerms) + s * kOperand);
        if (tc::elect_one(leader)) {
#pragma unroll
          for (int k = 0; k < 8 * kTerms; ++k) {  // hi, then lo
            const uint64_t at = (uint64_t)(((k >> 2) & 1) * (kOperand / 2) + (k & 3) * 32) >> 4;
            tc::mma_f16_ss(tS + 128 * s, qd + at + (uint64_t)(k >> 3) * (kOperand >> 4), kd + at,
                           idesc, k > 0);
          }
          tc::mma_commit(qk_done + 8 * s);
        }
        __syncwarp();
      };
      auto pv = [&](int j) {
        const int s = j & 1;
        ok = tc::mbar_wait(p_full + 8 * s, (j >> 1) & 1, p.err, 54) &&
             (kTerms == 1 ? tc::mbar_wait(v_full + 8 * s, (j >> 1) & 1, p.err, 55)
                          : tc::mbar_wait(v_full, j & 1, p.err, 55));
        if (!ok) return;
        tc::tc_fence_after();
        const uint64_t vd =
            tc::smem_desc_sw128(sbase + off_v(kTerms) + (kTerms == 1 ? s * kOperand : 0));
        if (tc::elect_one(leader)) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t at = (uint64_t)((k >> 2) * (kOperand / 2) + (k & 3) * 32) >> 4;
            // P of 16 positions: 8 columns; a record's hi and lo lie in the 32 columns of
            // its scores
            const uint32_t pc = tS + 128 * s + 32 * (k >> 1) + 8 * (k & 1);
            tc::mma_f16_ts(tO + 128 * s, pc, vd + at, idesc, j >= 2 || k > 0);
            tc::mma_f16_ts(tO + 128 * s, pc + 16, vd + at, idesc, 1);
          }
          tc::mma_commit(pv_done + 8 * s);
        }
        __syncwarp();
      };
      // the MMAs of one thread run in order, so P of tile j is read before the
      // scores of tile j + 2 replace it
      if (ok) qk(0);
      if (ok && n > 1) qk(1);
      for (int j = 0; j < n && ok; ++j) {
        pv(j);
        if (ok && j + 2 < n) qk(j + 2);
      }
      if (tc::elect_one(leader)) tc::mma_commit(fin);  // then nothing is in flight
      __syncwarp();
      tc::mbar_wait_sleep(fin, 0, p.err, 56);
    } else {
      // ----------------------------------------------------- factor warps --
      // scores are st x product + kc x sum(q) (K' is 1 + c/8, or centred), values
      // vst x product + vc x sum(p) (as (c - 3.5)/8)
      const int half = warp - 26;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        ok = tc::mbar_wait_sleep(raw_full + 8 * (j % kPreRaw), (j / kPreRaw) & 1, p.err, 57);
        if (ok && j >= 4) ok = tc::mbar_wait_sleep(fac_empty + 8 * (j & 3), ((j >> 2) - 1) & 1, p.err, 58);
        if (!ok) break;
        float* fac = reinterpret_cast<float*>(smem + kPreOffFac + (j & 3) * kFacBytes);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int w = 2 * half + i;
          const uint32_t* rec = reinterpret_cast<const uint32_t*>(
              smem + kPreOffRaw + (j % kPreRaw) * kTStageBytes + w * kRecBytes);
          const float2 km = reinterpret_cast<const float2*>(rec + kRecKmm)[mm_index(lane)];
          const float2 vm = reinterpret_cast<const float2*>(rec + kRecVmm)[mm_index(lane)];
          const float ks = (km.y - km.x) * 0.14285714285714285f;
          const float vs = (vm.y - vm.x) * 0.14285714285714285f * kValueScale;
          const int oe = lane >> 3;
          const int col = 32 * w + 8 * (lane & 3) + 4 * ((lane >> 2) & 1) +
                          (oe == 1 ? 2 : (oe == 2 ? 1 : oe));
          float* fp = fac + (col >> 1) * 8 + (col & 1);
          fp[0] = ks;
          fp[2] = fmaf(kTerms == 1 ? -8.0f : 3.5f, ks, km.x);
          const float vc = fmaf(3.5f, vs, vm.x * kValueScale);
          fp[4] = vs;
          fp[6] = vc;
          const int e = __reduce_max_sync(0xffffffffu, value_exp(vs, vc));
          if (lane == 0) reinterpret_cast<int*>(fac + 64 * 8)[w] = e;
        }
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(fac_full + 8 * (j & 3));
          tc::mbar_arrive(raw_empty + 8 * (j % kPreRaw));
        }
      }
    }
  } else if (warp >= 16) {
    // -------------------------------------------------- K' and V' warps --
    // Four warps each, one record a warp.  The words go to registers first, so that
    // the raw buffer is free for the tile after next while the operand's is awaited.
    fewer_regs<56>();
    const bool isv = warp >= 20;
    const int w = warp & 3;
    const int gk = ((g & 1) << 2) | (g >> 1);
    const uint32_t full = isv ? v_full : k_full, done = isv ? pv_done : qk_done;
    // K: the words of lane 4 gk + r, so that eight lanes of a store meet eight banks
    const int words = w * kRecWords + (isv ? kRecV + lane * 12 : (4 * gk + r) * 12);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = tc::mbar_wait_sleep(raw_full + 8 * (j % kPreRaw), (j / kPreRaw) & 1, p.err, 59);
      if (!ok) break;
      const uint4* src = reinterpret_cast<const uint4*>(
          reinterpret_cast<const uint32_t*>(smem + kPreOffRaw + (j % kPreRaw) * kTStageBytes) + words);
      uint32_t wd[12];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const uint4 x = src[i];
        wd[4 * i] = x.x, wd[4 * i + 1] = x.y, wd[4 * i + 2] = x.z, wd[4 * i + 3] = x.w;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(raw_empty + 8 * (j % kPreRaw));
      // the operand's buffer: K' j - 2 multiplied, V' j - 2, or j - 1 where there is one
      if (kTerms == 2 && isv) {
        if (j >= 1) ok = tc::mbar_wait_sleep(done + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1, p.err, 60);
      } else if (j >= 2) {
        ok = tc::mbar_wait_sleep(done + 8 * (j & 1), ((j >> 1) - 1) & 1, p.err, 60);
      }
      if (!ok) break;
      if (isv) {
        // triple m: dim 8 (4m + J) + g is row 8 (4m + J) + gk; chunk 4 (w % 2) + r of panel w / 2
        uint8_t* at = smem + off_v(kTerms) + (kTerms == 1 ? (j & 1) * kOperand : 0) +
                      (w >> 1) * (kOperand / 2) + gk * 128 + (((4 * (w & 1) + r) ^ gk) << 4);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint32_t w0 = wd[3 * m], w1 = wd[3 * m + 1], w2 = wd[3 * m + 2];
#define FT_PRE_V(J)                                                                                 \
  *reinterpret_cast<uint4*>(at + (4 * m + (J)) * 1024) =                                             \
      make_uint4(quad_centred<2 * (J), 0>(w0, w1, w2), quad_centred<2 * (J), 1>(w0, w1, w2),         \
                 quad_centred<2 * (J) + 1, 0>(w0, w1, w2), quad_centred<2 * (J) + 1, 1>(w0, w1, w2));
          FT_PRE_V(0) FT_PRE_V(1) FT_PRE_V(2) FT_PRE_V(3)
#undef FT_PRE_V
        }
      } else {
        // slot gk + 8e is row 32w + 8 (gk % 4) + 4 (gk / 4) + (0 2 1 3)[e]; quads 2J, 2J + 1 go to
        // chunk 4 (J % 2) + r of panel J / 2
        uint8_t* op = smem + off_k(kTerms) + (j & 1) * kOperand + (32 * w + 8 * (gk & 3)) * 128;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w0 = wd[3 * e], w1 = wd[3 * e + 1], w2 = wd[3 * e + 2];
          const int sub = 4 * (gk >> 2) + ((e & 1) << 1 | e >> 1);
          uint8_t* a0 = op + sub * 128 + ((r ^ sub) << 4);
          uint8_t* a1 = op + sub * 128 + (((r + 4) ^ sub) << 4);
#define FT_PRE_K(J, AT)                                                                  \
  *reinterpret_cast<uint4*>(AT) =                                                         \
      kTerms == 1                                                                         \
          ? make_uint4(quad_half2<2 * (J), 0>(w0, w1, w2), quad_half2<2 * (J), 1>(w0, w1, w2), \
                       quad_half2<2 * (J) + 1, 0>(w0, w1, w2),                            \
                       quad_half2<2 * (J) + 1, 1>(w0, w1, w2))                            \
          : make_uint4(quad_centred<2 * (J), 0>(w0, w1, w2),                              \
                       quad_centred<2 * (J), 1>(w0, w1, w2),                              \
                       quad_centred<2 * (J) + 1, 0>(w0, w1, w2),                          \
                       quad_centred<2 * (J) + 1, 1>(w0, w1, w2));
          FT_PRE_K(0, a0) FT_PRE_K(1, a1) FT_PRE_K(2, a0 + kOperand / 2) FT_PRE_K(3, a1 + kOperand / 2)
#undef FT_PRE_K
        }
      }
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full + (kTerms == 2 && isv ? 0 : 8 * (j & 1)));
    }
  } else {
    // ------------------------------------------------------- softmax warps --
    more_regs<88>();
    const float* qinfo = reinterpret_cast<const float*>(smem + kPreOffQinfo);
    const uint64_t* qmask = reinterpret_cast<const uint64_t*>(smem + kPreOffMask);
    bool ok = tc::mbar_wait_sleep(q_full, 0, p.err, 67);
    // warp: tiles st, st + 2, ..; lanes 32 quad + 16 half + {g, g + 8} (see row_lane)
    const int st = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3;
    const uint32_t lanes = (uint32_t)(32 * quad + 16 * half) << 16;
    const int row0 = 32 * quad + 16 * half + g;
    const bool live = (kDup ? 0 : 64 * half) + 16 * quad < nrows;  // this warp's rows exist
    const int c0 = kDup ? 2 * half : 0, c1 = kDup ? c0 + 2 : 4;    // its records of a tile
    // 32-bit slot arithmetic: the host keeps len below 2^31 - 512
    const int hoff = p.table ? 0 : (int)p.head_off, len32 = (int)len_b;
    const int P = len32 - p.T;  // prefix length; negative: the first drafts do not exist
    uint64_t qsum[2], qfac[2], l2[2], vm2[2], negM[2];
    bool unset = true;  // a row has no reference yet (warp-uniform)
    uint32_t have = 0;  // bit i: row i has one
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = qinfo[row0 + 8 * i], f = qinfo[kPreRows + row0 + 8 * i];
      qsum[i] = pair(a, a);
      qfac[i] = pair(f, f);
      l2[i] = vm2[i] = negM[i] = pair(0.0f, 0.0f);
    }
    // One tile: P of this warp's rows.  Two instances: with kMasked each score is
    // tested against the mask (the tiles at the sequence's ends), so that the
    // prefix's loop stays small.
    auto tile = [&](auto masked, int j) {
      constexpr bool kMasked = decltype(masked)::value;
      const uint32_t ts = tS + 128 * st + lanes;
      const float* fac = reinterpret_cast<const float*>(smem + kPreOffFac + (j & 3) * kFacBytes);
      uint32_t sv[16];
      tc::tmem_ld_16x256b_x4(ts + 32 * c0, sv);
#pragma unroll 1
      for (int c = c0; c < c1; ++c) {
        // 32 positions (a record); x[k][i]: row i, positions 8k + 2r, + 1
        const float4* f4 = reinterpret_cast<const float4*>(fac) + (16 * c + r) * 2;
        const float eb = (float)(15 - reinterpret_cast<const int*>(fac + 64 * 8)[c]);
        uint64_t x[4][2];
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 kf = f4[8 * k];
          const uint64_t ks = pair(kf.x, kf.y), kc = pair(kf.z, kf.w);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint64_t s2 = pair(__uint_as_float(sv[4 * k + 2 * i]),
                                     __uint_as_float(sv[4 * k + 2 * i + 1]));
            x[k][i] = fma2(ks, mul2(s2, qfac[i]), fma2(kc, qsum[i], negM[i]));
          }
        }
        if (c + 1 < c1) tc::tmem_ld_16x256b_x4(ts + 32 * (c + 1), sv);  // the next record's scores
        if (kMasked) {
          // position 8k + 2r + o of the record is slot k + 4 (r / 2) + 8 (r % 2) + 16 o
          const int base = ((int)(t_begin + j) * kTWarps + c) * kBlk - hoff;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint64_t mask = qmask[row0 + 8 * i];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = unpair(x[k][i]);
              const int p0 = base + k + 4 * (r >> 1) + 8 * (r & 1), p1 = p0 + 16;
              const bool s0 = p0 >= 0 && p0 < len32 && (p0 < P || ((mask >> (p0 - P)) & 1ull));
              const bool s1 = p1 >= 0 && p1 < len32 && (p1 < P || ((mask >> (p1 - P)) & 1ull));
              x[k][i] = pair(s0 ? f.x : -INFINITY, s1 ? f.y : -INFINITY);
            }
          }
        }
        bool above = unset;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = unpair(x[k][i]);
            t[k] = fmaxf(f.x, f.y);
          }
          above |= fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) > eb;
        }
        if (__builtin_expect(__any_sync(0xffffffffu, above), 0)) {
          // a score that may be above its row's bound, or a row's first: each position's
          // own e decides (masked places have x = -infinity)
          float top[2] = {-INFINITY, -INFINITY}, alpha[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 vf = f4[8 * k + 1];
            const float e0 = (float)value_exp(vf.x, vf.z), e1 = (float)value_exp(vf.y, vf.w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 f = unpair(x[k][i]);
              top[i] = fmaxf(top[i], fmaxf(f.x + e0, f.y + e1));
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            const bool first = !((have >> i) & 1u);
            // x - M + e so far; up by the even number that puts its maximum at 7 at most
            float up = first || top[i] > 15.0f ? 2.0f * ceilf(0.5f * top[i] - 3.5f) : 0.0f;
            // nothing seen yet, or NaN or infinite scores (the row then ends NaN)
            if (!(fabsf(up) < 1e30f)) up = 0.0f;
            else if (first) have |= 1u << i;
            // half of the factor's exponent; nothing is summed before the first
            alpha[i] = first ? 1.0f : exp2f(-0.5f * up);
            const uint64_t a2 = pair(alpha[i], alpha[i]), u2 = pair(-up, -up);
            negM[i] = add2(negM[i], u2);
            l2[i] = mul2(mul2(l2[i], a2), a2);
            vm2[i] = mul2(mul2(vm2[i], a2), a2);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k][i] = add2(x[k][i], u2);
          }
          unset = __any_sync(0xffffffffu, have != 3u);
          if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
            tc::tmem_wait_ld();
            tc::tmem_wait_st();
#pragma unroll 1
            for (int k = 2 * c0; k < 2 * c; ++k) {
              // P columns of this tile, 16 positions: hi + lo, scaled in fp32 (alpha as
              // fp16 would be 0 below 2^-25, where the weights still count) and split anew
              const uint32_t at = ts + 32 * (k >> 1) + 8 * (k & 1);
              uint32_t h[4], l[4];
              tc::tmem_ld_16x256b_x1(at, h);
              tc::tmem_ld_16x256b_x1(at + 16, l);
              tc::tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float2 a = unpack_half2(h[q]), b = unpack_half2(l[q]);
                const float u = scale2(a.x + b.x, alpha[q >> 1]), v = scale2(a.y + b.y, alpha[q >> 1]);
                h[q] = pack_half2(u, v);
                const float2 hi = unpack_half2(h[q]);
                l[q] = pack_half2(u - hi.x, v - hi.y);
              }
              tc::tmem_st_16x256b_x1(at, h);
              tc::tmem_st_16x256b_x1(at + 16, l);
            }
            if (j >= 2) {  // O, once the product of tile j - 2 is in it
              ok = ok && tc::mbar_wait_sleep(pv_done + 8 * st, ((j >> 1) - 1) & 1, p.err, 65);
              tc::tc_fence_after();
#pragma unroll 1
              for (int k = 0; ok && k < 8; ++k) {
                uint32_t t[8];
                tc::tmem_ld_16x256b_x2(tO + 128 * st + lanes + 16 * k, t);
                tc::tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  t[q] = __float_as_uint(scale2(__uint_as_float(t[q]), alpha[(q >> 1) & 1]));
                tc::tmem_st_16x256b_x2(tO + 128 * st + lanes + 16 * k, t);
              }
            }
            tc::tmem_wait_st();
          }
        }
        uint32_t pw[8], pl[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 vf = f4[8 * k + 1];
          const uint64_t vs = pair(vf.x, vf.y), vc = pair(vf.z, vf.w);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = unpair(x[k][i]);
            const uint64_t pr = pair(ex2(f.x), ex2(f.y));
            l2[i] = add2(l2[i], pr);
            float2 wt = unpair(mul2(pr, vs));
            if (!kMasked) {
              vm2[i] = fma2(pr, vc, vm2[i]);
            } else {  // whatever V holds in masked places
              float2 vt = unpair(mul2(pr, vc));
              if (f.x == -INFINITY) wt.x = vt.x = 0.0f;
              if (f.y == -INFINITY) wt.y = vt.y = 0.0f;
              vm2[i] = add2(vm2[i], pair(vt.x, vt.y));
            }
            pw[2 * k + i] = pack_half2(wt.x, wt.y);
            const float2 hi = unpack_half2(pw[2 * k + i]);
            pl[2 * k + i] = pack_half2(wt.x - hi.x, wt.y - hi.y);
          }
        }
        tc::tmem_st_16x128b_x4(ts + 32 * c, pw);
        tc::tmem_st_16x128b_x4(ts + 32 * c + 16, pl);
      }
      if (kDup) {  // nothing of the records that the row's other copy takes
        const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) tc::tmem_st_16x128b_x4(ts + 32 * (2 - c0) + 16 * k, zero);
      }
      tc::tmem_wait_st();
    };
    for (int j = st; j < n; j += 2) {
      ok = ok && tc::mbar_wait(fac_full + 8 * (j & 3), (j >> 2) & 1, p.err, 63) &&
           tc::mbar_wait(qk_done + 8 * st, (j >> 1) & 1, p.err, 64);
      if (!ok) break;
      tc::tc_fence_after();
      if (live) {
        const int base = (int)(t_begin + j) * (kTWarps * kBlk) - hoff;
        if (base < 0 || base + kTWarps * kBlk > P) tile(Masked<true>(), j);
        else tile(Masked<false>(), j);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(p_full + 8 * st);
        tc::mbar_arrive(fac_empty + 8 * (j & 3));
      }
    }
    // ---- the two groups merge: row statistics in the raw buffers, numerators in
    // the operand buffers (every product is done)
    if (ok) ok = tc::mbar_wait_sleep(fin, 0, p.err, 66);
    tc::tc_fence_after();
    float* stats = reinterpret_cast<float*>(smem + kPreOffRaw);  // [group][row]: M, l, sum term
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 lf = unpair(l2[i]), vf = unpair(vm2[i]);
      float l = lf.x + lf.y, v = vf.x + vf.y;
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, x);
        v += __shfl_xor_sync(0xffffffffu, v, x);
      }
      if (r == 0) {
        float* t = stats + (st * kPreRows + row0 + 8 * i) * 3;
        t[0] = l == 0.0f ? -INFINITY : -unpair(negM[i]).x;  // l == 0: the group saw nothing
        t[1] = l;
        t[2] = v;
      }
    }
    asm volatile("bar.sync 1, 512;" ::: "memory");
    const int myrow = 32 * quad + lane;  // here a warp takes 32 rows and half the dims
    if (16 * quad < nrows) {
      const float* mine = stats + (st * kPreRows + myrow) * 3;
      float Mx = fmaxf(stats[myrow * 3], stats[(kPreRows + myrow) * 3]);
      if (kDup) Mx = fmaxf(Mx, __shfl_xor_sync(0xffffffffu, Mx, 16));
      const bool some = st < n && mine[0] != -INFINITY;
      const float f = some ? exp2f(0.5f * (mine[0] - Mx)) : 0.0f, vterm = mine[2];
      float* arow = reinterpret_cast<float*>(smem) + st * kMergeArea + myrow * kMergeStride;
#pragma unroll 1
      for (int k = 4 * half; k < 4 * half + 4; ++k) {
        uint32_t t[16];
        tc::tmem_ld_x16(tO + 128 * st + ((uint32_t)(32 * quad) << 16) + 16 * k, t);
        tc::tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // column 8t' + 4 (d % 2) + d / 2 holds dim 8t' + d
          float o[8];
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const float v = __uint_as_float(t[8 * h + (d & 1) * 4 + (d >> 1)]);
            o[d] = some ? scale2(fmaf(8.0f, v, vterm), f) : 0.0f;
          }
          float4* dst = reinterpret_cast<float4*>(arow + 16 * k + 8 * h);
          dst[0] = make_float4(o[0], o[1], o[2], o[3]);
          dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
      }
    }
    tc::tc_fence_before();
    asm volatile("bar.sync 1, 512;" ::: "memory");
    // partial records, one warp a row
    for (int i = warp; i < nrows; i += 16) {
      const int at = row_lane(i);
      const int last = at + (kDup ? 16 : 0);  // row_lane(i + 64): its other copy
      float mx = -INFINITY, l = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int y = at; y <= last; y += 16)
        mx = fmaxf(mx, fmaxf(stats[y * 3], stats[(kPreRows + y) * 3]));
      for (int y = at; y <= last; y += 16)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float* t = stats + (x * kPreRows + y) * 3;
          if (t[0] != -INFINITY) l += scale2(t[1], exp2f(0.5f * (t[0] - mx)));
          const float4 w =
              reinterpret_cast<const float4*>(smem)[(x * kMergeArea + y * kMergeStride) / 4 + lane];
          v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
        }
      float* pp = part + (int64_t)i * p.nparts * kTPart;
      if (lane == 0) *reinterpret_cast<float2*>(pp) = make_float2(mx, l);
      float2* pn = reinterpret_cast<float2*>(pp + 2) + 2 * lane;
      pn[0] = make_float2(v.x, v.y);
      pn[1] = make_float2(v.z, v.w);
    }
  }
  __syncthreads();
  if (warp == 25) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Merges the split partials of a row: one CTA a row, its warps share the splits
// (so that more loads are in flight at once: with one warp the decode of 16 drafts
// over 32768 positions takes 51.2 us, so 46.7), 4 dims a lane; mode T: the output is rotated back.
constexpr int kCombineWarps = 4;
__global__ void __launch_bounds__(32 * kCombineWarps)
    tree_combine_kernel(const __grid_constant__ TreeParams p, void* __restrict__ out) {
  __shared__ float sm[kCombineWarps][2 + kD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nsplit = p.nparts;
  const int64_t R = blockIdx.x;
  const float* pp = p.part + R * nsplit * kTPart;
  tc::pdl_wait();  // the tiles' partials
  float M = -INFINITY, l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = warp; s < nsplit; s += kCombineWarps) {
    const float* ps = pp + (int64_t)s * kTPart;
    const float2 ml = *reinterpret_cast<const float2*>(ps);
    const float2 a = reinterpret_cast<const float2*>(ps + 2)[2 * lane];
    const float2 c = reinterpret_cast<const float2*>(ps + 2)[2 * lane + 1];
    if (ml.x == -INFINITY) continue;
    const float Mn = fmaxf(M, ml.x);
    const float f0 = exp2f(0.5f * (M - Mn)), f = exp2f(0.5f * (ml.x - Mn));  // M = -inf at first: 0
    M = Mn;
    l = scale2(ml.y, f) + scale2(l, f0);
    v[0] = scale2(a.x, f) + scale2(v[0], f0);
    v[1] = scale2(a.y, f) + scale2(v[1], f0);
    v[2] = scale2(c.x, f) + scale2(v[2], f0);
    v[3] = scale2(c.y, f) + scale2(v[3], f0);
  }
  if (lane == 0) {
    sm[warp][0] = M;
    sm[warp][1] = l;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) sm[warp][2 + 32 * k + lane] = v[k];
  __syncthreads();
  if (warp != 0) return;
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) M = fmaxf(M, sm[w][0]);
  l = v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) {
    if (sm[w][0] == -INFINITY) continue;
    const float f = exp2f(0.5f * (sm[w][0] - M));
    l += scale2(sm[w][1], f);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += scale2(sm[w][2 + 32 * k + lane], f);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)  // l = 0: the row saw nothing
    v[k] = l == 0.0f ? 0.0f : v[k] / l * (1.0f / kValueScale);
  if (p.signs) {
    warp_fwht128(v, lane);
    const float4 sg = reinterpret_cast<const float4*>(p.signs)[lane];
    v[0] *= 0.08838834764831845f * sg.x;
    v[1] *= 0.08838834764831845f * sg.y;
    v[2] *= 0.08838834764831845f * sg.z;
    v[3] *= 0.08838834764831845f * sg.w;
  }
  // row (b, kvh, t, head in group) -> out [b][t][kvh * G + head]
  const int64_t bk = R / p.rows;
  const int i = (int)(R % p.rows), t = i / p.G;
  const int64_t b = bk / p.Hkv, h = (bk % p.Hkv) * p.G + (i - t * p.G);
  const int64_t at = ((b * p.T + t) * p.Hq + h) * kD + 4 * lane;
  if (p.q_bf16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v[0], v[1]), y = __floats2bfloat162_rn(v[2], v[3]);
    uint2 w;
    w.x = *reinterpret_cast<const uint32_t*>(&x);
    w.y = *reinterpret_cast<const uint32_t*>(&y);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = w;
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) =
        make_float4(v[0], v[1], v[2], v[3]);
  }
}

// Opts the kernels into their dynamic shared memory, once per device.
void tree_opt_in(int device) {
  static bool done[64] = {false};
  if (device >= 0 && device < 64 && done[device]) return;
  for (auto kernel : {tree_tile_kernel<1, false>, tree_tile_kernel<1, true>,
                      tree_tile_kernel<2, false>, tree_tile_kernel<2, true>})
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPreSmem);
  if (device >= 0 && device < 64) done[device] = true;
}

// Tiles per split, at most `most`: fewest waves of `resident` CTAs x (tiles + a CTA's
// own cost, which is about three tiles' time: counted as 1 or 6 of them, 64 drafts over
// 8 x 32768 positions take 616 or 627 us, as 3 they take 616, all measured in one run).
// `rows` row tiles a sequence; `all` tiles of the batch's sequences together, of which
// the longest has ntiles.  Unequal sequences: CTAs that would start behind a sequence's
// end return at once and are not counted (each sequence's last split is taken as half
// full), and where more CTAs work than are resident the time is their work evenly
// shared and a quarter of a split.  24 drafts over 6 sequences of 2006 to 8191
// positions, 4 kv heads: 70 us, 78 with splits for equal lengths; 64 drafts over 8
// sequences of 500 to 11469, 8 kv heads: 179 and 257 (half a split: 188, an eighth: 200);
// over 24 of 200 to 29352: 475 and 468 (486, 465), the one where others are better.
constexpr int64_t kPreOverhead = 3;
constexpr int64_t kTailParts = 4;  // of a split
constexpr int64_t kTermTiles = 8;  // fp32 queries: most tiles of a split
int64_t split_tiles(int64_t batch, int64_t rows, int64_t ntiles, int64_t all, int64_t resident,
                    int64_t most) {
  int64_t best_cost = INT64_MAX, best = most < ntiles ? most : ntiles;
  for (int64_t sp = ceil_div(ntiles, best); sp <= 256 && sp <= ntiles; ++sp) {
    const int64_t per = ceil_div(ntiles, sp);
    const int64_t one = per + kPreOverhead;
    const bool equal = all == batch * ntiles;
    const int64_t splits = equal ? batch * ceil_div(ntiles, per)
                                 : ceil_div(2 * all + batch * (per - 1), 2 * per);
    const int64_t cost = equal || rows * splits <= resident
                             ? kTailParts * ceil_div(rows * splits, resident) * one
                             : kTailParts * rows * (all + splits * kPreOverhead) / resident + one;
    if (cost < best_cost) {
      best_cost = cost;
      best = per;
    }
  }
  return best;
}

// Launch that may start before the kernel in front of it has ended; the kernel
// waits for that one itself (griddepcontrol).
template <class Kernel, class... Args>
int launch_early(Kernel kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FT_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  FT_LAUNCH_CHECK();
  return FT_OK;
}

template <class Cache>
int launch_tree(ft_ctx* ctx, Cache* c, TreeParams p, int64_t batch, int64_t total_len,
                int64_t n_draft,
                const void* q_dev, int q_is_bf16, int64_t q_heads, const uint64_t* mask_dev,
                float scale, void* out_dev, cudaStream_t s) {
  FT_CHECK(q_heads > 0 && q_heads % c->kv_heads == 0, FT_ERR_SHAPE,
           "q_heads (%lld) must be a multiple of kv_heads (%lld)", (long long)q_heads,
           (long long)c->kv_heads);
  FT_CHECK(n_draft > 0, FT_ERR_SHAPE, "no drafts");
  FT_CHECK(n_draft <= kMaxDraft, FT_ERR_UNSUPPORTED, "%lld drafts: at most %d are supported",
           (long long)n_draft, kMaxDraft);
  FT_CHECK(q_heads / c->kv_heads <= 4096, FT_ERR_UNSUPPORTED, "too many q heads per kv head");
  FT_CHECK(((uintptr_t)q_dev | (uintptr_t)out_dev) % 16 == 0, FT_ERR_SHAPE,
           "q and out must be 16-byte aligned");
  p.q = q_dev;
  p.q_bf16 = q_is_bf16 ? 1 : 0;
  p.Hq = q_heads;
  p.Hkv = c->kv_heads;
  p.G = (int)(q_heads / c->kv_heads);
  p.T = (int)n_draft;
  p.rows = p.T * p.G;
  p.mask = mask_dev;
  p.nlb = (p.head_off + p.len + kBlk - 1) / kBlk;
  const float sc = scale > 0.0f ? scale : 1.0f / sqrtf((float)kD);
  p.qk_log2 = sc * 1.4426950408889634f;
  p.blocks = c->blocks;
  p.signs = c->signs;
  p.err = ctx->err_word;
  const int64_t total = batch * p.Hkv * p.rows;
  const int64_t ntiles = ceil_div(p.nlb, (int64_t)kTWarps);
  tree_opt_in(ctx->device);
  const int terms = q_is_bf16 && !p.signs ? 1 : 2;  // a rotated bf16 q is no bf16 value
  p.rgroups = (p.rows + kPreRows - 1) / kPreRows;
  FT_CHECK(p.Hkv * p.rgroups <= 65535 && batch <= 65535, FT_ERR_UNSUPPORTED,
           "decode grid too large");
  const int64_t tiles = batch * p.Hkv * p.rgroups;
  int64_t all = batch * ntiles;
  if (total_len > 0 && total_len < batch * p.len)
    all = std::min(all, ceil_div(total_len + batch * (kTWarps * kBlk / 2), kTWarps * kBlk));
  p.tiles_per = split_tiles(batch, p.Hkv * p.rgroups, ntiles, all, ctx->num_sms,
                            q_is_bf16 ? INT64_MAX : kTermTiles);
  p.nparts = (int)ceil_div(ntiles, p.tiles_per);
  const size_t images = (size_t)tiles * q_image(terms);
  FT_CHECK(total < INT32_MAX && tiles < INT32_MAX / 4, FT_ERR_UNSUPPORTED, "too many query rows");
  int rc = ensure_ws(c->tree, images + (size_t)(total * p.nparts * kTPart) * 4, s, "tree decode",
                     c->retired);
  if (rc != FT_OK) return rc;
  p.qimg = static_cast<uint8_t*>(c->tree.ptr);
  p.part = reinterpret_cast<float*>(p.qimg + images);
  const unsigned qgrid = (unsigned)(tiles * (kPreRows / kQueryRows));
  if (terms == 1)
    tree_query_kernel<1><<<qgrid, 256, 0, s>>>(p);
  else
    tree_query_kernel<2><<<qgrid, 256, 0, s>>>(p);
  FT_LAUNCH_CHECK();
  const dim3 grid((unsigned)p.nparts, (unsigned)(p.Hkv * p.rgroups), (unsigned)batch);
  const auto kernel = twice(p.rows)
                          ? (terms == 1 ? tree_tile_kernel<1, true> : tree_tile_kernel<2, true>)
                          : (terms == 1 ? tree_tile_kernel<1, false> : tree_tile_kernel<2, false>);
  rc = launch_early(kernel, grid, kPreWarps * 32, kPreSmem, s, p);
  if (rc != FT_OK) return rc;
  return launch_early(tree_combine_kernel, dim3((unsigned)total), 32 * kCombineWarps, 0, s, p,
                      out_dev);
}

}  // namespace
}  // namespace ft

using namespace ft;

extern "C" {

int ft_kv3_tree_decode(ft_ctx* ctx, ft_kv3* c, int64_t n_draft, const void* q_dev, int q_is_bf16,
                       int64_t q_heads, const uint64_t* mask_dev, float scale, void* out_dev,
                       void* stream) {
  FT_CHECK(ctx && c && q_dev && out_dev, FT_ERR_SHAPE, "null argument");
  FT_CHECK(n_draft <= c->len, FT_ERR_SHAPE, "%lld drafts in a cache of %lld positions",
           (long long)n_draft, (long long)c->len);
  FT_CHECK(c->len < (int64_t)INT32_MAX - 512, FT_ERR_UNSUPPORTED,
           "cache too long for the decode's 32-bit slot arithmetic");
  DeviceScope scope(c->device);
  TreeParams p{};
  p.nbc = c->cap / kBlk;
  p.head_off = c->head % kBlk;
  p.head_blk = c->head / kBlk;
  p.len = c->len;
  return launch_tree(ctx, c, p, c->batch, 0, n_draft, q_dev, q_is_bf16, q_heads, mask_dev, scale,
                     out_dev, static_cast<cudaStream_t>(stream));
}

int ft_kvp_tree_decode(ft_ctx* ctx, ft_kvp* c, int64_t batch, const int32_t* tables_dev,
                       int64_t table_stride, const int32_t* seq_lens_dev, int64_t max_seq_len,
                       int64_t total_len, int64_t n_draft, const void* q_dev, int q_is_bf16,
                       int64_t q_heads, const uint64_t* mask_dev, float scale, void* out_dev,
                       void* stream) {
  FT_CHECK(ctx && c && tables_dev && seq_lens_dev && q_dev && out_dev, FT_ERR_SHAPE,
           "null argument");
  FT_CHECK(batch > 0 && max_seq_len > 0 && total_len >= 0 && table_stride > 0 &&
               max_seq_len <= table_stride * kBlk,
           FT_ERR_SHAPE, "bad decode shape (batch %lld, max_seq_len %lld, table stride %lld)",
           (long long)batch, (long long)max_seq_len, (long long)table_stride);
  FT_CHECK(max_seq_len < (int64_t)INT32_MAX - 512, FT_ERR_UNSUPPORTED,
           "sequence too long for the decode's 32-bit slot arithmetic");
  DeviceScope scope(c->device);
  TreeParams p{};
  p.nbc = 1;
  p.len = max_seq_len;
  p.table = tables_dev;
  p.seq_lens = seq_lens_dev;
  p.tstride = table_stride;
  p.n_pages = c->n_pages;
  return launch_tree(ctx, c, p, batch, total_len, n_draft, q_dev, q_is_bf16, q_heads, mask_dev, scale,
                     out_dev, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
