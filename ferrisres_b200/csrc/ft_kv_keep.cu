// Eviction from the 3-bit KV cache by accumulated attention weight, and the
// compaction that moves the positions that stay.
//
// select_heavy, per (sequence, kv head): of the len positions the n_recent last
// and the n_keep - n_recent heaviest of the others stay, listed in ascending
// order; equal weights go to the lowest position, -0 equals 0 and NaN is
// heavier than everything.  A sequence of at most n_keep positions stays whole.
//
// keep, per (sequence, kv head): position start + i := position idx[i], in
// place, for i < count.  Any list with idx[i] >= start + i is allowed
// (ascending lists are), so a position is never overwritten before a later one
// reads it as long as lower positions are written no earlier than higher ones
// are still to be read: see keep_kernel.
#include <cooperative_groups.h>

#include "ft_kv3.cuh"
#include "ft_tc.cuh"

namespace cg = cooperative_groups;

namespace ft {
namespace {

// ---------------------------------------------------------------- select --
struct SelectParams {
  const float* w;      // [B][H] rows of wstride floats
  float* w_out;        // [B][H] rows of wout_stride floats, or null
  int32_t* idx;        // [B][H][n_keep]
  const int32_t* lens;  // [B], or null: every sequence holds len
  int64_t H, wstride, wout_stride;
  int64_t len, n_keep, n_recent, out_len;
  int* err;
};

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelBins = 2048;
static_assert(kSelBins == 2 * kSelThreads && kSelWarps == 32, "two bins a thread, a warp sum a lane");
constexpr int kSelKeys = 40960;  // keys held in shared memory; further ones are read again
constexpr int kSelSmem = kSelBins * 4 + 4 * 64 * 4;

// Order-preserving key of a weight: larger key = heavier.
__device__ __forceinline__ uint32_t weight_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 -> +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One cluster per (sequence, kv head); each CTA takes a contiguous share of
// the candidates.  Radix selection of the n-th largest key (11 + 11 + 10 bits,
// histograms summed over the cluster through distributed shared memory), then
// one ordered pass that ranks the kept positions.
__global__ void __launch_bounds__(kSelThreads)
    select_kernel(const __grid_constant__ SelectParams p, int cap) {
  extern __shared__ uint32_t ssm[];
  uint32_t* hist = ssm;              // this CTA's histogram
  uint32_t* red = ssm + kSelBins;    // [64] warp sums
  uint32_t* bc = red + 64;           // broadcast values and per-CTA counts
  uint32_t* keys = bc + 192;         // [cap]
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  auto meet = [&]() {  // a cluster of one needs no cluster barrier
    if (C > 1) cl.sync();
    else __syncthreads();
  };
  const int64_t row = blockIdx.x / C;
  const int64_t b = row / p.H;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int64_t len = p.len;
  if (p.lens) {
    len = p.lens[b];
    if (len < 0 || len > p.len) {
      if (tid == 0) atomicCAS(p.err, 0, 1009);
      len = len < 0 ? 0 : p.len;
    }
  }
  const float* w = p.w + row * p.wstride;
  float* wo = p.w_out ? p.w_out + row * p.wout_stride : nullptr;
  int32_t* idx = p.idx + row * p.n_keep;
  const int64_t kept = len < p.n_keep ? len : p.n_keep;
  const int64_t gt0 = (int64_t)rank * kSelThreads + tid, gstep = (int64_t)C * kSelThreads;
  // entries past the kept positions: no index, no weight
  for (int64_t i = kept + gt0; i < p.n_keep; i += gstep) idx[i] = -1;
  if (wo)
    for (int64_t i = kept + gt0; i < p.out_len; i += gstep) wo[i] = 0.0f;
  if (len <= p.n_keep) {  // uniform over the cluster
    for (int64_t i = gt0; i < len; i += gstep) {
      idx[i] = (int32_t)i;
      if (wo) wo[i] = w[i];
    }
    return;
  }
  const int64_t cand = len - p.n_recent, heavy = p.n_keep - p.n_recent;  // 0 <= heavy < cand
  for (int64_t i = gt0; i < p.n_recent; i += gstep) {
    idx[heavy + i] = (int32_t)(cand + i);
    if (wo) wo[heavy + i] = w[cand + i];
  }
  if (heavy == 0) return;
  const int64_t share = (cand + C - 1) / C;
  const int64_t lo = share * rank < cand ? share * rank : cand;
  const int n = (int)((lo + share < cand ? lo + share : cand) - lo);
  const float* wl = w + lo;
  for (int i = tid; i < n && i < cap; i += kSelThreads) keys[i] = weight_key(wl[i]);
  auto key_at = [&](int i) { return i < cap ? keys[i] : weight_key(wl[i]); };

  uint32_t prefix = 0, pmask = 0;
  uint32_t need = (uint32_t)heavy;  // still to be found among keys with this prefix
#pragma unroll 1  // small code: a launch fetches every instruction anew
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t bmask = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t k = key_at(i);
      if ((k & pmask) == prefix) atomicAdd(&hist[(k >> shift) & bmask], 1u);
    }
    meet();
    // thread t owns bins 2t, 2t + 1 of the cluster's histogram
    uint32_t own[2] = {0, 0}, sum = 0;
    for (int c = 0; c < C; ++c) {
      const uint2 v = *reinterpret_cast<const uint2*>(cl.map_shared_rank(hist, c) + 2 * tid);
      own[0] += v.x;
      own[1] += v.y;
    }
    sum = own[0] + own[1];
    // keys in bins above: suffix sums over the threads
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_down_sync(0xffffffffu, inc, o);
      if (lane + o < 32) inc += u;
    }
    if (lane == 0) red[warp] = inc;
    __syncthreads();
    const uint32_t above = inc - sum + __reduce_add_sync(0xffffffffu, lane > warp ? red[lane] : 0u);
    if (above < need && need <= above + sum) {  // exactly one thread
      const bool low = above + own[1] < need;
      bc[0] = (uint32_t)(2 * tid + (low ? 0 : 1));
      bc[1] = need - above - (low ? own[1] : 0u);
    }
    meet();  // also: every CTA has read the histograms before they are cleared
    prefix |= bc[0] << shift;
    pmask |= bmask << shift;
    need = bc[1];
  }
  // prefix: the key of the lightest kept position; `need` positions that equal
  // it stay.  Each warp takes a contiguous span of the CTA's share.
  const int span = (n + kSelWarps - 1) / kSelWarps;
  const int s0 = warp * span < n ? warp * span : n, s1 = s0 + span < n ? s0 + span : n;
  uint32_t gt = 0, eq = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const uint32_t k = key_at(i);
    gt += k > prefix;
    eq += k == prefix;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) {
    red[warp] = gt;
    red[32 + warp] = eq;
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, red[lane]);
    const uint32_t e = __reduce_add_sync(0xffffffffu, red[32 + lane]);
    if (lane == 0) {
      bc[2] = a;
      bc[3] = e;
    }
  }
  meet();
  uint32_t gt_before = 0, eq_before = 0;
  for (int c = 0; c < rank; ++c) {
    gt_before += cl.map_shared_rank(bc, c)[2];
    eq_before += cl.map_shared_rank(bc, c)[3];
  }
  gt_before += __reduce_add_sync(0xffffffffu, lane < warp ? red[lane] : 0u);
  eq_before += __reduce_add_sync(0xffffffffu, lane < warp ? red[32 + lane] : 0u);
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < s1 ? key_at(i) : 0u;
    const bool g = i < s1 && k > prefix, e = i < s1 && k == prefix;
    const uint32_t bg = __ballot_sync(0xffffffffu, g), be = __ballot_sync(0xffffffffu, e);
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t er = eq_before + __popc(be & below);
    if (g || (e && er < need)) {
      const uint32_t at = gt_before + __popc(bg & below) + (er < need ? er : need);
      idx[at] = (int32_t)(lo + i);
      if (wo) wo[at] = wl[i];
    }
    gt_before += __popc(bg);
    eq_before += __popc(be);
  }
  meet();  // no CTA leaves while another reads its counts
}

// ------------------------------------------------------------------ keep --
struct KeepParams {
  int64_t H, nbc, head_off, head_blk, len;
  uint32_t* blocks;
  const int32_t* idx;  // idx[b * ib + h * ih + i]
  int64_t ib, ih;
  int64_t start, count;        // ring; paged: count = the longest list
  const int32_t* starts;       // paged: per sequence
  const int32_t* counts;
  const int32_t* seq_lens;
  const int32_t* table;
  int64_t tstride, n_pages;
  int* err;
};

constexpr int kKeepWarps = 8;
constexpr int kKeepSpan = 11;  // source records a CTA stages in shared memory, twice
constexpr int kKeepSmem = (2 * kKeepSpan + kKeepWarps) * kRecBytes;

// One cluster per (sequence, kv head).  Rounds of (CTAs x warps) destination
// blocks in ascending order: every warp assembles one block in shared memory, the
// cluster meets at a barrier, then the blocks are written by bulk copies.  A round
// reads positions at or above its own first one and writes none above its last, so
// what a later round reads is still in place and what this round reads is read
// before the barrier.
// The sources of a CTA's 256 positions span few blocks when most positions stay:
// up to kKeepSpan records come in by one bulk copy, each read once, while the round
// before is assembled; a wider span is gathered from global memory.  (16384 of 17408
// positions of 128 rows: 133 us; all gathers from global memory 171 us, staged without
// the overlap 180.)
// Gathering one slot: its K codes are 4 triples (one a lane r, copied as they
// are); its V codes are one byte lane of three words in each of 8 lanes and 4
// triples, 6 bits of 8 x 3, which move to the byte and the half (a) of the
// destination slot.
__global__ void __launch_bounds__(32 * kKeepWarps, 2)
    keep_kernel(const __grid_constant__ KeepParams p) {
  extern __shared__ __align__(128) uint32_t assembled[];
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks();
  const int64_t row = blockIdx.x / C;
  const int64_t b = row / p.H, h = row % p.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, r = lane & 3;
  int64_t start = p.start, count = p.count, len = p.len;
  if (p.table) {
    start = p.starts[b];
    count = p.counts[b];
    len = p.seq_lens[b];
    // every length is bounded by the table, so that no page index leaves it
    if (len < 0 || len > p.len || start < 0 || count < 0 || count > p.count ||
        start + count > len) {
      if (threadIdx.x == 0) atomicCAS(p.err, 0, 1010);
      count = 0;
    }
  }
  if (count == 0) return;  // uniform over the cluster
  const int32_t* idx = p.idx + b * p.ib + h * p.ih;
  const int64_t off = p.table ? 0 : p.head_off;
  // record of logical block lb (positions off-shifted), null for a bad page
  auto record = [&](int64_t lb) -> uint32_t* {
    if (p.table) {
      const int64_t pg = checked_page(p.table, b * p.tstride + lb, p.n_pages, p.err, 1011);
      return pg < 0 ? nullptr : p.blocks + (pg * p.H + h) * kRecWords;
    }
    int64_t pb = p.head_blk + lb;
    if (pb >= p.nbc) pb -= p.nbc;
    return p.blocks + (row * p.nbc + pb) * kRecWords;
  };
  const int blk0 = (int)((start + off) / kBlk);
  const int blk1 = (int)((start + count + off + kBlk - 1) / kBlk);
  const int per = C * kKeepWarps;
  const int me = (int)cl.block_rank() * kKeepWarps + warp;
  uint32_t* buf = assembled + warp * kRecWords;
  __shared__ int span[2][2][kKeepWarps];
  __shared__ uint64_t bar[2];
  if (threadIdx.x == 0) {
    tc::mbar_init(tc::smem_u32(&bar[0]), 1);
    tc::mbar_init(tc::smem_u32(&bar[1]), 1);
    tc::fence_barrier_init();
  }
  // the list's entry for slot `lane` of block lb, or that position itself
  auto entry = [&](int lb) -> int {
    const int64_t pos = (int64_t)lb * kBlk + lane - off;
    return pos >= start && pos < start + count ? idx[pos - start] : (int)pos;
  };
  // Lane u's source for slot u of block lb (itself where the list does not reach),
  // and the span of the warp's sources.
  auto look = [&](int lb, int s, int at) -> int {
    const int pos = lb * kBlk + lane - (int)off;
    int src = pos;
    if (lb < blk1 && s != pos) {
      if (s >= pos && s < len) src = s;
      else atomicCAS(p.err, 0, 1012);  // would overwrite or leave the cache: skipped
    }
    const int sblk = (int)((src + off) / kBlk);
    const int lo = __reduce_min_sync(0xffffffffu, src != pos ? sblk : INT32_MAX);
    const int hi = __reduce_max_sync(0xffffffffu, src != pos ? sblk : -1);
    if (lane == 0) {
      span[at][0][warp] = lo;
      span[at][1][warp] = hi;
    }
    return src;
  };
  // Issues the copy of a round's sources, if they are few enough; its first block,
  // or -1.  Every thread gets the same answer.
  auto stage = [&](int at) -> int {
    const int lo = __reduce_min_sync(0xffffffffu, span[at][0][lane % kKeepWarps]);
    const int hi = __reduce_max_sync(0xffffffffu, span[at][1][lane % kKeepWarps]);
    if (hi < 0 || hi - lo >= kKeepSpan) return -1;
    if (threadIdx.x == 0) {
      const uint32_t full = tc::smem_u32(&bar[at]);
      tc::mbar_arrive_expect_tx(full, (hi - lo + 1) * kRecBytes);
      for (int i = lo; i <= hi; ++i) {
        const uint32_t* rec = record(i);
        // a bad page is reported, and none of its slots is taken from here
        tc::bulk_g2s(tc::smem_u32(assembled + (kKeepWarps + at * kKeepSpan + i - lo) * kRecWords),
                     rec ? rec : p.blocks, kRecBytes, full);
      }
    }
    return lo;
  };
  int src = look(blk0 + me, entry(blk0 + me), 0);
  int ahead = entry(blk0 + per + me);  // entries of the round after
  __syncthreads();
  int lo = stage(0), at = 0;
  uint32_t phases = 0;  // bit `at`: parity of the next wait on bar[at]
  for (int first = blk0; first < blk1; first += per) {
    const int lb = first + me;
    // the next round's sources are read while this one is assembled: they lie above
    // all that this round writes
    const int src_next = look(lb + per, ahead, at ^ 1);
    ahead = entry(lb + 2 * per);
    // the copy of the round before has read this warp's block
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncthreads();
    const int lo_next = first + per < blk1 ? stage(at ^ 1) : -1;
    bool staged = lo >= 0;
    if (staged) {
      staged = tc::mbar_wait(tc::smem_u32(&bar[at]), (phases >> at) & 1u, p.err, 70);
      phases ^= 1u << at;
    }
    const int pos = lb * kBlk + lane - (int)off;
    const bool moved = src != pos;
    uint32_t* home = lb < blk1 ? record(lb) : nullptr;
    const bool write = __any_sync(0xffffffffu, moved) && home != nullptr;
    if (write) {
      const int sblk = (int)((src + off) / kBlk);
      const uint32_t* mine = home;
      if (moved) {
        mine = record(sblk);
        if (mine && staged)
          mine = assembled + (kKeepWarps + at * kKeepSpan + sblk - lo) * kRecWords;
      }
      const bool bad = mine == nullptr;
      if (bad) mine = home;  // reported; the slot keeps what it holds
      const int slot = bad ? lane : (int)((src + off) % kBlk);
      const unsigned long long base = (unsigned long long)mine;
      reinterpret_cast<float2*>(buf + kRecKmm)[mm_index(lane)] =
          reinterpret_cast<const float2*>(mine + kRecKmm)[mm_index(slot)];
      reinterpret_cast<float2*>(buf + kRecVmm)[mm_index(lane)] =
          reinterpret_cast<const float2*>(mine + kRecVmm)[mm_index(slot)];
      // K: lane (g, r) assembles the triples of slots g + 8e
      uint4* k4 = reinterpret_cast<uint4*>(buf + lane * 12);
      uint32_t kd[12];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t* rec = (const uint32_t*)__shfl_sync(0xffffffffu, base, g + 8 * e);
        const int t = __shfl_sync(0xffffffffu, slot, g + 8 * e);
        const uint32_t* k = rec + (4 * (t & 7) + r) * 12 + 3 * (t >> 3);
#pragma unroll
        for (int y = 0; y < 3; ++y) kd[3 * e + y] = k[y];
      }
#pragma unroll
      for (int y = 0; y < 3; ++y)
        k4[y] = make_uint4(kd[4 * y], kd[4 * y + 1], kd[4 * y + 2], kd[4 * y + 3]);
      // V: lane (g, r) assembles slots u = r + 4a + 8bb, byte bb of its words, from
      // lane 4g + t % 4 of the source's record.  Positions that keep their distance
      // share that lane, so its 48 bytes are loaded when they change.
      // The work is done on the four triples m at once: z[w][bb] holds word w's byte
      // of triple m in byte m, and is transposed at the end.
      uint32_t x[12], z[3][4];
      unsigned long long have = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int a = q & 1, bb = q >> 1, u = r + 4 * q;
        const unsigned long long rb = __shfl_sync(0xffffffffu, base, u);
        const int t = __shfl_sync(0xffffffffu, slot, u);
        const unsigned long long from = rb + 4 * (kRecV + (4 * g + (t & 3)) * 12);
        if (from != have) {
          have = from;
          const uint4* v4 = reinterpret_cast<const uint4*>(from);
#pragma unroll
          for (int y = 0; y < 3; ++y) {
            const uint4 v = v4[y];
            x[4 * y] = v.x;
            x[4 * y + 1] = v.y;
            x[4 * y + 2] = v.z;
            x[4 * y + 3] = v.w;
          }
        }
        // byte t / 8 of word w of each triple; half a of a triple (quads 2j + a) is bits
        // 0-2 (a = 0) or 3-5 (a = 1) of each byte, plus bits 6-7 of byte 0 or 1 and bit 6
        // or 7 of byte 2
        const int sa = (t >> 2) & 1;
        const uint32_t sel = (uint32_t)(t >> 3) * 0x11u + 0x40u;
        uint32_t y[3];
#pragma unroll
        for (int w = 0; w < 3; ++w)
          y[w] = __byte_perm(__byte_perm(x[w], x[3 + w], sel), __byte_perm(x[6 + w], x[9 + w], sel),
                             0x5410);
        const uint32_t lo2 = ((sa ? y[1] : y[0]) >> 6) & 0x03030303u;
        const uint32_t hi1 = (y[2] >> (6 + sa)) & 0x01010101u;
        const uint32_t c0 = (y[0] >> (3 * sa)) & 0x07070707u;
        const uint32_t c1 = (y[1] >> (3 * sa)) & 0x07070707u;
        const uint32_t c2 = (y[2] >> (3 * sa)) & 0x07070707u;
        if (a == 0) {
          z[0][bb] = c0 | lo2 << 6;
          z[1][bb] = c1;
          z[2][bb] = c2 | hi1 << 6;
        } else {
          z[0][bb] |= c0 << 3;
          z[1][bb] |= c1 << 3 | lo2 << 6;
          z[2][bb] |= c2 << 3 | hi1 << 7;
        }
      }
      uint32_t vd[12];
#pragma unroll
      for (int w = 0; w < 3; ++w) {  // 4 x 4 bytes: (bb, m) to (m, bb)
        const uint32_t p01l = __byte_perm(z[w][0], z[w][1], 0x5140);
        const uint32_t p01h = __byte_perm(z[w][0], z[w][1], 0x7362);
        const uint32_t p23l = __byte_perm(z[w][2], z[w][3], 0x5140);
        const uint32_t p23h = __byte_perm(z[w][2], z[w][3], 0x7362);
        vd[w] = __byte_perm(p01l, p23l, 0x5410);
        vd[3 + w] = __byte_perm(p01l, p23l, 0x7632);
        vd[6 + w] = __byte_perm(p01h, p23h, 0x5410);
        vd[9 + w] = __byte_perm(p01h, p23h, 0x7632);
      }
      uint4* v4 = reinterpret_cast<uint4*>(buf + kRecV + lane * 12);
#pragma unroll
      for (int y = 0; y < 3; ++y)
        v4[y] = make_uint4(vd[4 * y], vd[4 * y + 1], vd[4 * y + 2], vd[4 * y + 3]);
    }
    tc::fence_async_smem();
    if (C > 1) cl.sync();
    else __syncthreads();
    if (write && lane == 0) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(home),
                   "r"(tc::smem_u32(buf)), "r"(kRecBytes)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    src = src_next;
    lo = lo_next;
    at ^= 1;
  }
  // the last copies are done before the CTA's shared memory goes
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// CTAs of a cluster (at most 8) for `rows` rows of `units` units of work, each CTA
// taking `per` units at a time: as many as are resident at once, none without work.
int cluster_size(int resident, int64_t rows, int64_t units, int64_t per) {
  int64_t c = resident / rows;
  if (c > ceil_div(units, per)) c = ceil_div(units, per);
  return c < 1 ? 1 : (c > 8 ? 8 : (int)c);
}

template <class Kernel, class... Args>
int launch_cluster(Kernel kernel, int64_t rows, int cluster, int threads, size_t smem,
                   cudaStream_t s, Args... args) {
  FT_CHECK(rows * cluster < INT32_MAX, FT_ERR_UNSUPPORTED, "too many (sequence, head) rows");
  if (cluster == 1) {  // a plain launch is a cluster of one, and cheaper
    kernel<<<(unsigned)rows, threads, smem, s>>>(args...);
    FT_LAUNCH_CHECK();
    return FT_OK;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FT_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  FT_LAUNCH_CHECK();
  return FT_OK;
}

int launch_keep(ft_ctx* ctx, const KeepParams& p, int64_t rows, cudaStream_t s) {
  const int64_t blocks = ceil_div(p.count, kBlk) + 1;
  const int c = cluster_size(2 * ctx->num_sms, rows, blocks, kKeepWarps);
  static bool opted[64] = {false};  // once per device
  if (ctx->device >= 64 || !opted[ctx->device]) {
    FT_CUDA(cudaFuncSetAttribute(keep_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kKeepSmem));
    if (ctx->device < 64) opted[ctx->device] = true;
  }
  return launch_cluster(keep_kernel, rows, c, 32 * kKeepWarps, kKeepSmem, s, p);
}

}  // namespace
}  // namespace ft

using namespace ft;

extern "C" {

int ft_kv_select_heavy(ft_ctx* ctx, int64_t batch, int64_t kv_heads, const float* weights_dev,
                       int64_t weights_stride, const int32_t* seq_lens_dev, int64_t max_seq_len,
                       int64_t n_keep, int64_t n_recent, int32_t* idx_dev, float* weights_out_dev,
                       int64_t weights_out_stride, void* stream) {
  FT_CHECK(ctx && weights_dev && idx_dev, FT_ERR_SHAPE, "null argument");
  FT_CHECK(batch >= 0 && kv_heads > 0 && max_seq_len >= 0 && max_seq_len < INT32_MAX,
           FT_ERR_SHAPE, "bad selection shape (batch %lld, %lld kv heads, %lld positions)",
           (long long)batch, (long long)kv_heads, (long long)max_seq_len);
  FT_CHECK(n_keep > 0 && n_recent >= 0 && n_recent <= n_keep && n_keep < INT32_MAX, FT_ERR_SHAPE,
           "n_recent (%lld) must lie in [0, n_keep = %lld]", (long long)n_recent,
           (long long)n_keep);
  FT_CHECK(weights_stride >= max_seq_len, FT_ERR_SHAPE,
           "weight rows of %lld entries do not hold %lld positions", (long long)weights_stride,
           (long long)max_seq_len);
  const int64_t kept = max_seq_len < n_keep ? max_seq_len : n_keep;
  FT_CHECK(!weights_out_dev || weights_out_stride >= kept, FT_ERR_SHAPE,
           "weight rows of %lld entries do not hold %lld kept positions",
           (long long)weights_out_stride, (long long)kept);
  if (batch == 0) return FT_OK;
  if (weights_out_dev) {
    // the last row is read up to its last position, not to the pitch
    const int64_t rows = batch * kv_heads;
    const uintptr_t a = (uintptr_t)weights_dev, o = (uintptr_t)weights_out_dev;
    FT_CHECK(o + (size_t)(rows * weights_out_stride) * 4 <= a ||
                 a + (size_t)((rows - 1) * weights_stride + max_seq_len) * 4 <= o,
             FT_ERR_SHAPE, "weights_out must not overlap weights");
  }
  DeviceScope scope(ctx->device);
  SelectParams p{};
  p.w = weights_dev;
  p.w_out = weights_out_dev;
  p.idx = idx_dev;
  p.lens = seq_lens_dev;
  p.H = kv_heads;
  p.wstride = weights_stride;
  p.wout_stride = weights_out_stride;
  p.len = max_seq_len;
  p.n_keep = n_keep;
  p.n_recent = n_recent;
  p.out_len = weights_out_stride;
  p.err = ctx->err_word;
  const int64_t rows = batch * kv_heads;
  // one CTA a row up to 32 keys a thread: the cluster's barriers cost more than they
  // save (16384 keys a row, 128 rows: 50 us on clusters of four, 22.5 so)
  const int c = cluster_size(ctx->num_sms, rows, max_seq_len, 32 * kSelThreads);
  // keys that do not fit shared memory are read from global memory again
  const int64_t share = ceil_div(max_seq_len, c);
  const int cap = (int)(share < kSelKeys ? share : kSelKeys);
  const size_t smem = kSelSmem + (size_t)cap * 4;
  static bool opted[64] = {false};  // once per device
  if (ctx->device >= 64 || !opted[ctx->device]) {
    FT_CUDA(cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kSelSmem + kSelKeys * 4));
    if (ctx->device < 64) opted[ctx->device] = true;
  }
  return launch_cluster(select_kernel, rows, c, kSelThreads, smem,
                        static_cast<cudaStream_t>(stream), p, cap);
}

int ft_kv3_keep(ft_ctx* ctx, ft_kv3* c, int64_t start, int64_t count, const int32_t* idx_dev,
                int64_t idx_batch_stride, int64_t idx_head_stride, void* stream) {
  FT_CHECK(ctx && c && (count == 0 || idx_dev), FT_ERR_SHAPE, "null argument");
  FT_CHECK(start >= 0 && count >= 0 && start + count <= c->len, FT_ERR_SHAPE,
           "%lld positions from %lld on do not come out of a cache of %lld", (long long)count,
           (long long)start, (long long)c->len);
  FT_CHECK(idx_batch_stride >= 0 && idx_head_stride >= 0, FT_ERR_SHAPE, "negative stride");
  FT_CHECK(c->len < (int64_t)INT32_MAX, FT_ERR_UNSUPPORTED, "cache too long for 32-bit indices");
  if (count > 0) {
    DeviceScope scope(c->device);
    // a full ring whose kept positions would end in the head's own block: two
    // destination blocks would share one record, so the ring is laid out anew
    if (c->head % kBlk + start + count > c->cap) {
      const int rc = kv3_grow(c, c->len, static_cast<cudaStream_t>(stream));
      if (rc != FT_OK) return rc;
    }
    KeepParams p{};
    p.H = c->kv_heads;
    p.nbc = c->cap / kBlk;
    p.head_off = c->head % kBlk;
    p.head_blk = c->head / kBlk;
    p.len = c->len;
    p.blocks = c->blocks;
    p.idx = idx_dev;
    p.ib = idx_batch_stride;
    p.ih = idx_head_stride;
    p.start = start;
    p.count = count;
    p.err = ctx->err_word;
    const int rc =
        launch_keep(ctx, p, c->batch * c->kv_heads, static_cast<cudaStream_t>(stream));
    if (rc != FT_OK) return rc;
  }
  c->len = start + count;
  return FT_OK;
}

int ft_kvp_keep(ft_ctx* ctx, ft_kvp* c, int64_t batch, const int32_t* tables_dev,
                int64_t table_stride, const int32_t* seq_lens_dev, const int32_t* start_dev,
                const int32_t* count_dev, int64_t max_count, const int32_t* idx_dev,
                int64_t idx_batch_stride, int64_t idx_head_stride, void* stream) {
  FT_CHECK(ctx && c && tables_dev && seq_lens_dev && start_dev && count_dev &&
               (max_count == 0 || idx_dev),
           FT_ERR_SHAPE, "null argument");
  FT_CHECK(batch >= 0 && table_stride > 0 && max_count >= 0 &&
               max_count <= table_stride * kBlk && table_stride < INT32_MAX / kBlk,
           FT_ERR_SHAPE, "bad shape (batch %lld, %lld positions, table stride %lld)",
           (long long)batch, (long long)max_count, (long long)table_stride);
  FT_CHECK(idx_batch_stride >= 0 && idx_head_stride >= 0, FT_ERR_SHAPE, "negative stride");
  if (batch == 0 || max_count == 0) return FT_OK;
  DeviceScope scope(c->device);
  KeepParams p{};
  p.H = c->kv_heads;
  p.nbc = 1;
  p.len = table_stride * kBlk;
  p.blocks = c->blocks;
  p.idx = idx_dev;
  p.ib = idx_batch_stride;
  p.ih = idx_head_stride;
  p.count = max_count;
  p.starts = start_dev;
  p.counts = count_dev;
  p.seq_lens = seq_lens_dev;
  p.table = tables_dev;
  p.tstride = table_stride;
  p.n_pages = c->n_pages;
  p.err = ctx->err_word;
  return launch_keep(ctx, p, batch * c->kv_heads, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
