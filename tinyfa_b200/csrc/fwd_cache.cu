// Attention over the paged 8-bit K/V cache, few query rows per request (decode steps, draft tokens): sm_100a.
//
//   S = (q . k) / sqrt(D), k = code * scale[block, head];  capped: S <- c tanh(S / c);  biased: S <- S - slope_h |pos - j|
//   O = sum_j exp(S_j) v_j / sum_j exp(S_j) over the keys j <= pos of a query at position pos (all keys without the causal mask)
//
// Bound by HBM: every code is read once per KV head, the products are a few per cent of the time.  So the kernel is a stream:
//   * the query rows that share a KV head form tiles of 8 (or 16) rows; the 64-key blocks of all (request, tile) units in a row are cut
//     into equal runs, one CTA per run and KV head, whatever the lengths are - which only the device knows;
//   * each of a CTA's four warps takes every fourth 16-key slice, with a ring of its own that cp.async fills slices ahead, across the
//     ends of requests, and a running reference value and sum of its own.  Nothing but the end of a unit synchronises the CTA;
//   * codes become fp16 exactly (int8 and e4m3 both fit its 11 bits), so mma.sync sees the codes themselves: the scale of a block of
//     keys multiplies the scores, the scale of a block of values the weights.  bf16 queries become fp16 with a power of two per row
//     taken out, which loses only what lies 2^-31 below the row's largest element;
//   * both products are transposed, S^T = K Q^T and O^T = V^T P^T, so that the 16 rows of an MMA are keys and head-dim elements and its
//     8 columns the query rows, of which a decode step has few: half the MMAs, half the accumulators and half the exponentials of
//     tiles of 16 query rows.  P^T becomes the other operand with two 8 x 8 transposes (movmatrix);
//   * the contraction index of S^T and the row index of O^T are permuted so that a lane's codes are 16 (D = 128) contiguous bytes of a
//     cache row; O^T needs two byte permutes per four codes to bring two keys together;
//   * weights are stored relative to a scale of V that is at most 2^3 below the largest seen and 2^4 up, so that the fp16 weights of a
//     block whose scale is 2^-18 of the largest still have all their bits;
//   * a unit that several runs share is put together by the CTA that finishes last, which it learns from a counter.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <mutex>

#include "../../include/tinyfa_b200.h"
#include "build_config.cuh"
#include "cache_codes.cuh"
#include "cta_scan.cuh"
#include "fwd_tc.cuh"
#include "ptx_sm100.cuh"
#include "tfa_common.cuh"

namespace tfa_b200 {

int device_num_sms(int device);  // c_abi.cu
int* device_join_counters(int device, cudaStream_t stream, int* rc);  // c_abi.cu
int* device_status_word(int device);
int next_epoch();
int option_cache_tc();

#define TFA_DECLARE_CACHE(HDP)                                                                              \
  int launch_fwd_cache_hdp##HDP##_bf0(const TcCacheParams&, int, bool, int, cudaStream_t);                  \
  int launch_fwd_cache_hdp##HDP##_bf1(const TcCacheParams&, int, bool, int, cudaStream_t);                  \
  static inline int cache_call_hdp##HDP(const TcCacheParams& p, bool bf16, int ctas, bool overlap, int device, cudaStream_t s) { \
    (void)p; (void)ctas; (void)overlap; (void)device; (void)s;                                              \
    if (bf16) {                                                                                             \
      if constexpr (TFA_HAVE_BF16) return launch_fwd_cache_hdp##HDP##_bf1(p, ctas, overlap, device, s);      \
    } else {                                                                                                \
      if constexpr (TFA_HAVE_FP16) return launch_fwd_cache_hdp##HDP##_bf0(p, ctas, overlap, device, s);      \
    }                                                                                                       \
    return kBadDtype;                                                                                       \
  }
#if TFA_HAVE_HDP64
TFA_DECLARE_CACHE(64)
#endif
#if TFA_HAVE_HDP128
TFA_DECLARE_CACHE(128)
#endif
#if TFA_HAVE_HDP192
TFA_DECLARE_CACHE(192)
#endif
#if TFA_HAVE_HDP256
TFA_DECLARE_CACHE(256)
#endif
#undef TFA_DECLARE_CACHE

namespace cache {

constexpr int kThreads = 128;
constexpr int kBlockKeys = 64;  // unit of the partition: a slice of 16 keys for each warp
constexpr int kRows = 16;       // most query rows of a tile
// A row's reference value follows its maximum when that is 2^8 ahead, the reference scale of V when a scale is 2^3 ahead; weights are stored
// 2^4 larger: at most 2^15, within fp16.
constexpr float kLag = 8.f, kScaleLag = 8.f, kUp = 16.f;

struct Params {
  const void* Q;
  void* O;
  const uint8_t* kCodes;
  const uint8_t* vCodes;
  const float* kScales;
  const float* vScales;
  const int* table;  // [batch][width]
  const int* lens;   // [batch] tokens of each request, its new ones included
  const int* cuQ;    // [batch + 1]
  const float* slopes;  // [headsQ] or null
  int batch, width, numBlocks, blockShift;
  int headsQ, headsKV, group;
  int causal;
  int runs;
  int totalQ;
  float scaleLog2;  // log2(e) / sqrt(D)
  float cap;        // 0: none
  float* partO;     // [runs][headsKV][2][rows of a tile][D] normalised
  float* partLse;   // [runs][headsKV][2][rows of a tile]
  int* join;        // [runs][headsKV], zero
};

// Bytes of a row of K and V in shared memory: a multiple of 16 that keeps the lanes of a load on different banks (K: eight rows of
// 64 bytes; V: rows 2 apart) for D = 32, 64, 128, 192 (V at 192 and 256, K at 96: two lanes to a bank).
template <int D>
constexpr int k_pitch() {
  return D % 128 == 0 ? D + 64 : D;
}
template <int D>
constexpr int v_pitch() {
  return D + 16;
}
constexpr int kHeader = 16;  // scale of K, scale of V, whether the block exists
template <int D>
constexpr int stage_bytes() {
  return 16 * (k_pitch<D>() + v_pitch<D>()) + kHeader;
}
// CTAs of an SM that registers allow (O^T and Q take 3 D / 8 a thread for 8 rows, twice that for 16), and slices in a warp's ring: what shared
// memory holds then, three to six of them.
template <int D, int NR>
constexpr int ctas_per_sm() {
  return D <= 64 ? (NR == 1 ? 5 : 4) : D <= 128 ? (NR == 1 ? 3 : 2) : NR == 1 ? 2 : 1;
}
template <int D, int NR>
constexpr int merge_bytes() {
  return (8 * NR * (D + 8) + 2 * 4 * 8 * NR) * (int)sizeof(float);
}
template <int D, int NR>
constexpr int stages() {
  constexpr int room = (227 * 1024 / ctas_per_sm<D, NR>() - 1536 - merge_bytes<D, NR>()) / (4 * stage_bytes<D>());
  return room > 6 ? 6 : room;
}
template <int D, int NR>
constexpr int ring_bytes() {
  return 4 * stages<D, NR>() * stage_bytes<D>();
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit elements, a row per quad of lanes -> its transpose
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// kWords consecutive words of a lane from shared memory, in the widest loads that its alignment (kAlign bytes) allows.
template <int kWords, int kAlign>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[kWords]) {
  if constexpr (kAlign >= 16 && kWords % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(addr + i * 4));
    }
  } else if constexpr (kAlign >= 8 && kWords % 2 == 0) {
#pragma unroll
    for (int i = 0; i < kWords; i += 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(addr + i * 4));
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i++) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[i]) : "r"(addr + i * 4));
  }
}

// Where a lane's bytes of a K row lie, and which elements of Q meet them: lane q of a quad has 16 bytes of every 64, and 8 of the
// last 32 where D is an odd multiple of 32.  Word w of the row's D / 16 words per lane is k-step w of the contraction.
template <int D>
__device__ __forceinline__ constexpr int k_byte(int w, int q) {
  return w / 4 * 64 + (w / 4 < D / 64 ? q * 16 + w % 4 * 4 : q * 8 + w % 4 * 4);
}

// A run's position in the row of units: blocks [blk, blocks) of query tile `tile` of request b.
struct Segment {
  int b, tile;
  int blk, end;       // key blocks of the segment
  int blocks;         // key blocks of the unit
  int q0, nq, len;    // request: first row of Q, rows, tokens
  int keyEnd;         // keys that some row of the tile sees
};

template <int NR>
__device__ __forceinline__ int tiles_of(int nq, int group) {
  return (int)(((long long)nq * group + 8 * NR - 1) / (8 * NR));
}

// The blocks of all units, in order, cut into runs of equal length.  A cut within `snap` blocks of a unit's end is moved there: some blocks more
// for one run cost less than parts of a unit that have to be put together.  us without -> with: 8 x 3000 tokens 21.2 -> 18.6, 256 x 500 to 1000
// 86.0 -> 80.8, 64 x 300 21.0 -> 19.5, 64 x 4000 94.8 -> 93.7 (8 KV heads of 128, e4m3).
struct Cuts {
  int total, base, extra, snap;
  __device__ __forceinline__ Cuts(int blocks, int runs) : total(blocks), base(blocks / runs), extra(blocks - base * runs), snap(min(4, base / 2)) {}
  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, extra); }
  __device__ __forceinline__ int run_of(int u) const {  // the c with begin(c) <= u < begin(c + 1)
    const int longer = extra * (base + 1);
    return u < longer ? u / (base + 1) : extra + (u - longer) / base;
  }
  // how far a cut moves that is blk blocks into a unit of `blocks`
  __device__ __forceinline__ int move(int blk, int blocks) const { return blk <= snap ? -blk : blocks - blk <= snap ? blocks - blk : 0; }
};

// NR: tiles of 8 NR query rows.
template <int D, bool kInt8, bool kBf16, int NR>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D, NR>()) cache_decode_kernel(const Params p) {
  constexpr int kS = stages<D, NR>(), kStage = stage_bytes<D>(), KP = k_pitch<D>(), VP = v_pitch<D>();
  static_assert(kS >= 2, "a slice to work on and one on its way");
  constexpr int kTile = 8 * NR;  // query rows
  constexpr int kMT = D / 16;    // 16-element row tiles of O^T
  constexpr int kLdO = D + 8;    // row pitch of the merge buffer
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sScan[2][kThreads / 32];
  __shared__ int sPlace[2][5];  // request that holds the run's first block, and the one behind its last: number, blocks ahead of it, q0, nq, len
  __shared__ int sLast;
  float* sO = reinterpret_cast<float*>(smem + ring_bytes<D, NR>());  // [kTile][kLdO]
  float* sM = sO + kTile * kLdO;                                     // [4][kTile]
  float* sL = sM + 4 * kTile;                                        // [4][kTile]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tig = lane & 3;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kS * kStage;

  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  // neighbouring CTAs are the KV heads of one run: they read neighbouring tiles of the same blocks at the same time
  const int run = (int)blockIdx.x / p.headsKV;
  const int hkv = (int)blockIdx.x - run * p.headsKV;
  const int capacity = p.width << p.blockShift;

  auto request = [&](int b, int& q0, int& nq, int& len) {
    q0 = min(max(p.cuQ[b], 0), p.totalQ);
    nq = min(max(p.cuQ[b + 1] - q0, 0), p.totalQ - q0);
    len = min(max(p.lens[b], 0), capacity);
  };
  auto unit_blocks = [&](int len) { return (len + kBlockKeys - 1) / kBlockKeys; };
  auto blocks_of = [&](int nq, int len) { return (long long)tiles_of<NR>(nq, p.group) * unit_blocks(len); };
  // ---- the blocks of all requests; the first kThreads requests stay in registers
  int q0 = 0, nq = 0, len = 0;
  if ((int)threadIdx.x < p.batch) request(threadIdx.x, q0, nq, len);
  const long long mine = blocks_of(nq, len);
  long long upto = mine, more = 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  for (int b = threadIdx.x + kThreads; b < p.batch; b += kThreads) {
    int a, n, m;
    request(b, a, n, m);
    more += blocks_of(n, m);
  }
  if (p.batch > kThreads) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) more += __shfl_xor_sync(0xffffffffu, more, d);
  }
  if (lane == 31) {
    sScan[0][warp] = upto;
    sScan[1][warp] = more;
  }
  __syncthreads();
  long long sum = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; w++) {
    if (w < warp) upto += sScan[0][w];
    sum += sScan[0][w];
    all += sScan[1][w];
  }
  all += sum;
  if (all > 0x7FFFFFFFll) return;  // offsets that are not ascending: the host has checked what rows and blocks can give
  const int total = (int)all;
  int carry = (int)sum;

  // ---- rows that no unit has: those of no request, and those of requests without a token; a share for every CTA
  auto zero_rest = [&]() {
    uint16_t* O = static_cast<uint16_t*>(p.O);
    auto zero_rows = [&](int r0, int r1) {  // this head's part of them
      constexpr int kVec = D / 8;
      const int per = p.group * kVec;
      for (long long i = threadIdx.x; i < (long long)(r1 - r0) * per; i += kThreads) {
        const long long row = r0 + i / per;
        *reinterpret_cast<uint4*>(O + (row * p.headsQ + hkv * p.group) * D + (i % per) * 8) = make_uint4(0, 0, 0, 0);
      }
    };
    if (run == 0) {
      zero_rows(0, min(max(p.cuQ[0], 0), p.totalQ));
      zero_rows(min(max(p.cuQ[p.batch], 0), p.totalQ), p.totalQ);
    }
    for (int b = run; b < p.batch; b += p.runs) {
      int q0, nq, len;
      request(b, q0, nq, len);
      if (len == 0) zero_rows(q0, q0 + nq);
    }
  };
  // The host sized the grid for the largest lengths: with fewer blocks, fewer runs of at least two blocks.
  const int runs = min(p.runs, (total + 1) / 2);
  if (run >= runs) {
    zero_rest();
    return;
  }
  const Cuts cuts(total, runs);
  int u0 = cuts.begin(run), u1 = cuts.begin(run + 1);
  auto place = [&](int b, int ahead, int n, int a, int rows, int tokens) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int u = i == 0 ? u0 : u1;
      if (u >= ahead && u < ahead + n) {
        sPlace[i][0] = b;
        sPlace[i][1] = ahead;
        sPlace[i][2] = a;
        sPlace[i][3] = rows;
        sPlace[i][4] = tokens;
      }
    }
  };
  place(threadIdx.x, (int)(upto - mine), (int)mine, q0, nq, len);
  for (int b0 = kThreads; b0 < p.batch && carry <= u1; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int a = 0, n = 0, m = 0;
    if (b < p.batch) request(b, a, n, m);
    const int blocks = (int)blocks_of(n, m);
    int v = blocks;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();  // sScan has been read
    if (lane == 31) sScan[0][warp] = v;
    __syncthreads();
    int here = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++) {
      if (w < warp) v += (int)sScan[0][w];
      here += (int)sScan[0][w];
    }
    place(b, carry + v - blocks, blocks, a, n, m);
    carry += here;
  }
  __syncthreads();

  auto finish = [&](Segment& s) {  // the fields that follow from the request and the tile
    const int lastRow = min((s.tile + 1) * kTile, s.nq * p.group) - 1;
    s.keyEnd = p.causal ? min(s.len, s.len - s.nq + lastRow / p.group + 1) : s.len;
  };
  auto next_segment = [&](Segment& s, int& rest) {  // rest > 0
    s.tile++;
    if (s.tile >= tiles_of<NR>(s.nq, p.group)) {
      s.tile = 0;
      do {  // ends: `rest` blocks are still to come
        s.b++;
        request(s.b, s.q0, s.nq, s.len);
      } while (s.nq == 0 || s.len == 0);
      s.blocks = unit_blocks(s.len);
    }
    s.blk = 0;
    s.end = min(s.blocks, rest);
    rest -= s.end;
    finish(s);
  };

  // ---- the loads: a cursor of its own, kS - 1 slices ahead
  Segment ls;
  ls.b = sPlace[0][0];
  ls.q0 = sPlace[0][2];
  ls.nq = sPlace[0][3];
  ls.len = sPlace[0][4];
  ls.blocks = unit_blocks(ls.len);
  ls.tile = (u0 - sPlace[0][1]) / ls.blocks;
  ls.blk = u0 - sPlace[0][1] - ls.tile * ls.blocks;
  const int moved = cuts.move(ls.blk, ls.blocks);
  u0 += moved;
  if (u1 < total) {
    const int blocks = unit_blocks(sPlace[1][4]);
    u1 += cuts.move((u1 - sPlace[1][1]) % blocks, blocks);
  }
  if (u0 >= u1) {
    zero_rest();
    return;
  }
  int left = u1 - u0;  // blocks of the run behind the segment
  if (moved > 0) {
    next_segment(ls, left);
  } else {
    ls.blk += moved;
    ls.end = min(ls.blocks, ls.blk + left);
    left -= ls.end - ls.blk;
    finish(ls);
  }
  Segment s = ls;
  int lsRest = left;
  bool loading = true;
  int ldKey = ls.blk * kBlockKeys + warp * 16, ldStage = 0;
  const long long headBytes = (long long)D << p.blockShift;
  auto seg_key_end = [&](const Segment& s) { return min(s.end * kBlockKeys, s.keyEnd); };
  // Pages of the next 32 slices of the segment, one to a lane: asked for together, and a slice ahead of their use.
  int ldPages = 0, ldTurn = 32;
  auto settle = [&]() {  // on to the next slice that exists
    while (loading && ldKey >= seg_key_end(ls)) {
      if (lsRest == 0) {
        loading = false;
      } else {
        next_segment(ls, lsRest);
        ldKey = warp * 16;
        ldTurn = 32;
      }
    }
    if (loading && ldTurn == 32) {
      const int key = ldKey + lane * kBlockKeys;
      ldPages = key < seg_key_end(ls) ? p.table[(long long)ls.b * p.width + (key >> p.blockShift)] : -1;
      ldTurn = 0;
    }
  };
  settle();
  auto issue = [&]() {
    if (loading) {
      const uint32_t st = ring + ldStage * kStage;
      const int ldPage = __shfl_sync(0xffffffffu, ldPages, ldTurn);
      ldTurn++;
      const bool ok = ldPage >= 0 && ldPage < p.numBlocks;
      const long long tile = ok ? (long long)ldPage * p.headsKV + hkv : 0;
      const int rows = ok ? min(16, ls.len - ldKey) : 0;  // keys of the slice
      const long long from = tile * headBytes + (ldKey & ((1 << p.blockShift) - 1)) * D + lane * 16;
      const uint8_t* k = p.kCodes + from;
      const uint8_t* v = p.vCodes + from;
      if (rows == 16) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const int c = lane + i * 32, r = c / (D / 16), col = c % (D / 16) * 16;
          cp_async16(st + r * KP + col, k + i * 512, true);
          cp_async16(st + 16 * KP + r * VP + col, v + i * 512, true);
        }
      } else {  // what the request does not have is zero
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const int c = lane + i * 32, r = c / (D / 16), col = c % (D / 16) * 16;
          cp_async16(st + r * KP + col, r < rows ? k + i * 512 : p.kCodes, r < rows);
          cp_async16(st + 16 * KP + r * VP + col, r < rows ? v + i * 512 : p.vCodes, r < rows);
        }
      }
      const uint32_t head = st + 16 * (KP + VP);
      if (lane == 0) {
        cp_async4(head, p.kScales + tile, ok);
        cp_async4(head + 4, p.vScales + tile, ok);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(head + 8), "r"(ok ? 1 : 0) : "memory");
      }
      ldStage = ldStage + 1 == kS ? 0 : ldStage + 1;
      ldKey += kBlockKeys;
      settle();
    }
    cp_async_commit();
  };
  // ---- the units of the run
  int stage = 0;
  bool started = false;
  for (;;) {
    const int nRows = min(s.nq * p.group - s.tile * kTile, kTile);
    // rows of the tile: row 0 is head `head0` of query `query0`.  (x + 1/2) / group in 32 bits: exact for the few rows of a tile
    const int query0 = s.tile * kTile / p.group, head0 = s.tile * kTile - query0 * p.group;
    const float byGroup = 1.f / (float)p.group;
    auto query_of = [&](int row) { return (int)(((float)(head0 + row) + 0.5f) * byGroup); };
    // Q as the columns of S^T: row 8 nr + g of the tile, permuted like the lanes' bytes of K
    uint32_t qf[D / 16][NR][2];
    float rowDown[NR], slope[NR][2];
    int pos[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
      const int row = nr * 8 + g < nRows ? nr * 8 + g : 0, query = query_of(row);
      const uint16_t* q = static_cast<const uint16_t*>(p.Q) +
                          ((long long)(s.q0 + query0 + query) * p.headsQ + hkv * p.group + head0 + row - query * p.group) * D;
#pragma unroll
      for (int w = 0; w < D / 16; w++) {
        const uint2 x = *reinterpret_cast<const uint2*>(q + k_byte<D>(w, tig));
        qf[w][nr][0] = x.x;
        qf[w][nr][1] = x.y;
      }
      // this thread's columns of S^T and O^T: rows 8 nr + 2 tig + e
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = nr * 8 + 2 * tig + e < nRows ? nr * 8 + 2 * tig + e : 0, query = query_of(col);
        pos[nr][e] = s.len - s.nq + query0 + query;
        slope[nr][e] = p.slopes != nullptr ? p.slopes[hkv * p.group + head0 + col - query * p.group] * 1.44269504f : 0.f;
      }
    }
    if (!started) {  // the first slices, while Q is on its way
#pragma unroll 1
      for (int i = 0; i < kS - 1; i++) issue();
      zero_rest();
      started = true;
    }
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
      const bool valid = nr * 8 + g < nRows;
      constexpr uint32_t kE = exponent_bits<kBf16>();
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < D / 16; w++) {
        qf[w][nr][0] = valid ? qf[w][nr][0] : 0u;
        qf[w][nr][1] = valid ? qf[w][nr][1] : 0u;
        top = max(max(top, qf[w][nr][0] & kE), max(qf[w][nr][0] >> 16 & kE, max(qf[w][nr][1] & kE, qf[w][nr][1] >> 16 & kE)));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float up;
      row_scale<kBf16>(top, up, rowDown[nr]);
#pragma unroll
      for (int w = 0; w < D / 16; w++) {
        qf[w][nr][0] = scale_to_half2<kBf16>(qf[w][nr][0], up);
        qf[w][nr][1] = scale_to_half2<kBf16>(qf[w][nr][1], up);
      }
    }
    // capped: scores as arguments 2 log2(e) S / c of the exponential that gives the tanh
    float fac[NR][2];
    const float capLog2 = p.cap * 1.44269504f, unit = p.scaleLog2 * (p.cap > 0.f ? 2.f / p.cap : 1.f);
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
#pragma unroll
      for (int e = 0; e < 2; e++) fac[nr][e] = __shfl_sync(0xffffffffu, rowDown[nr], (2 * tig + e) * 4) * unit;
    }

    float o[kMT][NR][4];
#pragma unroll
    for (int i = 0; i < kMT; i++) {
#pragma unroll
      for (int nr = 0; nr < NR; nr++) o[i][nr][0] = o[i][nr][1] = o[i][nr][2] = o[i][nr][3] = 0.f;
    }
    float ref[NR][2], limit[NR][2], l[NR][2];  // reference value (0 until a key is seen), score that moves it, sum of this thread's keys
#pragma unroll
    for (int nr = 0; nr < NR; nr++) ref[nr][0] = ref[nr][1] = l[nr][0] = l[nr][1] = 0.f, limit[nr][0] = limit[nr][1] = -INFINITY;
    float vRef = 0.f, vUp = 0.f;  // scale of V that O refers to: O holds sums of 2^4 p v / vRef

    const int keyStop = seg_key_end(s), seenByAll = p.causal ? s.len - s.nq + query0 : s.len - 1;
    for (int key0 = s.blk * kBlockKeys + warp * 16; key0 < keyStop; key0 += kBlockKeys) {
      cp_async_wait<kS - 2>();
      __syncwarp();  // ... and every lane has read the stage of the slice before
      if (kS == 2) issue();  // nothing else is on its way: D = 256, 64 x 4000 tokens 202 -> 176 us (and 99 -> 99.5 at 128, where two more are)
      const uint32_t st = ring + stage * kStage;
      float ks, vs;
      uint32_t there;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks) : "r"(st + 16 * (KP + VP)));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs) : "r"(st + 16 * (KP + VP) + 4));
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(there) : "r"(st + 16 * (KP + VP) + 8));
      // ---- S^T = K Q^T: 16 keys x 8 NR rows
      float sc[NR][4], sd[NR][4];  // two chains of MMAs
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
        sc[nr][0] = sc[nr][1] = sc[nr][2] = sc[nr][3] = 0.f;
        sd[nr][0] = sd[nr][1] = sd[nr][2] = sd[nr][3] = 0.f;
      }
      const uint32_t k0 = st + g * KP, k1 = k0 + 8 * KP;
      auto scores = [&](uint32_t w0, uint32_t w1, int step) {
        uint32_t a[4];
        widen<kInt8>(w0, a[0], a[2]);
        widen<kInt8>(w1, a[1], a[3]);
#pragma unroll
        for (int nr = 0; nr < NR; nr++) mma_f16((step & 1) ? sd[nr] : sc[nr], a, qf[step][nr][0], qf[step][nr][1]);
      };
#pragma unroll
      for (int c = 0; c < D / 64; c++) {
        uint32_t w0[4], w1[4];
        lds_words<4, 16>(k0 + c * 64 + tig * 16, w0);
        lds_words<4, 16>(k1 + c * 64 + tig * 16, w1);
#pragma unroll
        for (int i = 0; i < 4; i++) scores(w0[i], w1[i], c * 4 + i);
      }
      if constexpr (D % 64 != 0) {
        uint32_t w0[2], w1[2];
        lds_words<2, 8>(k0 + D / 64 * 64 + tig * 8, w0);
        lds_words<2, 8>(k1 + D / 64 * 64 + tig * 8, w1);
#pragma unroll
        for (int i = 0; i < 2; i++) scores(w0[i], w1[i], D / 64 * 4 + i);
      }
      // ---- scores in units of log2, capped, biased, masked
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
        const float f0 = fac[nr][0] * ks, f1 = fac[nr][1] * ks;
#pragma unroll
        for (int e = 0; e < 4; e++) sc[nr][e] = (sc[nr][e] + sd[nr][e]) * ((e & 1) ? f1 : f0);
        if (p.cap > 0.f) score::cap_few(sc[nr], capLog2);
        if (p.slopes != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            sc[nr][e] = fmaf(-slope[nr][e & 1], fabsf((float)(pos[nr][e & 1] - (key0 + g + (e >> 1) * 8))), sc[nr][e]);
          }
        }
      }
      if (!there || key0 + 16 > s.len || key0 + 15 > seenByAll) {
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int lim = !there ? 0 : p.causal ? min(s.len, pos[nr][e & 1] + 1) : s.len;
            if (key0 + g + (e >> 1) * 8 >= lim) sc[nr][e] = -INFINITY;
          }
        }
      }
      // ---- rows whose scores are far above their reference, or values far above theirs: rare
      bool move = vs > vRef * kScaleLag;
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
#pragma unroll
        for (int e = 0; e < 4; e++) move = move || sc[nr][e] > limit[nr][e & 1];
      }
      if (__any_sync(0xffffffffu, move)) {
        const float vNew = fmaxf(fmaxf(vRef, vs), kSmallestVRef);
        const float fv = vNew > vRef ? vRef / vNew : 1.f;
        vRef = vNew;
        vUp = 1.f / vNew * kUp;
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float top = fmaxf(sc[nr][e], sc[nr][e + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const bool none = limit[nr][e] == -INFINITY;  // no key so far
            const float now = none ? top : fmaxf(ref[nr][e], top);
            const float f = none ? 0.f : ex2(ref[nr][e] - now);
            if (now != -INFINITY) {
              ref[nr][e] = now;
              limit[nr][e] = now + kLag;
            }
            l[nr][e] *= f;
            const float fo = f * fv;
#pragma unroll
            for (int i = 0; i < kMT; i++) {
              o[i][nr][e] *= fo;
              o[i][nr][e + 2] *= fo;
            }
          }
        }
      }
      // ---- weights: 11 bits, half a step is 2^-12 of a weight
      const float wv = vs * vUp;
      uint32_t pf[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = ex2(sc[nr][e] - ref[nr][e & 1]);
        l[nr][0] += w[0] + w[2];
        l[nr][1] += w[1] + w[3];
        pf[nr][0] = transpose8x8(half2_of(w[0] * wv, w[1] * wv));
        pf[nr][1] = transpose8x8(half2_of(w[2] * wv, w[3] * wv));
      }
      // ---- O^T += V^T P^T: rows g and g + 8 of tile j are head-dim elements g D / 8 + 2 j and + 1, so that a lane's D / 8 codes of a key are
      // contiguous
      constexpr int kAlign = (D / 8) % 16 == 0 ? 16 : (D / 8) % 8 == 0 ? 8 : 4;
      constexpr int kPiece = kAlign / 4;
      const uint32_t vr = st + 16 * KP + g * (D / 8);
#pragma unroll
      for (int c = 0; c < D / 32; c += kPiece) {
        uint32_t w[4][kPiece];
#pragma unroll
        for (int i = 0; i < 4; i++) lds_words<kPiece, kAlign>(vr + (2 * tig + (i & 1) + (i >> 1) * 8) * VP + c * 4, w[i]);
#pragma unroll
        for (int i = 0; i < kPiece; i++) {
          uint32_t lo[4], hi[4];  // by head-dim element: keys 2 tig, 2 tig + 1 and 2 tig + 8, 2 tig + 9
          widen<kInt8>(__byte_perm(w[0][i], w[1][i], 0x5140), lo[0], lo[1]);
          widen<kInt8>(__byte_perm(w[0][i], w[1][i], 0x7362), lo[2], lo[3]);
          widen<kInt8>(__byte_perm(w[2][i], w[3][i], 0x5140), hi[0], hi[1]);
          widen<kInt8>(__byte_perm(w[2][i], w[3][i], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t a[4] = {lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1]};
#pragma unroll
            for (int nr = 0; nr < NR; nr++) mma_f16(o[(c + i) * 2 + j][nr], a, pf[nr][0], pf[nr][1]);
          }
        }
      }
      stage = stage + 1 == kS ? 0 : stage + 1;
      if (kS > 2) {
        __syncwarp();
        issue();
      }
    }

    // ---- the four warps' shares of the unit, one after the other
#pragma unroll
    for (int nr = 0; nr < NR; nr++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        l[nr][e] += __shfl_xor_sync(0xffffffffu, l[nr][e], 4);
        l[nr][e] += __shfl_xor_sync(0xffffffffu, l[nr][e], 8);
        l[nr][e] += __shfl_xor_sync(0xffffffffu, l[nr][e], 16);
        if (g == 0) {
          sM[warp * kTile + nr * 8 + 2 * tig + e] = limit[nr][e] == -INFINITY ? -INFINITY : ref[nr][e];
          sL[warp * kTile + nr * 8 + 2 * tig + e] = l[nr][e];
        }
      }
    }
    __syncthreads();
    {
      float f[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; nr++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float M = -INFINITY;
#pragma unroll
          for (int w = 0; w < 4; w++) M = fmaxf(M, sM[w * kTile + nr * 8 + 2 * tig + e]);
          f[nr][e] = (limit[nr][e] == -INFINITY ? 0.f : ex2(ref[nr][e] - M)) * vRef * (1.f / kUp);
        }
      }
#pragma unroll 1
      for (int w = 0; w < 4; w++) {
        if (w == warp) {
#pragma unroll
          for (int nr = 0; nr < NR; nr++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
              // elements g D / 8 + 2 j and + 1 of the row stand at 16 j + 2 g: the lanes of an access on different banks
              float2* at = reinterpret_cast<float2*>(sO + (nr * 8 + 2 * tig + e) * kLdO + 2 * g);
#pragma unroll
              for (int j = 0; j < kMT; j++) {
                const float2 z = w == 0 ? make_float2(0.f, 0.f) : at[j * 8];
                at[j * 8] = make_float2(fmaf(o[j][nr][e], f[nr][e], z.x), fmaf(o[j][nr][e + 2], f[nr][e], z.y));
              }
            }
          }
        }
        __syncthreads();
      }
    }
    const bool whole = s.blk == 0 && s.end == s.blocks;
    // parts of a run: of the unit that it begins and does not end, of the one that it does not begin
    const long long slot = ((long long)run * p.headsKV + hkv) * 2 + (s.blk == 0 ? 0 : 1);
    auto store = [&](int r, int c4, float4 acc) {
      const int query = query_of(r);
      uint16_t* dst = static_cast<uint16_t*>(p.O) + ((long long)(s.q0 + query0 + query) * p.headsQ + hkv * p.group + head0 + r - query * p.group) * D + c4 * 4;
      uint2 out;
      if constexpr (kBf16) {
        __nv_bfloat162 x = __floats2bfloat162_rn(acc.x, acc.y), y = __floats2bfloat162_rn(acc.z, acc.w);
        out.x = *reinterpret_cast<uint32_t*>(&x);
        out.y = *reinterpret_cast<uint32_t*>(&y);
      } else {
        out.x = half2_of(acc.x, acc.y);
        out.y = half2_of(acc.z, acc.w);
      }
      *reinterpret_cast<uint2*>(dst) = out;
    };
    for (int idx = threadIdx.x; idx < nRows * (D / 4); idx += kThreads) {
      const int r = idx / (D / 4), c4 = idx % (D / 4);
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) m = fmaxf(m, sM[w * kTile + r]);
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float mw = sM[w * kTile + r];
        l += sL[w * kTile + r] * (mw == -INFINITY ? 0.f : ex2(mw - m));
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays NaN
      const float* from = sO + r * kLdO + c4 * 4 % (D / 8) * 8 + c4 * 4 / (D / 8) * 2;
      const float2 lo = *reinterpret_cast<const float2*>(from), hi = *reinterpret_cast<const float2*>(from + 16);
      float4 acc = make_float4(lo.x, lo.y, hi.x, hi.y);
      acc.x *= inv;
      acc.y *= inv;
      acc.z *= inv;
      acc.w *= inv;
      if (whole) {
        store(r, c4, acc);
      } else {
        __stcg(reinterpret_cast<float4*>(p.partO + (slot * kTile + r) * D + c4 * 4), acc);
        if (c4 == 0) __stcg(p.partLse + slot * kTile + r, l == 0.f ? -INFINITY : m + log2f(l));
      }
    }
    if (!whole) {
      // ---- the unit is shared by runs c0 .. c1: whoever comes last puts the parts together
      const int a = (u1 - left) - s.end;  // the unit's first block (u1 - left: the block behind the segment)
      const int c0 = cuts.run_of(a + cuts.snap), c1 = cuts.run_of(a + s.blocks - 1 - cuts.snap);
      __syncthreads();
      if (threadIdx.x == 0) {  // releases what the CTA has stored before the barrier, acquires what the others' have
        int* counter = p.join + (long long)c0 * p.headsKV + hkv;
        int seen;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
        const bool last = seen == c1 - c0;
        if (last) *counter = 0;  // for the next call
        sLast = last;
      }
      __syncthreads();
      if (sLast) {
        auto part = [&](int c) { return ((long long)c * p.headsKV + hkv) * 2 + (c == c0 ? 0 : 1); };
        // Groups of D / 4 threads take turns over the parts, four rows of kAhead parts in flight at once: sums relative to the largest
        // log-sum-exp so far; then the groups' sums.
        constexpr int kVec = D / 4, kGroups = kThreads / kVec < 4 ? kThreads / kVec : 4, kAhead = D <= 64 ? 2 : 4;
        const int group = threadIdx.x / kVec, c4 = threadIdx.x % kVec;
#pragma unroll 1
        for (int r0 = 0; r0 < nRows; r0 += 4) {
          float4 acc[4];
          float M[4], sum[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            M[r] = -INFINITY;
            sum[r] = 0.f;
          }
          if (group < kGroups) {
#pragma unroll 1
            for (int c = c0 + group; c <= c1; c += kGroups * kAhead) {
              float lse[kAhead][4];
              float4 v[kAhead][4];
#pragma unroll
              for (int u = 0; u < kAhead; u++) {
                const bool there = c + u * kGroups <= c1;
                const long long at = part(there ? c + u * kGroups : c) * kTile + r0;
                const float4 x = __ldcg(reinterpret_cast<const float4*>(p.partLse + at));
                lse[u][0] = there ? x.x : -INFINITY;
                lse[u][1] = there ? x.y : -INFINITY;
                lse[u][2] = there ? x.z : -INFINITY;
                lse[u][3] = there ? x.w : -INFINITY;
#pragma unroll
                for (int r = 0; r < 4; r++) v[u][r] = __ldcg(reinterpret_cast<const float4*>(p.partO + (at + r) * D + c4 * 4));
              }
#pragma unroll
              for (int r = 0; r < 4; r++) {
                float top = M[r];
#pragma unroll
                for (int u = 0; u < kAhead; u++) top = fmaxf(top, lse[u][r]);
                const float ref = top == -INFINITY ? 0.f : top, f = ex2(M[r] - ref);
                M[r] = top;
                sum[r] *= f;
                acc[r] = make_float4(acc[r].x * f, acc[r].y * f, acc[r].z * f, acc[r].w * f);
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                  const float w = ex2(lse[u][r] - ref);  // NaN stays NaN
                  sum[r] += w;
                  acc[r].x = fmaf(w, v[u][r].x, acc[r].x);
                  acc[r].y = fmaf(w, v[u][r].y, acc[r].y);
                  acc[r].z = fmaf(w, v[u][r].z, acc[r].z);
                  acc[r].w = fmaf(w, v[u][r].w, acc[r].w);
                }
              }
            }
            if (c4 == 0) {
#pragma unroll
              for (int r = 0; r < 4; r++) {
                sM[group * 4 + r] = M[r];
                sL[group * 4 + r] = sum[r];
              }
            }
          }
          __syncthreads();
          float all[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            all[r] = sM[r];
#pragma unroll
            for (int i = 1; i < kGroups; i++) all[r] = fmaxf(all[r], sM[i * 4 + r]);
            if (all[r] == -INFINITY) all[r] = 0.f;
          }
#pragma unroll 1
          for (int i = 0; i < kGroups; i++) {  // (rows past nRows are rubbish that nobody reads)
            if (i == group) {
#pragma unroll
              for (int r = 0; r < 4; r++) {
                float4* at = reinterpret_cast<float4*>(sO + (r0 + r) * kLdO + c4 * 4);
                const float4 z = i == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
                const float f = ex2(M[r] - all[r]);
                *at = make_float4(fmaf(f, acc[r].x, z.x), fmaf(f, acc[r].y, z.y), fmaf(f, acc[r].z, z.z), fmaf(f, acc[r].w, z.w));
              }
            }
            __syncthreads();
          }
          for (int idx = threadIdx.x; idx < min(4, nRows - r0) * kVec; idx += kThreads) {
            const int r = idx / kVec, c = idx % kVec;
            float top = sM[r], total = 0.f;
#pragma unroll
            for (int i = 1; i < kGroups; i++) top = fmaxf(top, sM[i * 4 + r]);
            if (top == -INFINITY) top = 0.f;
#pragma unroll
            for (int i = 0; i < kGroups; i++) total += sL[i * 4 + r] * ex2(sM[i * 4 + r] - top);
            const float inv = total == 0.f ? 0.f : 1.f / total;
            const float4 x = *reinterpret_cast<const float4*>(sO + (r0 + r) * kLdO + c * 4);
            store(r0 + r, c, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
          }
          if (r0 + 4 < nRows) __syncthreads();  // sM and sL are written again
        }
      }
    }
    if (left == 0) break;
    next_segment(s, left);
    __syncthreads();  // the merge buffer is written again
  }
  cp_async_wait<0>();
}

template <int D, bool kInt8, bool kBf16, int NR>
int launch(const Params& p, int device, cudaStream_t stream) {
  constexpr int kSmem = ring_bytes<D, NR>() + merge_bytes<D, NR>();
  static_assert(kSmem <= 227 * 1024, "shared memory");
  auto kernel = cache_decode_kernel<D, kInt8, kBf16, NR>;
  static std::once_flag once[64];
  static cudaError_t attrErr[64];
  std::call_once(once[device], [&] {
    attrErr[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (attrErr[device] == cudaSuccess) {
      attrErr[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
  });
  if (attrErr[device] != cudaSuccess) {
    set_error_string("cudaFuncSetAttribute(%d bytes): %s", kSmem, cudaGetErrorString(attrErr[device]));
    return kCudaError;
  }
  const cudaError_t e = launch_kernel(kernel, dim3((unsigned)(p.runs * p.headsKV)), kThreads, kSmem, stream, may_overlap(stream), p);
  if (e != cudaSuccess) {
    set_error_string("cache attention kernel launch failed: %s", cudaGetErrorString(e));
    return kCudaError;
  }
  return kOk;
}

template <int D, int NR>
int launch_typed(const Params& p, bool int8, bool bf16, int device, cudaStream_t stream) {
  (void)p; (void)int8; (void)device; (void)stream;
  if (bf16) {
    if constexpr (TFA_HAVE_BF16) return int8 ? launch<D, true, true, NR>(p, device, stream) : launch<D, false, true, NR>(p, device, stream);
  } else {
    if constexpr (TFA_HAVE_FP16) return int8 ? launch<D, true, false, NR>(p, device, stream) : launch<D, false, false, NR>(p, device, stream);
  }
  return kBadDtype;
}

// Tiles of 8 query rows where no request has more, else of 16.
template <int D>
int launch_stream(Params& p, long long rows, int maxSeqLenKV, bool int8, bool bf16, int device, cudaStream_t stream) {
  const int nr = rows <= 8 ? 1 : 2;
  // as many runs as the GPU holds CTAs, and no more than there can be pairs of key blocks
  const long long slots = (long long)device_num_sms(device) * (nr == 1 ? ctas_per_sm<D, 1>() : ctas_per_sm<D, 2>());
  const long long tiles = (rows + 8 * nr - 1) / (8 * nr);
  const long long allTiles = ((long long)p.totalQ * p.group) / (8 * nr) + p.batch;  // of all requests, at most
  if (allTiles * ((((long long)p.width << p.blockShift) + kBlockKeys - 1) / kBlockKeys) > 0x7FFFFFFFll) {
    set_error_string("more than 2^31 - 1 tiles of query rows and 64 keys (%d rows of Q, block table for %lld tokens)", p.totalQ, (long long)p.width << p.blockShift);
    return kTooLarge;
  }
  const long long most = (tiles * ((maxSeqLenKV + kBlockKeys - 1) / kBlockKeys) * p.batch + 1) / 2;
  long long runs = slots / p.headsKV;
  if (runs > most) runs = most;
  if (runs < 1) runs = 1;
  p.runs = (int)runs;
  p.partO = p.partLse = nullptr;
  p.join = nullptr;
  void* scratch = nullptr;
  int rc = kOk;
  if (runs > 1) {
    p.join = device_join_counters(device, stream, &rc);
    if (p.join == nullptr) return rc;
    const size_t parts = (size_t)runs * p.headsKV * 2 * 8 * nr;
    rc = scratch_alloc(&scratch, parts * (D + 1) * sizeof(float), device, stream);
    if (rc != kOk) return rc;
    p.partO = static_cast<float*>(scratch);
    p.partLse = p.partO + parts * D;
  }
  rc = nr == 1 ? launch_typed<D, 1>(p, int8, bf16, device, stream) : launch_typed<D, 2>(p, int8, bf16, device, stream);
  if (scratch != nullptr) cudaFreeAsync(scratch, stream);
  return rc;
}

int dispatch_stream(Params& p, int headDim, long long rows, int maxSeqLenKV, bool int8, bool bf16, int device, cudaStream_t stream) {
  switch (headDim) {
#if TFA_HAVE_HD32
    case 32: return launch_stream<32>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
#if TFA_HAVE_HD64
    case 64: return launch_stream<64>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
#if TFA_HAVE_HD96
    case 96: return launch_stream<96>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
#if TFA_HAVE_HD128
    case 128: return launch_stream<128>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
#if TFA_HAVE_HD192
    case 192: return launch_stream<192>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
#if TFA_HAVE_HD256
    case 256: return launch_stream<256>(p, rows, maxSeqLenKV, int8, bf16, device, stream);
#endif
    default: return kBadHeadDim;
  }
}

// ------------------------------------------------------------------------------------------- many query rows: tensor cores
struct UnitParams {
  uint4* O;
  const int* cuQ;
  const int* lens;
  int batch, capacity, totalQ, group, causal, unitRows, rowChunks;
  int maxUnits;  // room for them: enough where cuQ does not decrease
  int* numUnits;
  int* unitBase;  // [batch + 1]
  long long* unitStart;
  int2* unitWhat;
};

// CTA 0: the units of a KV head (up to unitRows flat rows of a request each) and the key blocks ahead of each, by two prefix sums.  The
// others: zeros in the rows that no unit has, those of a request without tokens (CTA b + 1) and of no request (the last).
__global__ void __launch_bounds__(1024) cache_units_kernel(const UnitParams p) {
  __shared__ long long sWarp[32];
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  auto request = [&](int b, int& q0, int& nq, int& len) {
    q0 = min(max(p.cuQ[b], 0), p.totalQ);
    nq = min(max(p.cuQ[b + 1] - q0, 0), p.totalQ - q0);
    len = min(max(p.lens[b], 0), p.capacity);
  };
  if (blockIdx.x > 0) {
    const int b = (int)blockIdx.x - 1;
    auto zero = [&](int r0, int r1) {
      for (long long i = (long long)r0 * p.rowChunks + threadIdx.x; i < (long long)r1 * p.rowChunks; i += 1024) p.O[i] = make_uint4(0, 0, 0, 0);
    };
    if (b == p.batch) {
      zero(0, min(max(p.cuQ[0], 0), p.totalQ));
      zero(min(max(p.cuQ[p.batch], 0), p.totalQ), p.totalQ);
    } else {
      int q0, nq, len;
      request(b, q0, nq, len);
      if (len == 0) zero(q0, q0 + nq);
    }
    return;
  }
  long long units = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    int q0, nq = 0, len = 0;
    if (b < p.batch) request(b, q0, nq, len);
    const long long n = len > 0 ? ((long long)nq * p.group + p.unitRows - 1) / p.unitRows : 0;
    long long sum;
    const long long upto = cta_scan(n, sWarp, sum);
    if (b < p.batch) p.unitBase[b] = (int)min(units + upto - n, (long long)p.maxUnits);
    units += sum;
  }
  units = min(units, (long long)p.maxUnits);
  if (threadIdx.x == 0) {
    p.unitBase[p.batch] = (int)units;
    *p.numUnits = (int)units;
  }
  __syncthreads();
  long long blocks = 0;
  for (long long u0 = 0; u0 < units; u0 += 1024) {
    const long long u = u0 + threadIdx.x;
    long long n = 0;
    if (u < units) {
      int lo = 0, hi = p.batch - 1;  // the request b with unitBase[b] <= u < unitBase[b + 1]
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (u < p.unitBase[mid + 1]) {
          hi = mid;
        } else {
          lo = mid + 1;
        }
      }
      int q0, nq, len;
      request(lo, q0, nq, len);
      const int flat = (int)(u - p.unitBase[lo]) * p.unitRows;
      n = (len + tc::kBlockN - 1) / tc::kBlockN;
      if (p.causal) {
        const int last = (min(flat + p.unitRows, nq * p.group) - 1) / p.group;  // token of the unit's last row
        n = min(n, (long long)max(1, (len - nq + last + tc::kBlockN) / tc::kBlockN));
      }
      p.unitWhat[u] = make_int2(lo, flat);
    }
    long long sum;
    const long long upto = cta_scan(n, sWarp, sum);
    if (u < units) p.unitStart[u] = blocks + upto - n;
    blocks += sum;
  }
  if (threadIdx.x == 0) p.unitStart[units] = blocks;
}

// Units that several CTAs share: O = sum 2^(lse_c - M) O_c / sum 2^(lse_c - M) over their parts, which are [D / 4][128 rows] float4 each.  CTA
// (x, y): sixteen rows of every 128 of the unit that attention CTA x begins, 32 threads to a row; four parts in flight, relative to the
// largest log-sum-exp so far.  Bound by latency and the reads from L2; against the CTA that finishes a unit last doing it alone: one request of
// 16000 tokens, 64 rows a KV head, 8 heads of 128 (18 parts): 82 -> 44 us for the call; 2 heads of 256 (74 parts): 373 -> 58.
constexpr int kJoinRows = 16, kJoinThreads = 32 * kJoinRows, kJoinShares = tc::kBlockM / kJoinRows;
template <bool kBf16>
__global__ void __launch_bounds__(kJoinThreads) cache_join_kernel(const TcCacheJoin* joins, const float* partO, const float* partLse, uint16_t* O, int headsQ,
                                                                  int group, int headDim, int tiles) {
  ptx::grid_wait_previous();
  ptx::grid_allow_next();
  const int c0 = (int)blockIdx.x;
  const TcCacheJoin join = joins[c0];
  if (join.last < 0) return;
  const int r = (int)blockIdx.y * kJoinRows + threadIdx.x % kJoinRows, chunks = headDim / 4;
  for (int i = threadIdx.x / kJoinRows; i < tiles * chunks; i += 32) {
    const int t = i / chunks, c4 = i - t * chunks, flat = join.flat + t * tc::kBlockM + r;
    if (flat >= join.rows) break;
    constexpr int kAhead = 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, sum = 0.f;
    for (int c = c0; c <= join.last; c += kAhead) {
      float lse[kAhead];
      float4 x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const bool there = c + u <= join.last;
        const long long part = (2ll * (there ? c + u : c) + (c + u == c0 ? join.first : 0)) * tiles + t;
        const float v = __ldcg(partLse + part * tc::kBlockM + r);
        lse[u] = there ? v : -INFINITY;
        x[u] = __ldcg(reinterpret_cast<const float4*>(partO) + (part * chunks + c4) * tc::kBlockM + r);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < kAhead; u++) top = fmaxf(top, lse[u]);
      const float ref = top == -INFINITY ? 0.f : top, f = ex2(M - ref);
      M = top;
      sum *= f;
      acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const float w = ex2(lse[u] - ref);  // NaN stays NaN
        sum += w;
        if (w != 0.f) {  // (a part without a key is not written)
          acc.x = fmaf(w, x[u].x, acc.x);
          acc.y = fmaf(w, x[u].y, acc.y);
          acc.z = fmaf(w, x[u].z, acc.z);
          acc.w = fmaf(w, x[u].w, acc.w);
        }
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* dst = O + ((long long)(join.row0 + flat / group) * headsQ + join.head * group + flat % group) * headDim + c4 * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(tc::pack2<kBf16>(acc.x * inv, acc.y * inv), tc::pack2<kBf16>(acc.z * inv, acc.w * inv));
  }
}

int run_tc(const TcCacheParams& p, bool bf16, int ctas, bool overlap, int device, cudaStream_t s) {
  switch (p.headDim) {
#if TFA_HAVE_HDP64
    case 32:
    case 64: return cache_call_hdp64(p, bf16, ctas, overlap, device, s);
#endif
#if TFA_HAVE_HDP128
    case 96:
    case 128: return cache_call_hdp128(p, bf16, ctas, overlap, device, s);
#endif
#if TFA_HAVE_HDP192
    case 192: return cache_call_hdp192(p, bf16, ctas, overlap, device, s);
#endif
#if TFA_HAVE_HDP256
    case 256: return cache_call_hdp256(p, bf16, ctas, overlap, device, s);
#endif
    default: return kBadHeadDim;
  }
}

int dispatch_tc(const Params& d, int headDim, bool int8, bool bf16, int device, cudaStream_t s) {
  const int tiles = headDim <= 128 ? 2 : 1, unitRows = tiles * tc::kBlockM;
  const int ctas = device_num_sms(device);
  int rc = kOk;
  TcCacheParams p = {};
  const size_t maxUnits = (size_t)((long long)d.totalQ * d.group / unitRows) + d.batch;
  const size_t parts = (size_t)ctas * 2 * tiles * tc::kBlockM;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t oBytes = up(parts * headDim * sizeof(float)), lseBytes = up(parts * sizeof(float)), startBytes = up((maxUnits + 1) * sizeof(long long)),
               whatBytes = up((maxUnits + 1) * sizeof(int2)), baseBytes = up((size_t)(d.batch + 1) * sizeof(int)),
               joinBytes = up((size_t)ctas * sizeof(TcCacheJoin));
  void* scratch = nullptr;
  rc = scratch_alloc(&scratch, oBytes + lseBytes + startBytes + whatBytes + baseBytes + joinBytes + 256, device, s);
  if (rc != kOk) return rc;
  uint8_t* at = static_cast<uint8_t*>(scratch);
  p.partO = reinterpret_cast<float*>(at);
  p.partLse = reinterpret_cast<float*>(at += oBytes);
  long long* unitStart = reinterpret_cast<long long*>(at += lseBytes);
  int2* unitWhat = reinterpret_cast<int2*>(at += startBytes);
  int* unitBase = reinterpret_cast<int*>(at += whatBytes);
  p.joins = reinterpret_cast<TcCacheJoin*>(at += baseBytes);
  int* numUnits = reinterpret_cast<int*>(at += joinBytes);
  UnitParams u = {static_cast<uint4*>(d.O), d.cuQ, d.lens, d.batch, d.width << d.blockShift, d.totalQ, d.group, d.causal, unitRows, d.headsQ * headDim / 8,
                  (int)maxUnits, numUnits, unitBase, unitStart, unitWhat};
  const bool overlap = may_overlap(s);
  cudaError_t e = launch_kernel(cache_units_kernel, dim3((unsigned)d.batch + 2), 1024, 0, s, overlap, u);
  if (e != cudaSuccess) {
    set_error_string("cache unit kernel launch failed: %s", cudaGetErrorString(e));
    rc = kCudaError;
  }
  if (rc == kOk) {
    p.O = d.O;
    p.Q = d.Q;
    p.cuQ = d.cuQ;
    p.seqLenQ = d.totalQ;
    p.headsQ = d.headsQ;
    p.headsKV = d.headsKV;
    p.headDim = headDim;
    p.group = d.group;
    p.causal = d.causal;
    p.scaleLog2 = d.scaleLog2;
    p.status = device_status_word(device);
    p.epoch = next_epoch();
    p.cap = d.cap;
    p.slopes = d.slopes;
    p.codes[0] = d.kCodes, p.codes[1] = d.vCodes;
    p.scales[0] = d.kScales, p.scales[1] = d.vScales;
    p.table = d.table;
    p.lens = d.lens;
    p.width = d.width;
    p.numBlocks = d.numBlocks;
    p.blockShift = d.blockShift;
    p.int8 = int8 ? 1 : 0;
    p.numUnits = numUnits;
    p.unitStart = unitStart;
    p.unitWhat = unitWhat;
    rc = p.status == nullptr ? kCudaError : run_tc(p, bf16, ctas, overlap, device, s);
  }
  if (rc == kOk) {
    auto join = [&](auto kernel) {
      return launch_kernel(kernel, dim3((unsigned)ctas, kJoinShares), kJoinThreads, 0, s, overlap, p.joins, p.partO, p.partLse,
                           static_cast<uint16_t*>(d.O), d.headsQ, d.group, headDim, tiles);
    };
    e = bf16 ? join(cache_join_kernel<true>) : join(cache_join_kernel<false>);
    if (e != cudaSuccess) {
      set_error_string("cache join kernel launch failed: %s", cudaGetErrorString(e));
      rc = kCudaError;
    }
  }
  cudaFreeAsync(scratch, s);
  return rc;
}

}  // namespace cache
}  // namespace tfa_b200

using namespace tfa_b200;

extern "C" int tfa_b200_fwd_cache(const void* Q, void* O, const void* kCache, const void* vCache, const float* kScales, const float* vScales,
                                  const int* blockTable, const int* seqLens, const int* cuSeqLensQ, int dtype, int cacheType, int batchSize,
                                  int maxSeqLenQ, int maxSeqLenKV, long long totalQ, int numBlocks, int maxBlocks, int blockTokens, int numHeadsQ,
                                  int numHeadsKV, int headDim, int isCausal, float softcap, const float* alibiSlopes, void* stream) {
  using namespace cache;
  int rc = validate_common(Q, kCache, vCache, O, dtype, batchSize, maxSeqLenQ, maxSeqLenKV, numHeadsQ, numHeadsKV, headDim);
  if (rc != kOk) return rc;
  if (dtype == kFp32) {
    set_error_string("attention over an 8-bit cache takes fp16 and bf16 queries");
    return kBadDtype;
  }
  if (cacheType != TFA_B200_CACHE_INT8 && cacheType != TFA_B200_CACHE_E4M3) {
    set_error_string("unsupported cache type %d (1 = int8, 2 = e4m3)", cacheType);
    return kBadDtype;
  }
  int shift = 4;
  while (shift < 8 && (1 << shift) != blockTokens) shift++;
  if (shift == 8) {
    set_error_string("blocks hold 16, 32, 64 or 128 tokens (got %d)", blockTokens);
    return kBadArgument;
  }
  if (totalQ < 0 || numBlocks < 0 || maxBlocks < 0 || !(softcap >= 0.f) || isinf(softcap)) {
    set_error_string("negative size or softcap (totalQ=%lld numBlocks=%d maxBlocks=%d softcap=%g)", totalQ, numBlocks, maxBlocks, softcap);
    return kBadArgument;
  }
  if (totalQ == 0) return kOk;
  if (totalQ > 0x7FFFFFFFll || totalQ * numHeadsQ > 0x7FFFFFFFll || ((long long)maxBlocks << shift) > 0x7FFFFFFFll - kBlockKeys) {
    set_error_string("totalQ * numHeadsQ and maxBlocks * blockTokens must stay below 2^31");
    return kTooLarge;
  }
  if (cuSeqLensQ == nullptr || Q == nullptr || O == nullptr || (batchSize > 0 && (seqLens == nullptr || (maxBlocks > 0 && blockTable == nullptr))) ||
      (numBlocks > 0 && (kCache == nullptr || vCache == nullptr || kScales == nullptr || vScales == nullptr))) {
    set_error_string("null pointer");
    return kBadArgument;
  }
  if ((rc = check_device()) != kOk) return rc;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return kCudaError;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Params p;
  p.Q = Q;
  p.O = O;
  p.kCodes = static_cast<const uint8_t*>(kCache);
  p.vCodes = static_cast<const uint8_t*>(vCache);
  p.kScales = kScales;
  p.vScales = vScales;
  p.table = blockTable;
  p.lens = seqLens;
  p.cuQ = cuSeqLensQ;
  p.slopes = alibiSlopes;
  p.batch = batchSize;
  p.width = maxBlocks;
  p.numBlocks = numBlocks;
  p.blockShift = shift;
  p.headsQ = numHeadsQ;
  p.headsKV = numHeadsKV;
  p.group = numHeadsQ / numHeadsKV;
  p.causal = isCausal ? 1 : 0;
  p.totalQ = (int)totalQ;
  p.scaleLog2 = (float)(1.4426950408889634 / sqrt((double)headDim));
  p.cap = score::usable_cap(softcap);
  const bool int8 = cacheType == TFA_B200_CACHE_INT8, bf16 = dtype == kBf16;
  // Few query rows for a KV head: the stream kernel, whose time grows with every 16 of them; many: tensor-core tiles of 128, which cost the same for one
  // row as for all.  They meet near 64 rows.  us of stream / tensor form at 48, 64, 96 and 256 rows (8 KV heads of 128, e4m3): 4 x 4000 tokens
  // 40/42, 45/43, 56/44, 114/63; 16 x 2000 57/66, 73/68, 99/72, 228/106; 64 x 1000 113/140, 146/143, 207/152, 507/207; one of 16000 40/44, 46/44,
  // 57/45, 110/67; one of 1000 (launch and latency) 19/22, 19/22, 20/23, 24/32.  16 heads of 64, 16 x 2000: 66/84, 84/86, 116/89 at 96.
  const int tcOption = option_cache_tc();
  const long long rowsMost = (long long)maxSeqLenQ * p.group;  // query rows of a request that share a KV head
  if (tcOption > 0 || (tcOption < 0 && rowsMost > 4 * kRows)) return dispatch_tc(p, headDim, int8, bf16, device, s);
  return dispatch_stream(p, headDim, rowsMost > 0 ? rowsMost : 1, maxSeqLenKV, int8, bf16, device, s);
}
