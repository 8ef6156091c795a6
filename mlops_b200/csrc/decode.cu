// The routed layer for a few tokens (1 to 64), as a serving loop calls it: router logits, expert selection, up
// product with SwiGLU, down product with the weighted sum, residual and shared expert.
//
//   logits = x . bf16(router)^T                                          router_logits_kernel
//   (weights, ids) = the routing of route.cu
//   act[t,k] = bf16(silu(g) * u), [g | u] = x[t] . W13[e]^T              stream_kernel<UP>
//   y[t,k] = act[t,k] . W2[e]^T                                          stream_kernel<DOWN>
//   out[t] = residual[t] + sum_k w[t,k] y[t,k] (+ the shared expert's)   join_kernel
//
// Measured (calls one after the other, the bytes of the experts with tokens at 6.56 TB/s in brackets): one token of 8 of
// 128 experts, D = 2048, F = 768 36 us (6), 48 tokens 132 (89); one token of 8 of 256, D = 7168, F = 2048 with a shared
// expert 110 (68), 64 tokens 870 (720); 17 tokens of 2 of 8, D = 4096, F = 14336 267 (215).  The chain of six
// kernels takes 20 us however small the layer is.
//
// Bound: HBM.  The weights of the experts that got a token are read once, 3 D F bytes each in E4M3, for one
// or a few multiplications a byte; everything else is small.  So each product is one stream of weight rows
// through shared memory (boxes of 128 bytes of K, several stages of 32 KB in flight per SM), and the rows of all
// experts with tokens, one after the other, are cut evenly over the CTAs in groups of eight: with whole tiles of 64
// columns eight experts of F = 768 would leave 52 of 148 SMs idle.  Cutting the down product's output columns
// instead, which needs no y, left a CTA 14 to 24 rows of each expert: the tokens' columns then weigh as much as
// the weights'.
//
// The weights are the A operand of mma.sync.m16n8k16 (16 weight rows), the tokens the B operand (8 to a tile).
// Against bf16 weights the tokens are bf16.  E4M3 weights are widened to f16, one instruction for two values, and a
// token is f16 with a power of two of its own that puts its largest value in [2^14, 2^15): every bf16 value down to 2^-31
// of the largest exactly, what is smaller within 2^-39 of it (half of f16's smallest step, 2^-25, over 2^14).  The
// 128 x 128 block scales are applied in fp32 to the sums of one block, the tokens' powers of two to the finished sums.
// (Widening to bf16 takes four instructions for two values, 200 of the 356 issue slots an SM has per 2 KB of weights at
// full HBM rate; m16n8k32 on E4M3 operands widens them inside, again for every tile: 22 cycles against 8 of m16n8k16.)
//
// tcgen05 is not used: it has no product of E4M3 by 16-bit values, its tiles start at 64 rows, and at one to eight tokens
// a weight row the tensor rate is not what bounds this.  Sums are fp32; act is rounded to bf16 once, as the operand of the
// second product (the grouped layer rounds it likewise), and the output once.  Every sum has a fixed order: no
// atomics.
#include <atomic>

#include "common.cuh"
#include "host_util.h"
#include "../../include/b200moe.h"

namespace b200 {

constexpr int kDecodeThreads = 256;  // of the small kernels
constexpr int kDecodeWarps = 8;
constexpr int kMultiplyWarps = 16;    // of a stream
constexpr int kFillWarps = 4;         // of a stream: they keep its stages full
constexpr int kStreamThreads = 32 * (kMultiplyWarps + kFillWarps);
constexpr int kMaxTokens = 64;
constexpr int kSlab = 2048;           // 16 weight rows x 128 bytes of K
constexpr int kStageSlabs = 16;       // of a stage: row tiles x K blocks, one to a multiplying warp
constexpr int kStageA = kStageSlabs * kSlab;
constexpr int kTokenBytes = 256;      // a token's 128 columns beside an E4M3 block, and
constexpr int kTokenPitchBf16 = 192;  // its 64 beside a bf16 block: rows start in different banks
constexpr int kStageScales = 2 * kStageSlabs;  // of the weights: each slab's first and other eight rows
constexpr int kMaxStages = 8;
constexpr int kBlockColumns = 256;    // of y that the down product takes together (Stream)
constexpr int kPassTokens = 32;  // of one expert that a pass over its weights takes; rarely has an expert more

__device__ __forceinline__ void copy16(void* dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(read ? 16 : 0)
               : "memory");
}
// One arrival on `bar` (which counts it) when this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_from_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four E4M3 values as two pairs of f16 (exact).
__device__ __forceinline__ void widen(uint32_t w, uint32_t& first, uint32_t& second) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(first), "=r"(second)
      : "r"(w));
}

// A block scales a row of bf16 to f16 by the row's power of two (see the top), which it returns to thread 0.  Infinities
// and NaN stay what they are.  `width` is a multiple of 4; `largest` is scratch, one word per warp.
__device__ __forceinline__ float scale_row(const __nv_bfloat16* __restrict__ from, int width, __half* __restrict__ to,
                                           uint32_t* largest) {
  const uint2* in = reinterpret_cast<const uint2*>(from);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t m = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < width / 4; i += blockDim.x) {
    const uint2 raw = in[i];
    m = __vmaxu2(m, __vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu));
  }
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  if (lane == 0) largest[warp] = m;
  __syncthreads();
  m = __reduce_max_sync(0xffffffffu, lane < blockDim.x / 32 ? largest[lane] : 0u);
  // exponent of the largest, kept where both powers of two are normal numbers
  const int e = min(max((int)(m >> 7), 27), 254);
  const float inverse = __int_as_float((268 - e) << 23);  // largest / s in [2^14, 2^15)
#pragma unroll 4
  for (int i = threadIdx.x; i < width / 4; i += blockDim.x) {
    const uint2 raw = in[i];
    const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const float2 a = __bfloat1622float2(pairs[0]), b = __bfloat1622float2(pairs[1]);
    const __half2 first = __floats2half2_rn(a.x * inverse, a.y * inverse);
    const __half2 second = __floats2half2_rn(b.x * inverse, b.y * inverse);
    reinterpret_cast<uint2*>(to)[i] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&first), *reinterpret_cast<const uint32_t*>(&second));
  }
  return __int_as_float((e - 14) << 23);
}

// ---------------------------------------------------------------------------------------------
// Router logits, fp32 [T, E]: 16 experts per cluster of eight CTAs, which split the hidden width between
// them and their warps; partial sums meet in shared memory, then across the cluster, in a fixed order.
// Lane (g, t) of a warp owns 16 consecutive columns of a 64-column step (the order of the columns inside a sum is
// free as long as both operands agree).
// ---------------------------------------------------------------------------------------------
constexpr int kRouterCluster = 8;

template <typename W>
__device__ __forceinline__ void load_router(const W* row, int k, int width, bool valid, uint32_t (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // widths are multiples of 8
    uint4 o = make_uint4(0, 0, 0, 0);
    if (valid && k + 8 * h < width) {
      if constexpr (sizeof(W) == 2) {
        o = *reinterpret_cast<const uint4*>(row + k + 8 * h);
      } else {
        const float4 a = *reinterpret_cast<const float4*>(row + k + 8 * h);
        const float4 b = *reinterpret_cast<const float4*>(row + k + 8 * h + 4);
        o = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
      }
    }
    v[4 * h] = o.x, v[4 * h + 1] = o.y, v[4 * h + 2] = o.z, v[4 * h + 3] = o.w;
  }
}

template <typename W, int NT>
__global__ void __launch_bounds__(kDecodeThreads)
router_logits_kernel(const __nv_bfloat16* __restrict__ x, const W* __restrict__ router, int T, int E, int width,
                     float* __restrict__ logits, __half* __restrict__ x16, float* __restrict__ x16_scale) {
  __shared__ float partial[kDecodeWarps][NT * 8][16];
  __shared__ float sums[NT * 8][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)cluster_ctarank();
  dependency_release();
  const int routers = (E + 15) / 16 * kRouterCluster;
  if ((int)blockIdx.x >= routers) {  // the clusters behind the router's scale the tokens for the E4M3 products
    const int token = (int)blockIdx.x - routers;
    if (token >= T) return;
    const float scale = scale_row(x + (long long)token * width, width, x16 + (long long)token * width,
                                  reinterpret_cast<uint32_t*>(&sums[0][0]));
    if (threadIdx.x == 0) x16_scale[token] = scale;
    return;
  }
  const int e0 = (blockIdx.x / kRouterCluster) * 16;
  const W* lo = router + (long long)(e0 + g) * width;
  const W* hi = lo + 8LL * width;
  const bool has_lo = e0 + g < E, has_hi = e0 + g + 8 < E;
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  const int steps = (width + 63) / 64;
#pragma unroll 2
  for (int s = rank * kDecodeWarps + warp; s < steps; s += kRouterCluster * kDecodeWarps) {
    const int k = s * 64 + t * 16;
    uint32_t a[8], b[8];
    load_router(lo, k, width, has_lo, a);
    load_router(hi, k, width, has_hi, b);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      uint32_t v[8];
      load_router(x + (long long)(i * 8 + g) * width, k, width, i * 8 + g < T, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_bf16(acc[i], a[2 * j], b[2 * j], a[2 * j + 1], b[2 * j + 1], v[2 * j], v[2 * j + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    partial[warp][i * 8 + 2 * t][g] = acc[i][0];
    partial[warp][i * 8 + 2 * t + 1][g] = acc[i][1];
    partial[warp][i * 8 + 2 * t][g + 8] = acc[i][2];
    partial[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 128; i += kDecodeThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) v += partial[w][i >> 4][i & 15];
    sums[i >> 4][i & 15] = v;
  }
  cluster_sync_all();
  for (int i = rank * kDecodeThreads + threadIdx.x; i < NT * 128; i += kRouterCluster * kDecodeThreads) {
    const uint32_t mine = smem_u32(&sums[i >> 4][i & 15]);
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kRouterCluster; ++c) {
      uint32_t remote;
      float part;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(mine), "r"(c));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(remote) : "memory");
      v += part;
    }
    const int token = i >> 4, e = e0 + (i & 15);
    if (token < T && e < E) logits[(long long)token * E + e] = v;
  }
  cluster_sync_all();  // nobody leaves while its sums are being read
}

// ---------------------------------------------------------------------------------------------
// The two products
// ---------------------------------------------------------------------------------------------
struct DecodeParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* residual;
  const int* ids;
  const float* route_weights;
  const uint8_t* w2;  // E4M3 or bf16; the products read the weights through tensor maps, this is for prefetch_down
  const float *w13_scale, *w2_scale;
  const __half* x16;                      // x against E4M3 weights: [T, D], and
  const float* x16_scale;                 // its powers of two
  __nv_bfloat16* act;                     // [T * K, F] in expert order
  __nv_bfloat16* act_shared;              // [T, shared_inner]
  __half* act16;                          // act against E4M3 weights: [T * K, F]
  float* act16_scale;
  float* y;                               // [T * K (+ T), D] in expert order, the shared expert's last
  int* row_of;                            // [T * K] row of each assignment
  __nv_bfloat16* out;
  int T, D, F, E, K, shared_inner;
  int fp8, limited;
  float limit;
  int b_rows;  // capacity of a stage's token part, in rows of one K block
  int* status;
#ifdef B200_WAIT_TEST
  int withhold, withheld;  // test builds only: in product 1 (UP) or 2 (DOWN) fill warp `withheld` sends nothing
#endif
};

// Weight rows as [experts * rows, K], read in boxes of 128 bytes of K by 8, 32 or all rows of a full piece (UP: 128, DOWN:
// 256).  (A box takes the copy unit 50 cycles, 8 rows of it as much as 32: by eights alone the down product of F = 14336
// ran at 4.8 TB/s.)
struct WeightMaps {
  CUtensorMap tall, middle, flat;
};
struct DecodeMaps {
  WeightMaps routed, shared;
};
// Weights are read once: they go through L2 as the first to leave it, so that the kernels' own instructions, the tokens and
// the lists stay (a call that streamed 448 MB fetched its instructions from HBM again).
__device__ __forceinline__ uint64_t read_once() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void load_box(void* to, const CUtensorMap* map, uint64_t* full, int x, int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(to)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(full)), "r"(x), "r"(y), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void load_rows(uint8_t* to, const WeightMaps& maps, uint64_t* full, int x, int y, int count,
                                          uint64_t policy) {
  int row = 0;
  for (; row + 32 <= count; row += 32) load_box(to + row * 128, &maps.middle, full, x, y + row, policy);
  for (; row < count; row += 8) load_box(to + row * 128, &maps.flat, full, x, y + row, policy);
}

// A place in the stream: group of eight columns of an expert, in a block of the down product's columns.
struct Place {
  int block, index, group;
};
struct Part {  // a CTA's
  Place from, to;
};

// Where things are in shared memory behind the stages.
struct Lists {
  Part part, down;    // this CTA's of this stream; UP: and of the down product's
  unsigned long long* totals;  // [warps]
  int* begin;         // [experts with tokens + 1] first row of each
  float* scale;       // [T * K] UP, E4M3: the power of two of each row's token
  uint32_t* mask;     // [E][2] the tokens of each expert
  uint16_t* expert;   // [experts with tokens]
  uint16_t* first;    // [E] first row of each
  uint8_t* tokens;    // [T * K]
  __host__ __device__ static int bytes(int T, int E, int K) {
    const int R = T * K, most = E < R ? E : R;
    return 8 * (kStreamThreads / 32) + 4 * (most + 1) + 4 * R + 8 * E + 2 * (most + E) + R;
  }
  __device__ void place(uint8_t* base, int T, int E, int K) {
    const int R = T * K, most = E < R ? E : R;
    totals = reinterpret_cast<unsigned long long*>(base);
    begin = reinterpret_cast<int*>(totals + kStreamThreads / 32);
    scale = reinterpret_cast<float*>(begin + most + 1);
    mask = reinterpret_cast<uint32_t*>(scale + R);
    expert = reinterpret_cast<uint16_t*>(mask + 2 * E);
    first = expert + most;
    tokens = reinterpret_cast<uint8_t*>(first + E);
  }
};

// What eight columns of an expert with n tokens cost in the stream.  Measured with 16 experts of F = 2048, D = 7168 that all
// have n tokens, E4M3 (us without the 35 that no column costs): n <= 8 120, 16 160, 24 220, 32 240, 40 350, 64 470.
// bf16 weights are twice the bytes and as many products.  (64 tokens of E = 256: with columns that all counted alike the
// CTAs of the up product were ready after 510 to 838 us, those of the experts with most tokens last.)
__device__ __forceinline__ int weight_of(int n, bool fp8) {
  const int rest = (n % kPassTokens + 7) / 8;  // groups of eight tokens of the last pass
  return n / kPassTokens * (fp8 ? 5 : 6) + (rest == 0 ? 0 : fp8 ? 1 + rest : max(2 + rest, 4));
}
// ... of the shared expert: bf16, and in the down product with another K.
template <bool DOWN>
__device__ __forceinline__ int shared_weight(const DecodeParams& p) {
  if (p.shared_inner == 0) return 0;
  const int weight = weight_of(p.T, false);
  return !DOWN ? weight : min(max((int)(((long long)p.shared_inner * weight + p.F / 2) / p.F), 1), 512);
}

// The columns are cut between the CTAs by weight, in whole groups of eight, what the lowest box of weights holds: a flat
// position counts such groups times their weight.  The two ends of this CTA's part:
template <bool DOWN>
struct Cut {
  int routed, shared;  // weights
  int block[2], flat[2], groups[2];
  __device__ __forceinline__ Cut(const DecodeParams& p, int all_routed)
      : routed(all_routed), shared(shared_weight<DOWN>(p)) {
    const unsigned total =  // < 2^31: weights add up to less than 2^13, groups are at most 2^16
        DOWN ? (routed + shared) * (p.D / 8) : routed * (p.F / 8) + shared * (p.shared_inner / 8);
    const unsigned each = total / gridDim.x, rest = total - each * gridDim.x;
    const int size = kBlockColumns / 8 * (routed + shared);  // of a whole block
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // total * (block + i) / blocks, without a division of 64 bits
      const unsigned b = blockIdx.x + i;
      flat[i] = (int)(each * b + rest * b / gridDim.x);
      block[i] = DOWN ? flat[i] / size : 0;
      flat[i] -= block[i] * size;
      groups[i] = (DOWN ? min(kBlockColumns, p.D - block[i] * kBlockColumns) : p.F) / 8;
    }
  }
  // an end in the shared expert, or behind the last of all
  __device__ __forceinline__ void last(Part& part, int active) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int in = flat[i] - routed * groups[i];
      if (in >= 0)
        (i == 0 ? part.from : part.to) = shared ? Place{block[i], active, (in + shared - 1) / shared}
                                                : Place{block[i], active - 1, groups[i]};
    }
  }
  // an end in the expert in place `index`
  __device__ __forceinline__ void within(Part& part, int index, int before, int weight) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int in = flat[i] - before * groups[i];
      if (in >= 0 && in < weight * groups[i])
        (i == 0 ? part.from : part.to) = Place{block[i], index, (in + weight - 1) / weight};
    }
  }
};

// Rows by expert, in token order inside one, and this CTA's part of the stream; returns the number of experts with tokens.
// A token has an expert at most once, so an expert's tokens are a mask of 64 bits and a row's place in them a count of
// bits: nothing is serial.  (One warp that ranked 32 assignments at a time took 5 us longer for 48 tokens of 8.)
// Nothing is divided while the stream is walked either: its ends are found here.
template <bool DOWN>
__device__ __forceinline__ int build_lists(Lists& l, const DecodeParams& p, int* __restrict__ row_of,
                                           const float* __restrict__ token_scale) {
  const int* __restrict__ ids = p.ids;
  const int T = p.T, E = p.E, K = p.K;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = T * K;
  for (int e = tid; e < 2 * E; e += kStreamThreads) l.mask[e] = 0;
  __syncthreads();
  for (int i = tid; i < R; i += kStreamThreads) {
    const int token = i / K;
    atomicOr(l.mask + 2 * ids[i] + (token >> 5), 1u << (token & 31));
  }
  __syncthreads();
  // exclusive sums over the experts of (weight, experts with rows, rows), packed in one word
  const int per = (E + kStreamThreads - 1) / kStreamThreads;
  const auto rows = [&](int e) { return e < E ? __popc(l.mask[2 * e]) + __popc(l.mask[2 * e + 1]) : 0; };
  const auto packed = [&](int n) {
    return n ? (unsigned long long)weight_of(n, p.fp8) << 32 | 1ull << 16 | (unsigned long long)n : 0ull;
  };
  unsigned long long mine = 0;
  for (int j = 0; j < per; ++j) mine += packed(rows(tid * per + j));
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) l.totals[warp] = incl;
  __syncthreads();
  unsigned long long at = incl - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kStreamThreads / 32; ++w) {
    const unsigned long long n = l.totals[w];
    if (w < warp) at += n;
    all += n;
  }
  const int active = (int)(all >> 16) & 0xffff;
  const int routed = (int)(all >> 32);
  const Cut<DOWN> cut(p, routed);
  const Cut<true> down(p, routed);
  if (tid == 0) {
    cut.last(l.part, active);
    if (!DOWN) down.last(l.down, active);
  }
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j, n = rows(e);
    if (n) {
      const int place = (int)(at >> 16) & 0xffff, before = (int)(at >> 32), weight = weight_of(n, p.fp8);
      l.first[e] = (uint16_t)at;
      l.expert[place] = (uint16_t)e;
      l.begin[place] = (int)at & 0xffff;
      at += packed(n);
      cut.within(l.part, place, before, weight);
      if (!DOWN) down.within(l.down, place, before, weight);
    }
  }
  if (tid == 0) l.begin[active] = R;
  __syncthreads();
  for (int i = tid; i < R; i += kStreamThreads) {
    const int token = i / K, e = ids[i];
    const uint32_t low = l.mask[2 * e], high = l.mask[2 * e + 1], below = (1u << (token & 31)) - 1;
    const int at_row = l.first[e] + (token < 32 ? __popc(low & below) : __popc(low) + __popc(high & below));
    if (row_of != nullptr) row_of[i] = at_row;
    l.tokens[at_row] = (uint8_t)token;
    if (token_scale != nullptr) l.scale[at_row] = token_scale[token];
  }
  __syncthreads();
  return active;
}

// A piece of the stream: consecutive output columns of one expert (UP: of the activation, gate and up rows alike; DOWN:
// of y), at most 128 or 256, and at most kPassTokens of its tokens.  Its rows are cut into 1 << rt_log tiles of 16; a
// stage has 1 << ks_log K blocks of them.  Slab (K block << rt_log) + tile belongs to the warp of that number.
struct Piece {
  int index;         // expert with tokens, or `active` for the shared expert
  int first, count;  // output columns
  int n, begin;      // tokens, and the first of their rows
  int rt_log, ks_log;
  int steps, blocks;  // stages, K blocks
  bool fp8;
};

// Their order: UP expert by expert, the shared one last; DOWN the same within each kBlockColumns columns of y (a block).
template <bool DOWN>
struct Stream {
  const DecodeParams& p;
  const Lists& l;
  const int active;
  const int last;          // experts of a block
  Place at;
  const Place& to;
  int waiting;             // tokens of the current expert that need another pass over the same weights
  Piece piece;

  __device__ Stream(const DecodeParams& params, const Lists& lists, const Part& part, int n_active)
      : p(params), l(lists), active(n_active), last(n_active + (params.shared_inner > 0)), at(part.from), to(part.to),
        waiting(0) {}
  __device__ bool next() {
    if (waiting > 0) {
      piece.begin += piece.n;
    } else if (!next_columns()) {
      return false;
    }
    piece.n = min(waiting, kPassTokens);
    waiting -= piece.n;
    piece.ks_log = 0;
    while (piece.ks_log + piece.rt_log < 4 && (2 << piece.ks_log) * piece.n <= p.b_rows) ++piece.ks_log;
    piece.steps = (piece.blocks + (1 << piece.ks_log) - 1) >> piece.ks_log;
    return true;
  }
  // Of `left` columns those of a piece: half of `most`, twice the K blocks to a stage, where all of them would leave more
  // than a quarter of the stages empty.  Not where the tokens of two K blocks are more than a stage has room for.
  __device__ int fill(int left, int most) const {
    const bool twice = 2 * min(waiting, kPassTokens) <= p.b_rows;
    return twice && left > most / 2 && left < most * 3 / 4 ? most / 2 : min(left, most);
  }
  __device__ bool next_columns() {
    int columns;
    for (;; at.group = 0) {
      const bool ends = at.block == to.block && at.index == to.index;
      const int width = DOWN                 ? min(kBlockColumns, p.D - at.block * kBlockColumns)
                        : at.index == active ? p.shared_inner
                                             : p.F;
      columns = (ends ? to.group * 8 : width) - at.group * 8;
      if (columns > 0) break;
      if (ends || at.block * kBlockColumns >= p.D) return false;
      if (++at.index == last) at.index = 0, ++at.block;
    }
    const bool shared = at.index == active;
    piece.index = at.index;
    piece.first = at.block * kBlockColumns + at.group * 8;
    piece.fp8 = p.fp8 && !shared;
    piece.begin = shared ? 0 : l.begin[at.index];
    waiting = shared ? p.T : l.begin[at.index + 1] - piece.begin;
    piece.count = fill(columns, DOWN ? 256 : 128);
    at.group += piece.count / 8;
    const int tiles = DOWN ? (piece.count + 15) / 16 : (piece.count + 7) / 8;
    piece.rt_log = tiles <= 1 ? 0 : 32 - __clz(tiles - 1);
    piece.blocks = (inner() * (piece.fp8 ? 1 : 2) + 127) / 128;
    return true;
  }
  __device__ int inner() const { return !DOWN ? p.D : piece.index == active ? p.shared_inner : p.F; }
};

// Where the K slices of a tile meet: a value of every lane for each of at most 16 tokens (a pass of more has one slice).
__host__ __device__ inline int meet_bytes(int T) { return kMultiplyWarps * 32 * 4 * (T <= 8 ? 4 : 8); }

struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];
  int abort;
};

// Asks for the first rows this CTA's part of the down product will read: HBM would idle while the last sums of the up
// product are formed, act is scaled and the next kernel starts.
constexpr long long kPrefetchBytes = 256 << 10;
__device__ __forceinline__ void prefetch_down(const DecodeParams& p, const Lists& l, int active) {
  Stream<true> now(p, l, l.down, active);
  const long long pitch = (long long)p.F * (p.fp8 ? 1 : 2);
  for (long long left = kPrefetchBytes; left > 0 && now.next();) {
    const int e = now.piece.index;
    if (e == active || now.piece.begin > l.begin[e]) continue;  // (the shared expert; another pass over the same rows)
    const uint8_t* from = p.w2 + ((long long)l.expert[e] * p.D + now.piece.first) * pitch;
    const long long bytes = min(left, now.piece.count * pitch);
    for (long long at = 0; at < bytes; at += 16384)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from + at), "r"((uint32_t)min(16384LL, bytes - at))
                   : "memory");
    left -= bytes;
  }
}

// A stage's weights: [K block][row], UP: the piece's gate rows, then its up rows, in whole tiles; rows of 128 bytes.
// Its tokens: [K block][token].  Beside E4M3 weights two scales for each slab.  Fill
// warp w has stages w, w + 4, ...: its first lane sends for the boxes, all its lanes bring the scales and the tokens'
// columns.  There are at least as many stages as fill warps: a warp that fills stage s has filled s - 4, so
// s - 4 - count has been read and a wait for s - count cannot take the phase before that one for it.
// Where a wait runs out: a multiplying warp that has not seen a stage filled no longer says that it has read one, so no
// slot with copies on their way is filled again (the wait for it ends by the abort flag); and a fill warp leaves, then as
// always, when its own copies have landed or a bounded wait for them has run out.
template <bool DOWN, int MOST>
__device__ __forceinline__ void keep_full(const DecodeParams& p, const DecodeMaps& maps, const Lists& l, int active,
                                          uint8_t* stages, uint8_t* token_stages, float* weight_scales,
                                          int count, Barriers& bars) {
  const int lane = threadIdx.x & 31, turn = (threadIdx.x >> 5) - kMultiplyWarps;
  Stream<DOWN> now(p, l, l.part, active);
  const uint64_t policy = read_once();
  int slot = 0, stage = 0;
  uint32_t phase = 0;
  bool dead = false;
  while (!dead && now.next()) {
    const Piece& piece = now.piece;
    const bool shared = piece.index == active;
    const WeightMaps& weights = shared ? maps.shared : maps.routed;
    const int inner = now.inner(), ks_count = 1 << piece.ks_log;
    const int columns = piece.fp8 ? 128 : 64;  // of a K block
    const int up = shared ? p.shared_inner : p.F;
    const int y = (shared ? 0 : l.expert[piece.index] * (DOWN ? p.D : 2 * p.F)) + piece.first;
    const int block_bytes = kSlab << piece.rt_log;
    const __nv_bfloat16* tokens = !DOWN ? p.x : (shared ? p.act_shared : p.act) + (long long)piece.begin * inner;
    // Beside E4M3 weights a lane has 16 bytes of every other row of the tokens, at the same places of every stage.  Where a
    // call can have many rows they are found once: 16 experts with 16 tokens each 192 us instead of 216, with 8 tokens 154
    // instead of 164.  For the one to eight tokens of a small call that is more than it saves (36.8 us instead of 36.2).
    const uint8_t* tokens16 = reinterpret_cast<const uint8_t*>(DOWN ? p.act16 + (long long)piece.begin * inner : p.x16);
    uint32_t offset[kPassTokens / 2];
    bool placed = false;
    // a lane has the scale of half `lane & 1` of slab `lane >> 1`
    const float* scale = nullptr;
    const int scale_ks = lane >> (1 + piece.rt_log);
    if (piece.fp8) {
      const int rt = (lane >> 1) & ((1 << piece.rt_log) - 1), rows = DOWN ? p.D : p.F;
      const int column = min(piece.first + rt * (DOWN ? 16 : 8) + (DOWN ? (lane & 1) * 8 : 0), rows - 1);
      const int row = column + (DOWN ? 0 : (lane & 1) * p.F);
      scale = (DOWN ? p.w2_scale : p.w13_scale) +
              ((long long)l.expert[piece.index] * ((DOWN ? p.D : 2 * p.F) >> 7) + (row >> 7)) * piece.blocks + scale_ks;
    }
    for (int step = 0; step < piece.steps; ++step, ++stage) {
#ifdef B200_WAIT_TEST
      const bool sends = p.withhold != (DOWN ? 2 : 1) || turn != p.withheld;
#else
      constexpr bool sends = true;
#endif
      if (sends && (stage & (kFillWarps - 1)) == turn) {
        const int block0 = step << piece.ks_log, here = min(ks_count, piece.blocks - block0);  // K blocks of this stage
        const int rows = here * piece.n;
        if (stage >= count && !mbar_wait_warp(&bars.empty[slot], phase ^ 1, &bars.abort, p.status, 70)) {
          dead = true;
          break;
        }
        if (scale != nullptr && scale_ks < here) copy4(weight_scales + slot * kStageScales + lane, scale + block0);
        uint64_t* full = &bars.full[slot];
        if (lane == 0) {
          uint8_t* to = stages + slot * kStageA;
          mbar_arrive_expect_tx(full, here * piece.count * (DOWN ? 128 : 256));
          for (int ks = 0; ks < here; ++ks, to += block_bytes) {
            const int x = (block0 + ks) * columns;
            if (piece.count == (DOWN ? 256 : 128)) {
              load_box(to, &weights.tall, full, x, y, policy);
              if (!DOWN) load_box(to + 16384, &weights.tall, full, x, y + up, policy);
            } else {
              load_rows(to, weights, full, x, y, piece.count, policy);
              if (!DOWN) load_rows(to + block_bytes / 2, weights, full, x, y + up, piece.count, policy);
            }
          }
        }
        __syncwarp();
        if (DOWN && stage < kFillWarps) dependency_wait();  // the first weights are on their way, act must be there
        uint8_t* b = token_stages + slot * p.b_rows * kTokenBytes;
        if (!piece.fp8) {
          for (int i = lane; i < rows * 8; i += 32) {
            const int at = i >> 3, ks = here == 1 ? 0 : at / piece.n, row = at - ks * piece.n;
            const int token = DOWN ? row : shared ? piece.begin + row : l.tokens[piece.begin + row];
            const int k = (block0 + ks) * 64 + (i & 7) * 8;  // behind the end of a row: zeros, as the boxes have
            copy16(b + at * kTokenPitchBf16 + (i & 7) * 16, tokens + (long long)token * inner + (k < inner ? k : 0),
                   k < inner);
          }
        } else {
          const uint8_t* from = tokens16 + (long long)block0 * 256;
          uint8_t* to = b + (lane >> 4) * kTokenBytes + (((lane & 15) ^ (lane >> 4)) << 4);
          const auto place = [&](int at) {  // in bytes from `from`
            const int ks = MOST == 1 && ks_count == 1 ? 0 : min(at / piece.n, ks_count - 1);
            const int row = min(at - ks * piece.n, piece.n - 1);
            return 2 * ((DOWN ? row : l.tokens[piece.begin + row]) * inner + ks * 128 + (lane & 15) * 8);
          };
          if (MOST == 1) {
            for (int at = lane >> 4; at < rows; at += 2, to += 2 * kTokenBytes) copy16(to, from + place(at), true);
          } else {
            if (!placed) {  // (the first weights are on their way)
              placed = true;
#pragma unroll
              for (int j = 0; j < kPassTokens / 2; ++j) {
                if (2 * j >= piece.n << piece.ks_log) break;
                offset[j] = place(2 * j + (lane >> 4));
              }
            }
#pragma unroll
            for (int j = 0; j < kPassTokens / 2; ++j) {
              if (2 * j >= rows) break;
              if (2 * j + (lane >> 4) < rows) copy16(to + j * 2 * kTokenBytes, from + offset[j], true);
            }
          }
        }
        copies_arrive(full);
      }
      if (++slot == count) {
        slot = 0;
        phase ^= 1;
      }
    }
  }
  if (!DOWN && turn == 0 && lane == 0) prefetch_down(p, l, active);
  // the latest fill of each slot; earlier ones have been read, or the loop has ended in front of them
  volatile int go_on = 0;
  for (int i = 1; i <= min(stage, count); ++i) {
    slot = slot == 0 ? count - 1 : slot - 1;
    if (slot == count - 1) phase ^= 1;
    if (((stage - i) & (kFillWarps - 1)) == turn && lane == 0) mbar_wait(&bars.full[slot], phase, &go_on, p.status, 71);
  }
  __syncwarp();
}

// One warp's slab of a stage: 16 weight rows x 128 bytes of K by up to 8 * MOST tokens.  Lane (g, t) reads the same
// 16 (bf16: 8) consecutive columns of its weight rows and of its token, which is one order of the columns for both
// operands.  Rows behind the last token are read as that token's; their sums go nowhere.
// Weight rows j and j + 4 of a box go to neighbouring lanes: under the 128-byte swizzle they lie in different banks.
__device__ __forceinline__ int box_row(int g) { return (g >> 1) + ((g & 1) << 2); }

__device__ __forceinline__ uint4 load16(uint32_t shared_address) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(shared_address));
  return v;
}

// The widened slab by GROUPS tiles of eight tokens.
template <int GROUPS>
__device__ __forceinline__ void multiply_groups(const uint32_t (&a)[8][4], float2 s, uint32_t b_at, const uint32_t* token,
                                                float* acc) {
  float c[GROUPS][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 v[GROUPS];
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) v[h] = load16(((b_at + token[h]) ^ ((q & 1) << 4)) + (q >> 1) * 128);
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) {
      if (q == 0)
        mma_f16_from_zero(c[h], a[0], v[h].x, v[h].y);
      else
        mma_f16(c[h], a[2 * q], v[h].x, v[h].y);
    }
#pragma unroll
    for (int h = 0; h < GROUPS; ++h) mma_f16(c[h], a[2 * q + 1], v[h].z, v[h].w);
  }
#pragma unroll
  for (int h = 0; h < GROUPS; ++h) {
    acc[4 * h] = fmaf(c[h][0], s.x, acc[4 * h]);
    acc[4 * h + 1] = fmaf(c[h][1], s.x, acc[4 * h + 1]);
    acc[4 * h + 2] = fmaf(c[h][2], s.y, acc[4 * h + 2]);
    acc[4 * h + 3] = fmaf(c[h][3], s.y, acc[4 * h + 3]);
  }
}

// `a`: this lane's first 16 bytes of the slab, the other eight rows `high` bytes further; `b` + token[i]: its first 16 bytes
// of tile i of the tokens.  acc[4 i + h], acc[4 i + 2 + h] are the sums of token 8 i + 2 t + h for the lane's two weight
// rows.
template <int MOST>
__device__ __forceinline__ void multiply_e4m3(uint32_t a_at, int high, float2 s, uint32_t b_at,
                                              const uint32_t (&token)[MOST], int n, float (&acc)[MOST * 4]) {
  uint32_t a[8][4];
#pragma unroll
  for (int segment = 0; segment < 2; ++segment) {
    const uint4 lo = load16(a_at ^ (segment * 64)), hi = load16((a_at ^ (segment * 64)) + high);
    const int j = segment * 4;
    widen(lo.x, a[j][0], a[j][2]), widen(hi.x, a[j][1], a[j][3]);
    widen(lo.y, a[j + 1][0], a[j + 1][2]), widen(hi.y, a[j + 1][1], a[j + 1][3]);
    widen(lo.z, a[j + 2][0], a[j + 2][2]), widen(hi.z, a[j + 2][1], a[j + 2][3]);
    widen(lo.w, a[j + 3][0], a[j + 3][2]), widen(hi.w, a[j + 3][1], a[j + 3][3]);
  }
  // two groups of tokens at a time where there are two: their sums do not wait for one another
  if (MOST == 1 || n <= 8) {
    multiply_groups<1>(a, s, b_at, &token[0], &acc[0]);
  } else {
    multiply_groups<2>(a, s, b_at, &token[0], &acc[0]);
    if (n > 24)
      multiply_groups<2>(a, s, b_at, &token[MOST / 2], &acc[4 * (MOST / 2)]);
    else if (n > 16)
      multiply_groups<1>(a, s, b_at, &token[MOST / 2], &acc[4 * (MOST / 2)]);
  }
}

// The same on bf16 weights.
template <int MOST>
__device__ __forceinline__ void multiply_bf16(uint32_t a_at, int high, uint32_t b_at, const uint32_t (&token)[MOST], int n,
                                              float (&acc)[MOST * 4]) {
  const uint4 l0 = load16(a_at), h0 = load16(a_at + high), l1 = load16(a_at ^ 64), h1 = load16((a_at ^ 64) + high);
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    if (i * 8 < n) {
      const uint4 v0 = load16(b_at + token[i]), v1 = load16(b_at + token[i] + 64);
      float(&c)[4] = *reinterpret_cast<float(*)[4]>(&acc[4 * i]);
      mma_bf16(c, l0.x, h0.x, l0.y, h0.y, v0.x, v0.y);
      mma_bf16(c, l0.z, h0.z, l0.w, h0.w, v0.z, v0.w);
      mma_bf16(c, l1.x, h1.x, l1.y, h1.y, v1.x, v1.y);
      mma_bf16(c, l1.z, h1.z, l1.w, h1.w, v1.z, v1.w);
    }
  }
}

__device__ __forceinline__ float gated(float gate, float up, int limited, float limit) {
  if (limited) {
    gate = min_or_nan(gate, limit);
    up = min_or_nan(max_or_nan(up, -limit), limit);
  }
  return gate * __frcp_rn(1.0f + expf(-gate)) * up;
}

// MOST: groups of 8 tokens that a pass can have.
template <bool DOWN, int MOST>
__global__ void __launch_bounds__(kStreamThreads, 1)
stream_kernel(const DecodeParams p, const __grid_constant__ DecodeMaps maps, int stages) {
  extern __shared__ __align__(1024) uint8_t shared_memory[];
  __shared__ Barriers bars;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* token_stages = shared_memory + stages * kStageA;
  float* weight_scales = reinterpret_cast<float*>(token_stages + stages * p.b_rows * kTokenBytes);
  float* meet = weight_scales + stages * kStageScales;  // [slab][value][lane]
  __shared__ Lists l;  // (in shared memory: its pointers took ten registers)
  if (tid == 0) {
    l.place(reinterpret_cast<uint8_t*>(meet) + meet_bytes(p.T), p.T, p.E, p.K);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bars.full[i], 1 + 32);  // boxes and copies
      mbar_init(&bars.empty[i], kMultiplyWarps);
    }
    bars.abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.routed.tall);
    tma_prefetch_desc(&maps.routed.middle);
    tma_prefetch_desc(&maps.routed.flat);
  }
  __syncthreads();
  // UP starts from the routing; when its blocks have seen that finished they let the next kernels start, so that
  // DOWN finds the routing finished and waits for act alone (keep_full)
  if (!DOWN) dependency_wait();
  dependency_release();
  const int active = build_lists<DOWN>(l, p, !DOWN && blockIdx.x == 0 ? p.row_of : nullptr,
                                       !DOWN && p.fp8 ? p.x16_scale : nullptr);
  if (warp >= kMultiplyWarps) {
    keep_full<DOWN, MOST>(p, maps, l, active, shared_memory, token_stages, weight_scales, stages, bars);
    return;
  }

  const auto meet_all = [] { named_sync(1, 32 * kMultiplyWarps); };  // the multiplying warps
  Stream<DOWN> now(p, l, l.part, active);
  int slot = 0;
  uint32_t phase = 0;
  bool dead = false;  // a wait ran out: go on to the end without waiting or releasing a stage, the status says so
  while (now.next()) {
    const Piece& piece = now.piece;
    const bool is_shared = piece.index == active;
    constexpr int kTile = DOWN ? 16 : 8;  // output columns
    const int rt = warp & ((1 << piece.rt_log) - 1), ks = warp >> piece.rt_log, ks_count = 1 << piece.ks_log;
    const bool mine = ks < ks_count && rt * kTile < piece.count;
    // this lane's two weight rows are `column` and, 8 further (DOWN) or the up row of the same column (UP)
    const int column = rt * kTile + box_row(g);
    const int high = DOWN ? 1024 : 1024 << piece.rt_log;
    const uint32_t a_first = smem_u32(shared_memory) + (ks << piece.rt_log) * kSlab + rt * (DOWN ? 2048 : 1024) +
                             box_row(g) * 128 + ((t ^ box_row(g)) << 4);
    const int pitch = piece.fp8 ? kTokenBytes : kTokenPitchBf16;
    const uint32_t b_first = smem_u32(token_stages) + ks * piece.n * pitch;
    uint32_t token[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      const int j = min(i * 8 + g, piece.n - 1);
      token[i] = j * pitch + (piece.fp8 ? ((2 * t) ^ ((ks * piece.n + j) & 1)) << 4 : t << 4);
    }
    float acc[MOST * 4];
#pragma unroll
    for (int i = 0; i < MOST * 4; ++i) acc[i] = 0.f;
    const int n = piece.n, blocks = mine ? piece.blocks : 0;
    const bool fp8 = piece.fp8;
    int block = ks;
    // No stage is full before act is there; how long that takes is not for the waits below to bound.
    if (DOWN) dependency_wait();
    for (int step = piece.steps; step > 0; --step, block += ks_count) {
      if (!dead) dead = !mbar_wait_warp(&bars.full[slot], phase, &bars.abort, p.status, 72);
      if (block < blocks) {
        const uint32_t a = a_first + slot * kStageA, b = b_first + slot * p.b_rows * kTokenBytes;
        if (fp8)
          multiply_e4m3<MOST>(a, high, reinterpret_cast<const float2*>(weight_scales + slot * kStageScales)[warp], b, token,
                              n, acc);
        else
          multiply_bf16<MOST>(a, high, b, token, n, acc);
      }
      __syncwarp();
      if (lane == 0 && !dead) mbar_arrive(&bars.empty[slot]);
      if (++slot == stages) {
        slot = 0;
        phase ^= 1;
      }
    }
    // The piece's sums are complete.
    if (ks_count > 1) {  // the warps of a tile add up
      const int used = 4 * ((piece.n + 7) >> 3);
      meet_all();
      if (mine && ks > 0) {
#pragma unroll
        for (int i = 0; i < MOST * 4; ++i)
          if (i < used) meet[(warp * used + i) * 32 + lane] = acc[i];
      }
      meet_all();
      if (mine && ks == 0) {
        for (int s = 1; s < ks_count; ++s)
#pragma unroll
          for (int i = 0; i < MOST * 4; ++i)
            if (i < used) acc[i] += meet[(((s << piece.rt_log) + rt) * used + i) * 32 + lane];
      }
    }
    if (mine && ks == 0 && column < piece.count) {
      const int width = DOWN ? p.D : is_shared ? p.shared_inner : p.F;
#pragma unroll
      for (int q = 0; q < MOST * 2; ++q) {
        const int j = (q >> 1) * 8 + 2 * t + (q & 1);
        float first = acc[(q >> 1) * 4 + (q & 1)], second = acc[(q >> 1) * 4 + 2 + (q & 1)];
        if (j < piece.n) {
          if (!DOWN && piece.fp8) {
            const float scale = l.scale[piece.begin + j];
            first *= scale, second *= scale;
          }
          const long long at = (long long)(piece.begin + j) * width + piece.first + column;
          if (DOWN) {
            float* to = p.y + (is_shared ? (long long)p.T * p.K * p.D : 0) + at;
            to[0] = first;
            if (column + 8 < piece.count) to[8] = second;
          } else {
            (is_shared ? p.act_shared : p.act)[at] = __float2bfloat16_rn(gated(first, second, p.limited, p.limit));
          }
        }
      }
    }
  }
}

// act [rows, F] for the E4M3 down product, a block to a row.  Latency: 1024 threads where the row has more than four
// loads for each of 256 (34 rows of 14336: 10 us with 256).
__global__ void __launch_bounds__(1024)
scale_act_kernel(const __nv_bfloat16* __restrict__ act, int F, __half* __restrict__ act16, float* __restrict__ act16_scale) {
  __shared__ uint32_t largest[32];
  const long long at = (long long)blockIdx.x * F;
  dependency_release();
  dependency_wait();
  const float scale = scale_row(act + at, F, act16 + at, largest);
  if (threadIdx.x == 0) act16_scale[blockIdx.x] = scale;
}

// out[t] = residual[t] + sum_k w[t,k] y[row_of[t,k]] (+ the shared expert's row of t): fp32, k ascending, one rounding.
// A thread has four columns of a token.
__global__ void __launch_bounds__(kDecodeThreads)
join_kernel(const DecodeParams p) {
  const int t = blockIdx.y, c = (blockIdx.x * kDecodeThreads + threadIdx.x) * 4;
  dependency_wait();
  if (c >= p.D) return;
  const long long at = (long long)t * p.D + c;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __bfloat162float(p.residual[at + i]);
  for (int k0 = 0; k0 < p.K; k0 += 8) {  // eight rows asked for at once
    float w[8];
    float4 y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (k0 + i < p.K) {
        const int row = p.row_of[t * p.K + k0 + i];
        w[i] = p.route_weights[t * p.K + k0 + i];
        if (p.fp8) w[i] *= p.act16_scale[row];  // (a power of two)
        y[i] = *reinterpret_cast<const float4*>(p.y + (long long)row * p.D + c);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (k0 + i < p.K) {
        v[0] = fmaf(w[i], y[i].x, v[0]), v[1] = fmaf(w[i], y[i].y, v[1]);
        v[2] = fmaf(w[i], y[i].z, v[2]), v[3] = fmaf(w[i], y[i].w, v[3]);
      }
    }
  }
  if (p.shared_inner > 0) {
    const float4 y = *reinterpret_cast<const float4*>(p.y + (long long)(p.T * p.K + t) * p.D + c);
    v[0] += y.x, v[1] += y.y, v[2] += y.z, v[3] += y.w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p.out[at + i] = __float2bfloat16_rn(v[i]);
}

struct DecodeWorkspace {
  long long logits, x16, x16_scale, act, act_shared, act16, act16_scale, y, row_of, bytes;
  DecodeWorkspace(long long T, long long D, long long E, long long K, long long F, long long shared_inner) {
    const auto up = [](long long n) { return (n + 255) / 256 * 256; };
    logits = 0;
    x16 = up(4 * T * E);
    x16_scale = x16 + up(2 * T * D);
    act = x16_scale + up(4 * T);
    act_shared = act + up(2 * T * K * F);
    act16 = act_shared + up(2 * T * shared_inner);
    act16_scale = act16 + up(2 * T * K * F);
    y = act16_scale + up(4 * T * K);
    row_of = y + up(4 * (T * K + (shared_inner > 0 ? T : 0)) * D);
    bytes = row_of + up(4 * T * K);
  }
};

static int decode_sizes(long long tokens, int width, int inner, int experts, int top_k, int shared_inner) {
  if (tokens < 0 || width <= 0 || inner <= 0 || experts <= 0 || top_k <= 0 || top_k > experts || shared_inner < 0)
    return B200MOE_ERR_ARG;
  if (tokens > kMaxTokens || experts > 1024 || top_k > 32 || width > (1 << 19) || inner > (1 << 19) ||
      shared_inner > (1 << 19))
    return B200MOE_ERR_LIMIT;
  if (width % 8 || inner % 8 || shared_inner % 8) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

template <typename W>
static int launch_router(const b200moe_decode_args* a, float* logits, __half* x16, float* x16_scale,
                         cudaStream_t s) {
  cudaLaunchConfig_t config = {};
  const int scaling = x16 != nullptr ? ((int)a->tokens + kRouterCluster - 1) / kRouterCluster : 0;  // a block to a token
  config.gridDim = dim3((unsigned)(((a->experts + 15) / 16 + scaling) * kRouterCluster));
  config.blockDim = dim3(kDecodeThreads);
  config.stream = s;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = kRouterCluster;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  const auto kernel = a->tokens <= 8 ? router_logits_kernel<W, 1> : a->tokens <= 32 ? router_logits_kernel<W, 4>
                                                                                   : router_logits_kernel<W, 8>;
  if (cudaLaunchKernelEx(&config, kernel, (const __nv_bfloat16*)a->x, (const W*)a->router, (int)a->tokens, a->experts,
                         a->width, logits, x16, x16_scale) == cudaSuccess)
    return B200MOE_OK;
  cudaGetLastError();  // this call's, reported here
  return B200MOE_ERR_LAUNCH;
}

// [rows, k] weights in boxes of `height` rows x 128 bytes
static int encode_weights(CUtensorMap* map, const void* base, bool fp8, long long rows, long long k, int height) {
  const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows}, strides[1] = {(uint64_t)(k * (fp8 ? 1 : 2))};
  const uint32_t box[2] = {fp8 ? 128u : 64u, (uint32_t)height};
  return encode_tensor_map(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims,
                           strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool DOWN, int MOST>
static int launch_stream(const DecodeParams& p, const DecodeMaps& maps, cudaStream_t s) {
  const int stage = kStageA + p.b_rows * kTokenBytes + kStageScales * 4;
  const int rest = meet_bytes(p.T) + Lists::bytes(p.T, p.E, p.K);
  int stages = (225 * 1024 - rest) / stage;
  if (stages > kMaxStages) stages = kMaxStages;
  if (stages < kFillWarps) return B200MOE_ERR_LIMIT;
  const int bytes = stages * stage + rest;
  const auto kernel = stream_kernel<DOWN, MOST>;
  static std::atomic<unsigned long long> allowed{0};  // devices on which the kernel may have that much shared memory
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return B200MOE_ERR_LAUNCH;
  if (!((allowed.load(std::memory_order_relaxed) >> device) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024) != cudaSuccess) {
      cudaGetLastError();
      return B200MOE_ERR_LAUNCH;
    }
    allowed.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  return launch_dependent(kernel, sm_count(), kStreamThreads, bytes, s, true, p, maps, stages);
}

template <int MOST>
static int launch_streams(const DecodeParams& p, const DecodeMaps& up, const DecodeMaps& down, cudaStream_t s) {
  int code = launch_stream<false, MOST>(p, up, s);
  if (code != B200MOE_OK) return code;
  if (p.fp8) {
    const int threads = p.F > 16 * kDecodeThreads ? 1024 : kDecodeThreads;
    code = launch_dependent(scale_act_kernel, p.T * p.K, threads, 0, s, true, p.act, p.F, p.act16, p.act16_scale);
    if (code != B200MOE_OK) return code;
  }
  code = launch_stream<true, MOST>(p, down, s);
  if (code != B200MOE_OK) return code;
  return launch_dependent(join_kernel, dim3((p.D / 4 + kDecodeThreads - 1) / kDecodeThreads, p.T), kDecodeThreads, 0, s,
                          true, p);
}

}  // namespace b200

using namespace b200;

#ifdef B200_WAIT_TEST
// Test builds only: which product of the next calls (0: none) lacks the stages of which fill warp; the waits for them run
// out.
static int g_withhold_decode[2] = {0, 0};
extern "C" int b200moe_debug_withhold_decode(int product, int warp) {
  g_withhold_decode[0] = product;
  g_withhold_decode[1] = warp;
  return B200MOE_OK;
}
#endif

extern "C" long long b200moe_decode_workspace_bytes(long long tokens, int width, int inner, int experts, int top_k,
                                                    int shared_inner) {
  if (decode_sizes(tokens, width, inner, experts, top_k, shared_inner) != B200MOE_OK) return -1;
  return DecodeWorkspace(tokens, width, experts, top_k, inner, shared_inner).bytes;
}

extern "C" int b200moe_decode(const b200moe_decode_args* a, void* stream) {
  if (a == nullptr) return B200MOE_ERR_ARG;
  const int bad = decode_sizes(a->tokens, a->width, a->inner, a->experts, a->top_k, a->shared_inner);
  if (bad != B200MOE_OK) return bad;
  if (a->mode < 0 || a->mode > 2) return B200MOE_ERR_ARG;
  if (a->mode == B200MOE_ROUTE_SIGMOID_NOAUX_TC) {
    if (a->n_group <= 0 || a->topk_group <= 0 || a->experts % a->n_group) return B200MOE_ERR_ARG;
    if (a->n_group > 32 && a->topk_group < a->n_group) return B200MOE_ERR_LIMIT;
  }
  const bool fp8 = a->w13_scale != nullptr;
  if (!a->x || !a->residual || !a->router || !a->w13 || !a->w2 || !a->route_weights || !a->ids || !a->output ||
      !a->workspace || !a->status || fp8 != (a->w2_scale != nullptr) ||
      (a->shared_inner > 0 && (!a->shared_w13 || !a->shared_w2)))
    return B200MOE_ERR_ARG;
  if (fp8 && (a->width % 128 || a->inner % 128)) return B200MOE_ERR_ALIGN;
  for (const void* q : {a->x, a->router, a->w13, a->w2, a->shared_w13, a->shared_w2})
    if ((uintptr_t)q & 15) return B200MOE_ERR_ALIGN;
  for (const void* q : {(const void*)a->w13_scale, (const void*)a->w2_scale, (const void*)a->bias,
                        (const void*)a->route_weights, (const void*)a->ids, (const void*)a->status})
    if ((uintptr_t)q & 3) return B200MOE_ERR_ALIGN;
  if (((uintptr_t)a->workspace & 255) || ((uintptr_t)a->output & 1) || ((uintptr_t)a->residual & 1))
    return B200MOE_ERR_ALIGN;
  if (a->tokens == 0) return B200MOE_OK;

  DecodeMaps up, down;
  const long long E = a->experts, D = a->width, F = a->inner, Fs = a->shared_inner;
  int code = B200MOE_OK;
  const auto encode = [&](WeightMaps& maps, const void* weights, bool e4m3, long long rows, long long k, int tall) {
    if (code == B200MOE_OK) code = encode_weights(&maps.tall, weights, e4m3, rows, k, tall);
    if (code == B200MOE_OK) code = encode_weights(&maps.middle, weights, e4m3, rows, k, 32);
    if (code == B200MOE_OK) code = encode_weights(&maps.flat, weights, e4m3, rows, k, 8);
  };
  encode(up.routed, a->w13, fp8, 2 * E * F, D, 128);
  encode(down.routed, a->w2, fp8, E * D, F, 256);
  if (Fs > 0) {
    encode(up.shared, a->shared_w13, false, 2 * Fs, D, 128);
    encode(down.shared, a->shared_w2, false, D, Fs, 256);
  }
  if (code != B200MOE_OK) return code;
  const DecodeWorkspace w(a->tokens, a->width, a->experts, a->top_k, a->inner, a->shared_inner);
  char* base = reinterpret_cast<char*>(a->workspace);
  float* logits = reinterpret_cast<float*>(base + w.logits);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  __half* x16 = fp8 ? reinterpret_cast<__half*>(base + w.x16) : nullptr;
  float* x16_scale = reinterpret_cast<float*>(base + w.x16_scale);
  code = a->router_is_fp32 ? launch_router<float>(a, logits, x16, x16_scale, s)
                           : launch_router<__nv_bfloat16>(a, logits, x16, x16_scale, s);
  if (code != B200MOE_OK) return code;
  code = launch_route_topk(logits, a->experts, (int)a->tokens, a->experts, a->top_k, a->mode, a->bias, a->n_group,
                           a->topk_group, a->routed_scaling, a->route_weights, a->ids, true, s);
  if (code != B200MOE_OK) return code;
  DecodeParams p = {};
  p.x = reinterpret_cast<const __nv_bfloat16*>(a->x);
  p.residual = reinterpret_cast<const __nv_bfloat16*>(a->residual);
  p.ids = a->ids;
  p.route_weights = a->route_weights;
  p.w2 = reinterpret_cast<const uint8_t*>(a->w2);
  p.w13_scale = a->w13_scale;
  p.w2_scale = a->w2_scale;
  p.x16 = x16;
  p.x16_scale = x16_scale;
  p.act = reinterpret_cast<__nv_bfloat16*>(base + w.act);
  p.act16 = reinterpret_cast<__half*>(base + w.act16);
  p.act16_scale = reinterpret_cast<float*>(base + w.act16_scale);
  p.y = reinterpret_cast<float*>(base + w.y);
  p.row_of = reinterpret_cast<int*>(base + w.row_of);
  p.act_shared = reinterpret_cast<__nv_bfloat16*>(base + w.act_shared);
  p.out = reinterpret_cast<__nv_bfloat16*>(a->output);
  p.T = (int)a->tokens, p.D = a->width, p.F = a->inner, p.E = a->experts, p.K = a->top_k;
  p.shared_inner = a->shared_inner;
  p.fp8 = fp8, p.limited = a->limited, p.limit = a->limit;
  p.b_rows = p.T <= 2 ? 16 * p.T : kPassTokens;
  p.status = a->status;
#ifdef B200_WAIT_TEST
  p.withhold = g_withhold_decode[0], p.withheld = g_withhold_decode[1];
#endif
  return p.T <= 8 ? launch_streams<1>(p, up, down, s) : launch_streams<kPassTokens / 8>(p, up, down, s);
}
