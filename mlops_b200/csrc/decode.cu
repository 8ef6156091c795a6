// The routed layer for a few tokens (1 to 64), as a serving loop calls it: router logits, expert selection, up
// product with SwiGLU, down product with the weighted sum, residual and shared expert.
//
//   logits = x . bf16(router)^T                          router_logits_kernel
//   (weights, ids) = the routing of route.cu
//   act[t,k] = bf16(silu(g) * u), [g | u] = x[t] . W13[e]^T          stream_kernel<UP>
//   out[t] = residual[t] + sum_k w[t,k] act[t,k] . W2[e]^T (+ the shared expert's)   stream_kernel<DOWN>
//
// Bound: HBM.  The weights of the experts that got a token are read once, 3 D F bytes each in E4M3, for one
// or a few multiplications a byte; everything else is small.  So the two products are one stream of weight
// rows through shared memory (16-byte asynchronous copies, several stages of 16 KB in flight per SM), cut evenly over
// the SMs to the single row: with whole tiles of 64 columns eight experts of F = 768 would leave 52 of 148 SMs idle.
//
// The weights are the A operand of mma.m16n8k16 (16 weight rows), the tokens the B operand (8 to a
// tile).  Activations stay bf16: E4M3 weights are widened to bf16, which holds every E4M3 value, and the
// 128 x 128 block scales are applied in fp32 to the sums of one 128-column block, so nothing is quantised.  tcgen05
// has no product of E4M3 by bf16 and its tiles start at 64 rows; at one to eight tokens a weight row the
// tensor rate is not what bounds this.  Sums are fp32; act is rounded to bf16 once, as the operand of the second product
// (the grouped layer rounds it likewise), and the output once.  Every sum has a fixed order: no atomics.
#include "common.cuh"
#include "host_util.h"
#include "../../include/b200moe.h"

namespace b200 {

constexpr int kDecodeThreads = 256;
constexpr int kDecodeWarps = 8;
constexpr int kMaxTokens = 64;
constexpr int kSlab = 2048;               // 16 weight rows x 128 bytes of K
constexpr int kStageA = 8 * kSlab;        // a stage holds eight slabs: row tiles x K blocks
constexpr int kStageScales = 8 * 16 * 4;  // one scale per row of a slab

__device__ __forceinline__ void copy16(void* dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(read ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two E4M3 values as bf16 (through f16, exact both ways).
__device__ __forceinline__ uint32_t widen2(uint32_t pair) {
  const __half2 h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
  const float2 f = __half22float2(h);
  return pack_bf16x2(f.x, f.y);
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

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
                     float* __restrict__ logits) {
  __shared__ float partial[kDecodeWarps][NT * 8][16];
  __shared__ float sums[NT * 8][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)cluster_ctarank();
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
  const uint8_t *w13, *w2;  // E4M3 or bf16
  const float *w13_scale, *w2_scale;
  const uint8_t *shared_w13, *shared_w2;  // bf16, or null
  __nv_bfloat16* act;                     // [T * K, F] in expert order
  __nv_bfloat16* act_shared;              // [T, shared_inner]
  __nv_bfloat16* out;
  int T, D, F, E, K, shared_inner;
  int fp8, limited;
  float limit;
  int b_rows;  // capacity of a stage's B part, in rows of one K block
};

// Where things are in shared memory behind the stages.
struct Lists {
  int* begin;          // [experts with tokens + 1] first row of each
  float* weights;      // [T * K] route weight of each row
  uint16_t* expert;    // [experts with tokens]
  uint8_t* tokens;     // [T * K]
  int* scratch;        // [E + 64]
  uint16_t* rank;      // [T * K]
  __host__ __device__ static int bytes(int T, int E, int K) {
    const int R = T * K, most = E < R ? E : R;
    return 4 * (most + 1) + 4 * R + 4 * (E + 64) + 2 * (most + R) + R + 64;
  }
  __device__ void place(uint8_t* base, int T, int E, int K) {
    const int R = T * K, most = E < R ? E : R;
    begin = reinterpret_cast<int*>(base);
    weights = reinterpret_cast<float*>(begin + most + 1);
    scratch = reinterpret_cast<int*>(weights + R);
    expert = reinterpret_cast<uint16_t*>(scratch + E + 64);
    rank = expert + most;
    tokens = reinterpret_cast<uint8_t*>(rank + R);
  }
};

// Rows by expert, in token order inside one; returns the number of experts with tokens.
__device__ __forceinline__ int build_lists(const Lists& l, const int* __restrict__ ids,
                                           const float* __restrict__ route_weights, int T, int E, int K) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = T * K;
  int* count = l.scratch;           // per expert: rows, then first row
  int* totals = l.scratch + E;      // per warp
  for (int e = tid; e < E; e += kDecodeThreads) count[e] = 0;
  __syncthreads();
  if (warp == 0) {
    for (int base = 0; base < R; base += 32) {
      const int i = base + lane;
      const bool in = i < R;
      const int e = in ? ids[i] : -1 - lane;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int before = __popc(same & ((1u << lane) - 1));
      if (in) l.rank[i] = (uint16_t)(count[e] + before);
      __syncwarp();
      if (in && before == 0) count[e] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  // exclusive sums over the experts of (rows, experts with rows), packed in one word
  const int per = (E + kDecodeThreads - 1) / kDecodeThreads;
  int mine = 0;
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j;
    if (e < E && count[e]) mine += count[e] | (1 << 16);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) totals[warp] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < warp; ++w) at += totals[w];
  int active = 0;
  for (int w = 0; w < kDecodeWarps; ++w) active += totals[w];
  active >>= 16;
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j;
    if (e >= E) break;
    const int n = count[e];
    count[e] = at & 0xffff;
    if (n) {
      l.expert[at >> 16] = (uint16_t)e;
      l.begin[at >> 16] = at & 0xffff;
      at += n | (1 << 16);
    }
  }
  if (tid == 0) l.begin[active] = R;
  __syncthreads();
  for (int i = tid; i < R; i += kDecodeThreads) {
    const int at_row = count[ids[i]] + l.rank[i];
    l.weights[at_row] = route_weights[i];
    l.tokens[at_row] = (uint8_t)(i / K);
  }
  __syncthreads();
  return active;
}

// A piece of the stream: consecutive output columns (UP: of the activation, gate and up rows alike; DOWN: of the
// output) of one expert.  Its rows are cut into 1 << rt_log tiles of 16, the K blocks of a stage go to the
// 1 << ks_log warps of each tile.
struct Piece {
  int index;         // expert with tokens, or `active` for the shared expert
  int first, count;  // output columns
  int n, begin;      // tokens, and the first of their rows
  int rt_log, ks_log;
  int steps, blocks;  // stages, K blocks
  bool fp8;
};

template <bool DOWN>
struct Stream {
  const DecodeParams& p;
  const Lists& l;
  int active;
  int at, end;  // UP: flat activation columns of the experts with tokens, then the shared expert's; DOWN: output columns
  int row_first, row_count, which;  // DOWN: current run of output columns, next expert
  int step;
  bool done;
  Piece piece;

  __device__ Stream(const DecodeParams& params, const Lists& lists, int n_active) : p(params), l(lists), active(n_active) {
    const long long b = blockIdx.x, grid = gridDim.x;
    if (DOWN) {
      at = (int)(p.D * b / grid);
      end = (int)(p.D * (b + 1) / grid);
      row_first = at;
      row_count = min(128, end - at);
      which = 0;
    } else {
      const long long total = (long long)active * p.F + (long long)shared_weight() * p.shared_inner;
      at = (int)(total * b / grid);
      end = (int)(total * (b + 1) / grid);
    }
    done = false;
    open();
  }
  // a column of a bf16 shared expert costs twice what an E4M3 expert's does
  __device__ int shared_weight() const { return p.fp8 ? 2 : 1; }
  __device__ int shared_column(int flat) const { return (flat - active * p.F + shared_weight() - 1) / shared_weight(); }

  __device__ void open() {
    step = 0;
    if (DOWN) {
      const int experts = active + (p.shared_inner > 0 ? 1 : 0);
      if (which == experts) {
        which = 0;
        row_first += row_count;
        row_count = min(128, end - row_first);
      }
      if (row_count <= 0) {
        done = true;
        return;
      }
      piece.index = which++;
      piece.first = row_first;
      piece.count = row_count;
    } else {
      for (;;) {
        if (at >= end) {
          done = true;
          return;
        }
        if (at < active * p.F) {
          piece.index = at / p.F;
          piece.first = at - piece.index * p.F;
          piece.count = min(min(64, p.F - piece.first), end - at);
          at += piece.count;
          break;
        }
        const int from = shared_column(at), to = shared_column(end);
        piece.index = active;
        piece.first = from;
        piece.count = min(64, to - from);
        at = piece.count > 0 && from + piece.count < to ? active * p.F + shared_weight() * (from + piece.count) : end;
        if (piece.count > 0) break;
      }
    }
    const bool shared = piece.index == active;
    piece.fp8 = p.fp8 && !shared;
    piece.begin = shared ? 0 : l.begin[piece.index];
    piece.n = shared ? p.T : l.begin[piece.index + 1] - piece.begin;
    const int tiles = DOWN ? (piece.count + 15) / 16 : (piece.count + 7) / 8;
    piece.rt_log = tiles <= 1 ? 0 : 32 - __clz(tiles - 1);
    piece.ks_log = 0;
    while (piece.ks_log + piece.rt_log < 3 && (2 << piece.ks_log) * piece.n <= p.b_rows) ++piece.ks_log;
    piece.blocks = (inner() * (piece.fp8 ? 1 : 2) + 127) / 128;
    piece.steps = (piece.blocks + (1 << piece.ks_log) - 1) >> piece.ks_log;
  }
  __device__ int inner() const { return DOWN ? (piece.index == active ? p.shared_inner : p.F) : p.D; }
  __device__ void advance() {
    if (++step == piece.steps) open();
  }
};

// Fills stages: the next stage's weights, scales and tokens.
template <bool DOWN>
struct Loader : Stream<DOWN> {
  const uint8_t* src[4];  // this thread's four chunks of 16 bytes
  uint32_t has;           // which of them exist
  const float* scale;     // and its scale, per K block
  using Stream<DOWN>::p;
  using Stream<DOWN>::l;
  using Stream<DOWN>::piece;

  __device__ Loader(const DecodeParams& params, const Lists& lists, int n_active)
      : Stream<DOWN>(params, lists, n_active) {
    aim();
  }
  // the weight row behind row `r` of tile `rt`, or -1
  __device__ int weight_row(int rt, int r) const {
    if (DOWN) {
      const int row = rt * 16 + r;
      return row < piece.count ? piece.first + row : -1;
    }
    const int column = rt * 8 + (r & 7);
    const int half = piece.index == this->active ? p.shared_inner : p.F;
    return column < piece.count ? (r >> 3) * half + piece.first + column : -1;
  }
  __device__ void aim() {
    if (this->done) return;
    const bool shared = piece.index == this->active;
    const int inner = this->inner();
    const long long pitch = (long long)inner * (piece.fp8 ? 1 : 2);
    const uint8_t* base = DOWN ? (shared ? p.shared_w2 : p.w2) : (shared ? p.shared_w13 : p.w13);
    const float* scales = DOWN ? p.w2_scale : p.w13_scale;
    if (!shared) {
      const long long e = l.expert[piece.index], rows = DOWN ? p.D : 2LL * p.F;
      base += e * rows * pitch;
      if (piece.fp8) scales += e * (rows / 128) * piece.blocks;
    }
    const int tid = threadIdx.x, r = (tid >> 3) & 15;
    has = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int slab = (tid >> 7) + 2 * i, rt = slab & ((1 << piece.rt_log) - 1), ks = slab >> piece.rt_log;
      const int row = ks < (1 << piece.ks_log) ? weight_row(rt, r) : -1;
      src[i] = base + (row < 0 ? 0 : row) * pitch + ks * 128 + (tid & 7) * 16;
      if (row >= 0) has |= 1u << i;
    }
    if (tid < 128) {
      const int slab = tid >> 4, rt = slab & ((1 << piece.rt_log) - 1), ks = slab >> piece.rt_log;
      const int row = piece.fp8 && ks < (1 << piece.ks_log) ? weight_row(rt, tid & 15) : -1;
      scale = row < 0 ? nullptr : scales + (long long)(row >> 7) * piece.blocks + ks;
    }
  }
  __device__ void fill(uint8_t* stage) {
    if (!this->done) {
      const int tid = threadIdx.x, inner = this->inner(), ks_count = 1 << piece.ks_log;
      const int block0 = this->step << piece.ks_log;  // first K block of the stage
      const int pitch = inner * (piece.fp8 ? 1 : 2);
      const int r = (tid >> 3) & 15;
      const int to = r * 128 + (((tid & 7) ^ ((r & 1) << 2)) << 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int slab = (tid >> 7) + 2 * i, block = block0 + (slab >> piece.rt_log);
        const bool in = block * 128 + (tid & 7) * 16 < pitch;  // zeros behind the end of a row
        if (((has >> i) & 1) && block < piece.blocks)
          copy16(stage + slab * kSlab + to, in ? src[i] : (const uint8_t*)p.x, in);
        src[i] += ks_count * 128;
      }
      if (tid < 128) {
        if (scale != nullptr && block0 + (tid >> (4 + piece.rt_log)) < piece.blocks)
          copy4(stage + kStageA + tid * 4, scale);
        scale += scale != nullptr ? ks_count : 0;
      }
      // the tokens' columns of the same K blocks: [K block][token][256 or 128 bytes]
      const bool shared = piece.index == this->active;
      const int chunk_log = piece.fp8 ? 4 : 3, total = (ks_count * piece.n) << chunk_log;
      uint8_t* b = stage + kStageA + kStageScales;
      for (int i = tid; i < total; i += kDecodeThreads) {
        const int chunk = i & ((1 << chunk_log) - 1), at_row = i >> chunk_log;
        const int ks = ks_count == 1 ? 0 : at_row / piece.n, row = at_row - ks * piece.n;
        const int block = block0 + ks;
        if (block >= piece.blocks) continue;
        const int k = (block << (chunk_log + 3)) + chunk * 8;
        const __nv_bfloat16* from;
        if (DOWN)
          from = shared ? p.act_shared + (long long)row * inner : p.act + (long long)(piece.begin + row) * inner;
        else
          from = p.x + (long long)(shared ? row : l.tokens[piece.begin + row]) * inner;
        const int swizzle = piece.fp8 ? (row & 1) : (row & 1) << 2;
        copy16(b + (at_row << (chunk_log + 4)) + ((chunk ^ swizzle) << 4), from + (k < inner ? k : 0), k < inner);
      }
      const int before = this->step;
      this->advance();
      if (this->step != before + 1) aim();
    }
    copies_commit();
  }
};

// One warp's slab of a stage: 16 weight rows x 128 bytes of K by NT tiles of 8 tokens.  Lane (g, t) reads the
// same 16 (bf16: 8) consecutive columns of its weight rows and of its token, which is one order of the columns
// for both operands.  Rows behind the last token are read as that token's; their sums go nowhere.
template <bool FP8, int NT>
__device__ __forceinline__ void multiply(const uint8_t* slab, const float* scales, const uint8_t* b, int n,
                                         float (&acc)[8][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint8_t* rows = slab + g * 128;
  const int swizzle = (g & 1) << 2;
  float part[NT][4];
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < NT; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
  }
#pragma unroll
  for (int segment = 0; segment < 2; ++segment) {
    const int at = ((segment * 4 + t) ^ swizzle) << 4;
    const uint4 lo = *reinterpret_cast<const uint4*>(rows + at);
    const uint4 hi = *reinterpret_cast<const uint4*>(rows + 1024 + at);
    if constexpr (FP8) {
      uint32_t a[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j][0] = widen2(word(lo, j));
        a[j][1] = widen2(word(hi, j));
        a[j][2] = widen2(word(lo, j) >> 16);
        a[j][3] = widen2(word(hi, j) >> 16);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = min(i * 8 + g, n - 1), chunk = segment * 8 + 2 * t;
        const uint4 v0 = *reinterpret_cast<const uint4*>(b + row * 256 + ((chunk ^ (row & 1)) << 4));
        const uint4 v1 = *reinterpret_cast<const uint4*>(b + row * 256 + (((chunk + 1) ^ (row & 1)) << 4));
        mma_bf16(part[i], a[0][0], a[0][1], a[0][2], a[0][3], v0.x, v0.y);
        mma_bf16(part[i], a[1][0], a[1][1], a[1][2], a[1][3], v0.z, v0.w);
        mma_bf16(part[i], a[2][0], a[2][1], a[2][2], a[2][3], v1.x, v1.y);
        mma_bf16(part[i], a[3][0], a[3][1], a[3][2], a[3][3], v1.z, v1.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = min(i * 8 + g, n - 1);
        const uint4 v = *reinterpret_cast<const uint4*>(b + row * 128 + (((segment * 4 + t) ^ ((row & 1) << 2)) << 4));
        mma_bf16(acc[i], lo.x, hi.x, lo.y, hi.y, v.x, v.y);
        mma_bf16(acc[i], lo.z, hi.z, lo.w, hi.w, v.z, v.w);
      }
    }
  }
  if constexpr (FP8) {
    const float s0 = scales[g], s1 = scales[g + 8];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      acc[i][0] = fmaf(part[i][0], s0, acc[i][0]);
      acc[i][1] = fmaf(part[i][1], s0, acc[i][1]);
      acc[i][2] = fmaf(part[i][2], s1, acc[i][2]);
      acc[i][3] = fmaf(part[i][3], s1, acc[i][3]);
    }
  }
}

__device__ __forceinline__ float gated(float gate, float up, int limited, float limit) {
  if (limited) {
    gate = fminf(gate, limit);
    up = fminf(fmaxf(up, -limit), limit);
  }
  return gate * __frcp_rn(1.0f + expf(-gate)) * up;
}

template <bool DOWN, int STAGES>
__global__ void __launch_bounds__(kDecodeThreads, 2)
stream_kernel(const DecodeParams p) {
  extern __shared__ __align__(128) uint8_t shared_memory[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int stage_bytes = kStageA + kStageScales + p.b_rows * 256;
  uint8_t* behind = shared_memory + STAGES * stage_bytes;
  float* sums = reinterpret_cast<float*>(behind);  // DOWN: [slab][token][16 output columns]
  Lists l;
  l.place(behind + (DOWN ? 8 * 16 * 4 * p.T : 0), p.T, p.E, p.K);
  const int active = build_lists(l, p.ids, p.route_weights, p.T, p.E, p.K);
  if (DOWN) {
    for (int i = tid; i < 8 * 16 * p.T; i += kDecodeThreads) sums[i] = 0.f;
    __syncthreads();
  }

  Loader<DOWN> loader(p, l, active);
  Stream<DOWN> now(p, l, active);
  for (int i = 0; i < STAGES - 1; ++i) loader.fill(shared_memory + i * stage_bytes);
  float acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  int slot = 0;
  while (!now.done) {
    copies_wait<STAGES - 2>();
    __syncthreads();  // this stage is there for everybody, and the one before it is free
    loader.fill(shared_memory + (slot == 0 ? STAGES - 1 : slot - 1) * stage_bytes);
    const Piece piece = now.piece;
    uint8_t* stage = shared_memory + slot * stage_bytes;
    const int rt = warp & ((1 << piece.rt_log) - 1), ks = warp >> piece.rt_log;
    const bool mine = ks < (1 << piece.ks_log) && rt * (DOWN ? 16 : 8) < piece.count;
    const int block = (now.step << piece.ks_log) + ks, tiles = (piece.n + 7) >> 3;
    if (mine && block < piece.blocks) {
      const uint8_t* slab = stage + warp * kSlab;
      const float* scales = reinterpret_cast<const float*>(stage + kStageA) + warp * 16;
      const uint8_t* b = stage + kStageA + kStageScales + ((ks * piece.n) << (piece.fp8 ? 8 : 7));
      if (piece.fp8) {
        if (tiles == 1) multiply<true, 1>(slab, scales, b, piece.n, acc);
        else if (tiles == 2) multiply<true, 2>(slab, scales, b, piece.n, acc);
        else if (tiles <= 4) multiply<true, 4>(slab, scales, b, piece.n, acc);
        else multiply<true, 8>(slab, scales, b, piece.n, acc);
      } else {
        if (tiles == 1) multiply<false, 1>(slab, scales, b, piece.n, acc);
        else if (tiles == 2) multiply<false, 2>(slab, scales, b, piece.n, acc);
        else if (tiles <= 4) multiply<false, 4>(slab, scales, b, piece.n, acc);
        else multiply<false, 8>(slab, scales, b, piece.n, acc);
      }
    }
    const int step = now.step;
    now.advance();
    if (step + 1 == piece.steps) {  // the piece's sums are complete
      const bool is_shared = piece.index == active;
      if (DOWN) {
        if (mine) {
          float* to = sums + warp * 16 * p.T;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = i * 8 + 2 * t + h;
              if (j < piece.n) {
                const int token = is_shared ? j : l.tokens[piece.begin + j];
                const float w = is_shared ? 1.0f : l.weights[piece.begin + j];
                float* at = to + token * 16 + g;
                at[0] = fmaf(w, acc[i][h], at[0]);
                at[8] = fmaf(w, acc[i][2 + h], at[8]);
              }
            }
          }
        }
        __syncwarp();  // the next expert may give this warp's sums to other lanes
        if (now.done || now.piece.first != piece.first) {  // the last expert of these columns
          __syncthreads();
          for (int i = tid; i < p.T << (piece.rt_log + 4); i += kDecodeThreads) {
            const int column = i & ((16 << piece.rt_log) - 1), token = i >> (piece.rt_log + 4);
            if (column < piece.count) {
              const long long at = (long long)token * p.D + piece.first + column;
              float v = __bfloat162float(p.residual[at]);
              for (int s = column >> 4; s < 8; s += 1 << piece.rt_log) v += sums[(s * p.T + token) * 16 + (column & 15)];
              p.out[at] = __float2bfloat16_rn(v);
            }
          }
          __syncthreads();
          for (int i = tid; i < 8 * 16 * p.T; i += kDecodeThreads) sums[i] = 0.f;
          __syncthreads();
        }
      } else {
        if (piece.ks_log > 0) {  // the warps of a tile meet in the stage that has just been read
          float* meet = reinterpret_cast<float*>(stage);
          __syncthreads();
          if (mine && ks > 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (i < tiles)
#pragma unroll
                for (int h = 0; h < 4; ++h) meet[((warp * tiles + i) * 4 + h) * 32 + lane] = acc[i][h];
          }
          __syncthreads();
          if (mine && ks == 0) {
            for (int s = 1; s < 1 << piece.ks_log; ++s)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (i < tiles)
#pragma unroll
                  for (int h = 0; h < 4; ++h)
                    acc[i][h] += meet[((((s << piece.rt_log) + rt) * tiles + i) * 4 + h) * 32 + lane];
          }
        }
        const int column = rt * 8 + g;
        if (mine && ks == 0 && column < piece.count) {
          const int width = is_shared ? p.shared_inner : p.F;
          __nv_bfloat16* to = (is_shared ? p.act_shared : p.act + (long long)piece.begin * p.F) + piece.first + column;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = i * 8 + 2 * t + h;
              if (j < piece.n)
                to[(long long)j * width] = __float2bfloat16_rn(gated(acc[i][h], acc[i][2 + h], p.limited, p.limit));
            }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    }
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  copies_wait<0>();
}

struct DecodeWorkspace {
  long long logits, act, act_shared, bytes;
  DecodeWorkspace(long long T, long long E, long long K, long long F, long long shared_inner) {
    const auto up = [](long long n) { return (n + 255) / 256 * 256; };
    logits = 0;
    act = up(4 * T * E);
    act_shared = act + up(2 * T * K * F);
    bytes = act_shared + up(2 * T * shared_inner);
  }
};

static int decode_sizes(long long tokens, int width, int inner, int experts, int top_k, int shared_inner) {
  if (tokens < 0 || width <= 0 || inner <= 0 || experts <= 0 || top_k <= 0 || top_k > experts || shared_inner < 0)
    return B200MOE_ERR_ARG;
  if (tokens > kMaxTokens || experts > 1024 || top_k > 32 || width > (1 << 20) || inner > (1 << 20) ||
      shared_inner > (1 << 20))
    return B200MOE_ERR_LIMIT;
  if (width % 8 || inner % 8 || shared_inner % 8) return B200MOE_ERR_ALIGN;
  return B200MOE_OK;
}

template <typename W>
static int launch_router(const b200moe_decode_args* a, float* logits, cudaStream_t s) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((a->experts + 15) / 16 * kRouterCluster));
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
  return cudaLaunchKernelEx(&config, kernel, (const __nv_bfloat16*)a->x, (const W*)a->router, (int)a->tokens, a->experts,
                            a->width, logits) == cudaSuccess
             ? launch_status()
             : B200MOE_ERR_LAUNCH;
}

template <bool DOWN, int STAGES>
static int launch_stream(const DecodeParams& p, cudaStream_t s) {
  const int bytes = STAGES * (kStageA + kStageScales + p.b_rows * 256) + (DOWN ? 8 * 16 * 4 * p.T : 0) +
                    Lists::bytes(p.T, p.E, p.K);
  const auto kernel = stream_kernel<DOWN, STAGES>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return B200MOE_ERR_LAUNCH;
  }
  kernel<<<sm_count(), kDecodeThreads, bytes, s>>>(p);
  return launch_status();
}

}  // namespace b200

using namespace b200;

extern "C" long long b200moe_decode_workspace_bytes(long long tokens, int width, int inner, int experts, int top_k,
                                                    int shared_inner) {
  if (decode_sizes(tokens, width, inner, experts, top_k, shared_inner) != B200MOE_OK) return -1;
  return DecodeWorkspace(tokens, experts, top_k, inner, shared_inner).bytes;
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
      !a->workspace || fp8 != (a->w2_scale != nullptr) ||
      (a->shared_inner > 0 && (!a->shared_w13 || !a->shared_w2)))
    return B200MOE_ERR_ARG;
  if (fp8 && (a->width % 128 || a->inner % 128)) return B200MOE_ERR_ALIGN;
  for (const void* q : {a->x, a->router, a->w13, a->w2, a->shared_w13, a->shared_w2})
    if ((uintptr_t)q & 15) return B200MOE_ERR_ALIGN;
  if (((uintptr_t)a->workspace & 255) || ((uintptr_t)a->output & 1) || ((uintptr_t)a->residual & 1))
    return B200MOE_ERR_ALIGN;
  if (a->tokens == 0) return B200MOE_OK;

  const DecodeWorkspace w(a->tokens, a->experts, a->top_k, a->inner, a->shared_inner);
  char* base = reinterpret_cast<char*>(a->workspace);
  float* logits = reinterpret_cast<float*>(base + w.logits);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int code = a->router_is_fp32 ? launch_router<float>(a, logits, s) : launch_router<__nv_bfloat16>(a, logits, s);
  if (code != B200MOE_OK) return code;
  code = b200moe_route_topk(logits, a->experts, (int)a->tokens, a->experts, a->top_k, a->mode, a->bias, a->n_group,
                            a->topk_group, a->routed_scaling, a->route_weights, a->ids, stream);
  if (code != B200MOE_OK) return code;
  DecodeParams p = {};
  p.x = reinterpret_cast<const __nv_bfloat16*>(a->x);
  p.residual = reinterpret_cast<const __nv_bfloat16*>(a->residual);
  p.ids = a->ids;
  p.route_weights = a->route_weights;
  p.w13 = reinterpret_cast<const uint8_t*>(a->w13);
  p.w2 = reinterpret_cast<const uint8_t*>(a->w2);
  p.w13_scale = a->w13_scale;
  p.w2_scale = a->w2_scale;
  p.shared_w13 = reinterpret_cast<const uint8_t*>(a->shared_w13);
  p.shared_w2 = reinterpret_cast<const uint8_t*>(a->shared_w2);
  p.act = reinterpret_cast<__nv_bfloat16*>(base + w.act);
  p.act_shared = reinterpret_cast<__nv_bfloat16*>(base + w.act_shared);
  p.out = reinterpret_cast<__nv_bfloat16*>(a->output);
  p.T = (int)a->tokens, p.D = a->width, p.F = a->inner, p.E = a->experts, p.K = a->top_k;
  p.shared_inner = a->shared_inner;
  p.fp8 = fp8, p.limited = a->limited, p.limit = a->limit;
  p.b_rows = p.T < 8 ? 8 * p.T : 64;
  if (p.T <= 4) {
    code = launch_stream<false, 4>(p, s);
    return code != B200MOE_OK ? code : launch_stream<true, 4>(p, s);
  }
  code = launch_stream<false, 5>(p, s);
  return code != B200MOE_OK ? code : launch_stream<true, 5>(p, s);
}
