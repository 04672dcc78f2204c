// linear_ce.hip - softmax cross entropy of a linear classifier, value and gradient, tile by tile: the logits are never stored.
//
//   z_nv = x_n . W_v + b_v          lse_n = log sum_v exp z_nv
//   loss_n = lse_n - (1-e) z_n,t(n) - (e/V) sum_v z_nv               (label smoothing e; rows with ignore_index: 0)
//   dz_nv = g_n (exp(z_nv - lse_n) - (1-e) [v = t(n)] - e/V)
//   dx = dz W       dW = dz^T x      db = sum_n dz_n
//
// Matrix products, all of the time at sizes that matter; the matrix cores bound them:
//   forward     z = W x^T tile by tile (scores_kernel); the epilogue leaves a running maximum and a sum of exponentials per row and tile and,
//               for training, the exponentials in the operands' type (kKeepBytes)
//   backward    for a piece of the vocabulary: dz from the kept exponentials (kept_kernel, a memory pass) or, where there are none, from z
//               formed again; 16 bits for 16-bit inputs, the operand that the matrix instructions of the next two products take.  Then
//               dx += dz W[piece] and dW[piece] = dz^T x in one launch (gemm_tile)
// so a call holds one piece of dz (kPieceBytes) and what is kept, which is as large as logits of the operands' type up to kKeepBytes; a
// caller who would rather have the memory, or the one rounding less, says so (Y6_CE_RECOMPUTE).  A kept exponential is rounded and dz once more
// (twice u of a probability; the label's own entry has one rounding, from RowStat).  8192 rows x 131072 classes x 1024, bf16: 6.9-7.1 ms, 0.91 to
// 0.94 PFLOP/s over the three products; without the kept ones 8.2.  torch's product of such operands reaches 1.01 (K = 1024) to 1.29 (8192^3) on
// the same card, which lowers its clock under either.
// Labelled rows are gathered first (gather_kernel): rows with ignore_index cost nothing, and an infinity or a NaN in one of them reaches no
// gradient.  What the forward gathered, and its statistics, are kept for the backward.
//
// No atomics: partial statistics and split products are joined in a fixed order, the same inputs give the same bits.
#include <atomic>
#include <type_traits>

#include "common.hpp"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

constexpr unsigned kOob = 0xf0000000u;     // offset of a piece that must read zeros
constexpr size_t kPieceBytes = (size_t)128 << 20;     // of dz: half the last-level cache, and tiles enough to fill the chip
// Training keeps the forward's exponentials, in the operands' type, instead of forming the scores again, while they take at most kKeepBytes
// (below 1 % of the card's memory); what is behind that, by whole pieces, is formed again.  Measured with gradients and bias, formed again
// against kept, us.  bf16: 4096 rows x 16000 classes x 128 wide 207 -> 196, 256 249 -> 226, 384 320 -> 281, 8192 x 32000 x 64 645 -> 663; few
// classes leave lanes empty, 20000 x 600 x 256 111 -> 113; few scores are latency, 512 x 1000 x 512 45.7 -> 47.1, 1024 x 4001 x 256 61.8 -> 59.3.
// fp32, whose scores take six products: 4096 x 8000 x 64 264 -> 246, 2600 x 21000 x 256 907 -> 763, 512 x 1000 x 512 82 -> 75.
constexpr size_t kKeepBytes = (size_t)2 << 30;
constexpr long long kKeepWidth[2] = {128, 64}, kKeepClasses[2] = {1024, 512}, kKeepScores[2] = {1 << 22, 1 << 19};     // 16 bits, fp32
constexpr size_t kPartBytes = (size_t)256 << 20;      // of the tiles' statistics: the forward takes the rows in as many pieces
constexpr float kLog2e = 1.44269504088896340736f;
// dz of fp16 inputs is stored times 2^14 (|dz| <= 1 before): fp16's normal range then reaches down to 2^-28, below which a class
// adds nothing that fp16 gradients show.  bf16 and fp32 have the range.
constexpr float kHalfScale = 16384.f;
// Kept exponentials are relative to the largest of their tile; fp16 ones times 2^15, normal down to 2^-29 of it.

// Types: S of the caller's tensors; PLANES 16-bit operands (O) that stand for one value in LDS, RB bytes of each plane that a step takes
// from a row.  fp32 goes as three bf16 planes, h = the upper 8 significant bits, m = the next 8, l = the last 8: their sum is the value,
// exactly, and six of their nine products (the other three are below 2^-23 of the whole) on the bf16 matrix cores take 6 / 16 of what
// the fp32 ones take for the one.
struct Half {
    static constexpr int ES = 2, TYPE = Y6_F16, PLANES = 1, RB = 128;
    static constexpr float kScale = kHalfScale, kKeepExp = 15.f, kKeepUnit = 1.f / 32768;
    typedef _Float16 S;
    typedef _Float16 O;
    static __device__ __forceinline__ float get(S v) { return (float)v; }
    static __device__ __forceinline__ S put(float v) { return (S)v; }
};
struct Brain {
    static constexpr int ES = 2, TYPE = Y6_BF16, PLANES = 1, RB = 128;
    static constexpr float kScale = 1.f, kKeepExp = 0.f, kKeepUnit = 1.f;
    typedef __bf16 S;
    typedef __bf16 O;
    static __device__ __forceinline__ float get(S v) { return (float)v; }
    static __device__ __forceinline__ S put(float v) { return (S)v; }
};
struct Single {
    static constexpr int ES = 4, TYPE = Y6_F32, PLANES = 3, RB = 64;
    static constexpr float kScale = 1.f, kKeepExp = 0.f, kKeepUnit = 1.f;
    typedef float S;
    typedef __bf16 O;
    static __device__ __forceinline__ float get(S v) { return v; }
    static __device__ __forceinline__ S put(float v) { return v; }
};

// the planes of a value: cut, not rounded (a large value stays finite), so that each remainder is exact; an infinity or a NaN is the first
// plane's alone
__device__ __forceinline__ void split3(float v, unsigned short (&p)[3]) {
    const unsigned u = __float_as_uint(v);
    if ((u & 0x7f800000u) == 0x7f800000u) {
        p[0] = (unsigned short)((u >> 16) | ((u & 0xffffu) ? 0x40u : 0u));
        p[1] = p[2] = 0;
        return;
    }
    const unsigned h = u & 0xffff0000u;
    const float r = v - __uint_as_float(h);
    const unsigned m = __float_as_uint(r) & 0xffff0000u;
    const float q = r - __uint_as_float(m);
    p[0] = (unsigned short)(h >> 16), p[1] = (unsigned short)(m >> 16), p[2] = (unsigned short)(__float_as_uint(q) >> 16);
}

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_fast(float v) { return __builtin_amdgcn_logf(v); }

// ------------------------------------------------------------------------------------------------------------- rows with a label
// Block b of gather_kernel takes rows [16 b, 16 b + 16): finds how many labelled rows lie before them, then copies its labelled rows to
// their places, each padded with zeros to a multiple of 16 bytes, a row per wave.  Up to kCountRows rows it counts them itself (4 loads a
// thread at most).  Above, count_kernel counts kTotalRows rows a block and leaves each 16 rows' place within them and the block's total; a
// gather block's first wave adds up the totals before its own, 16 loads a lane at most, and with more than kTotals of them scan_kernel has
// done that once: the work grows with the rows (value of 2^20 rows x 8 x 2 classes, fp16, 0.49 ms, of 2^23 rows 3.80; with every block adding the
// counts of all blocks before it 0.89 and 30.7).
constexpr int kGatherRows = 16;
constexpr int kGatherThreads = kGatherRows * 64;
constexpr int kCountRows = 4096;
constexpr int kTotalRows = 1024;
constexpr int kTotals = 1024;

struct GatherArgs {
    const char* x;
    long long pitch;               // bytes
    const int64_t* target;
    long long ignore;
    int rows, width, classes;
    int vec;                       // rows start at 16-byte addresses, and 16-bit ones are multiples of 16 bytes
    const int* seg;                // above kCountRows rows: labelled rows before each 16 within their kTotalRows; or null
    const int* total;              // of each kTotalRows, or, `scanned`, of all before them
    int scanned;
    char* xc;
    long long cpitch, plane;       // bytes between rows, planes
    int* rowmap;                   // place -> row
    int* place;                    // row -> place, -1: no label
    int* label;                    // place -> label, -1: not a class
    int* count;
    float* loss_rows;              // 0 for rows without a label (reduction none), or null
};

__device__ __forceinline__ int block_count(int mine, int* sh) {       // sum over gather_kernel's threads
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) mine += __shfl_down(mine, d);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = mine;
    __syncthreads();
    int r = 0;
#pragma unroll
    for (int w = 0; w < kGatherRows; ++w) r += sh[w];
    return r;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {           // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

__global__ __launch_bounds__(256) void count_kernel(const int64_t* __restrict__ target, long long ignore, int rows, int* __restrict__ seg, int segs,
                                                    int* __restrict__ total) {
    constexpr int S = kTotalRows / kGatherRows;
    static_assert(S == 64, "one wave adds them up");
    __shared__ int n16[S];
    const int r0 = blockIdx.x * kTotalRows, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kTotalRows / 256; ++i) {
        const int k = i * 256 + threadIdx.x, r = rows - r0 > k ? r0 + k : -1;
        const unsigned long long m = __ballot(r >= 0 && target[r >= 0 ? r : 0] != ignore);
        if (lane % kGatherRows == 0) n16[k / kGatherRows] = __popcll((m >> lane) & ((1ull << kGatherRows) - 1));
    }
    __syncthreads();
    if (threadIdx.x >= S) return;
    const int mine = n16[lane], upto = wave_scan(mine, lane), s = r0 / kGatherRows + lane;
    if (s < segs) seg[s] = upto - mine;
    if (lane == S - 1) total[blockIdx.x] = upto;
}

// totals -> sums of those before each; one block, a chunk at a time
__global__ __launch_bounds__(1024) void scan_kernel(int* __restrict__ total, int n) {
    __shared__ int wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + threadIdx.x, mine = i < n ? total[i] : 0, upto = wave_scan(mine, lane);
        if (lane == 63) wave_sum[wave] = upto;
        __syncthreads();
        int before = carry + upto - mine, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        if (i < n) total[i] = before;
        carry += all;
        __syncthreads();
    }
}

// the planes of four values of a row, zeros behind its width
__device__ __forceinline__ void split_row4(const float* src, int c, int width, int vec, char* dst, long long plane) {
    float v[4];
    if (vec && c + 4 <= width) {
        const float4 f = *reinterpret_cast<const float4*>(src + c);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < width ? src[c + e] : 0.f;
    }
    unsigned short p[4][3];
#pragma unroll
    for (int e = 0; e < 4; ++e) split3(v[e], p[e]);
#pragma unroll
    for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint2*>(dst + k * plane + c * 2) = make_uint2(p[0][k] | (unsigned)p[1][k] << 16, p[2][k] | (unsigned)p[3][k] << 16);
}

template <int ES>
__global__ __launch_bounds__(kGatherThreads) void gather_kernel(const GatherArgs a) {
    __shared__ int sh[kGatherRows];
    __shared__ int place[kGatherRows];
    const int r0 = blockIdx.x * kGatherRows;
    int before = 0;
    if (!a.seg) {
        for (int i = threadIdx.x; i < r0; i += kGatherThreads) before += a.target[i] != a.ignore ? 1 : 0;
        before = block_count(before, sh);
    } else if (threadIdx.x < 64) {     // (only the first wave asks)
        const int c = r0 / kTotalRows, in = a.seg[blockIdx.x];
        if (a.scanned) {
            before = a.total[c];
        } else {
#pragma unroll 4
            for (int i = threadIdx.x; i < c; i += 64) before += a.total[i];
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
        }
        before += in;
    }
    if (threadIdx.x < 64) {
        const int r = r0 + threadIdx.x;
        const bool mine = threadIdx.x < kGatherRows && r < a.rows;
        const long long t = mine ? a.target[r] : a.ignore;
        const bool has = mine && t != a.ignore;
        const unsigned long long m = __ballot(has);
        const int p = before + __popcll(m & ((1ull << threadIdx.x) - 1));
        if (threadIdx.x < kGatherRows) place[threadIdx.x] = has ? p : -1;
        if (mine) a.place[r] = has ? p : -1;
        if (has) {
            a.rowmap[p] = r;
            a.label[p] = t >= 0 && t < a.classes ? (int)t : -1;
        } else if (mine && a.loss_rows) {
            a.loss_rows[r] = 0.f;
        }
        if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *a.count = before + __popcll(m);
    }
    __syncthreads();
    const int rows = a.rows - r0 < kGatherRows ? a.rows - r0 : kGatherRows;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (wave >= rows || place[wave] < 0) return;
    const char* const src = a.x + (long long)(r0 + wave) * a.pitch;
    char* const dst = a.xc + (long long)place[wave] * a.cpitch;
    if (ES == 4) {
        for (int c = lane * 4; c < a.cpitch / 2; c += 256) split_row4(reinterpret_cast<const float*>(src), c, a.width, a.vec, dst, a.plane);
    } else if (a.vec) {
        for (int o = lane * 16; o < a.width * 2; o += 1024) *reinterpret_cast<uint4*>(dst + o) = *reinterpret_cast<const uint4*>(src + o);
    } else {
#pragma unroll 8
        for (int e = lane; e < a.cpitch / 2; e += 64)
            reinterpret_cast<unsigned short*>(dst)[e] = e < a.width ? reinterpret_cast<const unsigned short*>(src)[e] : (unsigned short)0;
    }
}

// The planes of an fp32 weight
__global__ __launch_bounds__(256) void split_kernel(const char* __restrict__ src, long long pitch, int rows, int width, int vec, char* __restrict__ dst,
                                                    long long dpitch, long long plane) {
    const int q = (int)(dpitch / 8);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * q; i += (long long)gridDim.x * 256) {
        const long long r = i / q;
        split_row4(reinterpret_cast<const float*>(src + r * pitch), (int)(i - r * q) * 4, width, vec, dst + r * dpitch, plane);
    }
}

// Rows of a 16-bit weight padded with zeros to multiples of 16 bytes (its width or address is not one the wide loads take).  A thread writes 16
// bytes; where its elements are all there it reads the aligned 4-byte words that hold them and shifts, else element by element.
__global__ __launch_bounds__(256) void pad_kernel(const char* __restrict__ src, long long pitch, int rows, int width, char* __restrict__ dst,
                                                  long long dpitch) {
    typedef unsigned short U;
    const int q = (int)(dpitch / 16);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * q; i += (long long)gridDim.x * 256) {
        const long long r = i / q;
        const int c = (int)(i - r * q) * 8;
        const U* const s = reinterpret_cast<const U*>(src + r * pitch) + c;
        uint4 o;
        if (c + 8 < width && (r > 0 || c > 0)) {                      // (the words around them are the tensor's own)
            const unsigned sh = (unsigned)((uintptr_t)s & 2) * 8;
            const unsigned* const w = reinterpret_cast<const unsigned*>((uintptr_t)s & ~(uintptr_t)3);
            unsigned x[5];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = w[k];
            x[4] = sh ? w[4] : 0;
            o.x = __builtin_amdgcn_alignbit(x[1], x[0], sh), o.y = __builtin_amdgcn_alignbit(x[2], x[1], sh);
            o.z = __builtin_amdgcn_alignbit(x[3], x[2], sh), o.w = __builtin_amdgcn_alignbit(x[4], x[3], sh);
        } else {
            U e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = c + k < width ? s[k] : (U)0;
            __builtin_memcpy(&o, e, 16);
        }
        *reinterpret_cast<uint4*>(dst + r * dpitch + (long long)c * 2) = o;
    }
}

// --------------------------------------------------------------------------------------------------------------------- the product
__device__ __forceinline__ i32x4_t make_rsrc(const void* base, unsigned bytes) {
    const unsigned long long p = (unsigned long long)base;
    i32x4_t r;
    r[0] = (int)(unsigned)(p & 0xffffffffu);
    r[1] = (int)(unsigned)((p >> 32) & 0xffffu);   // stride 0: raw buffer, byte offsets, range check against the byte count
    r[2] = (int)bytes;
    r[3] = 0x00020000;
    return r;
}
// lane i: 16 bytes from rsrc.base + voff(lane) to lds_dst + 16 i; out of range: zeros.  The compiler does not count these requests;
// the kernel waits for them itself (vmcnt) in front of the barrier that hands the stage over.
__device__ __forceinline__ void dma16(const i32x4_t& rsrc, unsigned voff, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds_dst))
                 : "memory");
}
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)p; }

// One operand's tile of a stage: ROWS rows (of the result's m or n) by RB bytes of the reduction, for each plane an image.
//   KC (reduction contiguous in memory): image [row][RB], its 16-byte pieces permuted so that eight consecutive rows read the same
//      piece from eight different bank groups
//   else (rows of the reduction, m / n contiguous): image [32 columns][reduction RB / 2][64 B], read by the transposing ds_read_b64_tr_b16
template <class E, bool KC, int ROWS, int NW>
struct Operand {
    static constexpr int RB = E::RB, kPlane = ROWS * RB, kBytes = kPlane * E::PLANES;
    static constexpr int kInstr = kBytes / 1024;
    static constexpr int kPer = kInstr / NW;
    static constexpr int KS = RB / 2;                    // values of the reduction per stage
    static constexpr int kSubs = RB / 32;                // sub-steps of the matrix instructions per stage
    static_assert(kInstr % NW == 0 && kPlane % 1024 == 0, "requests divide over the waves and the planes");
    static_assert(RB == 128 || RB == 64, "eight or four pieces a row");

    static __device__ __forceinline__ int permuted(int row, int piece) { return RB == 128 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3); }

    // requests of the stage that starts at value k0 of the reduction; rows r0.. of `extent`, reduction `depth` long
    static __device__ __forceinline__ void issue(const char* base, long long pitch, long long plane, int r0, int extent, int k0, int depth, unsigned lds,
                                                 int wave, int lane) {
        const long long left = KC ? (long long)(extent - r0) * pitch : (long long)(depth - k0) * pitch;
        const char* const at = base + (KC ? (long long)r0 : (long long)k0) * pitch;
        const unsigned bytes = (unsigned)(left < kOob ? left : kOob);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int ins = wave * kPer + i;
            const int p = E::PLANES == 1 ? 0 : ins / (kPlane / 1024), in = E::PLANES == 1 ? ins : ins - p * (kPlane / 1024);
            const i32x4_t rs = make_rsrc(at + p * plane, bytes);
            unsigned voff;
            bool inside;
            if (KC) {
                const int lr = lane / (RB / 16);         // 1024 / RB rows a request
                const int kb = k0 * 2 + (permuted(lr, lane & (RB / 16 - 1)) << 4);
                inside = kb < depth * 2;
                voff = (unsigned)(in * (1024 / RB) + lr) * (unsigned)pitch + (unsigned)kb;
            } else {
                const int k = in % (RB / 32) * 16 + (lane >> 2), col = in / (RB / 32) * 32 + (lane & 3) * 8;
                inside = r0 + col < extent;
                voff = (unsigned)k * (unsigned)pitch + (unsigned)(r0 + col) * 2;
            }
            dma16(rs, inside ? voff : kOob, lds + ins * 1024);
        }
    }
    // plane p of the 32 rows from row f: lane's 16 bytes of sub-step kk, reduction values 16 kk + 8 (lane >> 5) + 0..7
    static __device__ __forceinline__ u32x4 frag(const char* img, int p, int f, int kk, int lane) {
        const int half = lane >> 5, l31 = lane & 31;
        img += p * kPlane;
        if (KC) {
            return *reinterpret_cast<const u32x4*>(img + (f + l31) * RB + (permuted(l31, kk * 2 + half) << 4));
        } else {
            const char* const q = img + (f >> 5) * (RB * 32) + (kk * 16 + half * 8 + ((lane & 15) >> 2)) * 64 + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(q));
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(q + 256));
            typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
            u32x4 r;
            r[0] = l2[0], r[1] = l2[1], r[2] = h2[0], r[3] = h2[1];
            return r;
        }
    }
};

template <class E>
__device__ __forceinline__ f32x16_t mma(const u32x4& a, const u32x4& b, f32x16_t c) {
    if constexpr (E::TYPE == Y6_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// acc += the products of sub-step kk of a stage; of three planes the six products that count, the small ones first
template <class E, class OA, class OB, int FM, int FN>
__device__ __forceinline__ void sub_step(f32x16_t (&acc)[FM][FN], const char* ia, const char* ib, int fm, int fn, int kk, int lane) {
    u32x4 fa[E::PLANES][FM], fb[E::PLANES][FN];
#pragma unroll
    for (int p = 0; p < E::PLANES; ++p) {
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[p][i] = OA::frag(ia, p, fm + i * 32, kk, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[p][j] = OB::frag(ib, p, fn + j * 32, kk, lane);
    }
#pragma unroll
    for (int order = E::PLANES - 1; order >= 0; --order)
#pragma unroll
        for (int p = 0; p <= order; ++p)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma<E>(fa[p][i], fb[order - p][j], acc[i][j]);
}

enum { EPI_STATS, EPI_KEEP, EPI_DZ };
enum { COUNT_N, COUNT_K };

// What the backward pass needs of a row's softmax: p_j = 2^((z_j - top) log2 e - log2s), s = sum exp(z_j - top), and 1 - p of the label from
// the others' sum.  Neither the loss, log(1 + sum over the others of exp(z_j - z_label)) where the label is the largest, nor its gradient
// p - 1 is a difference of large numbers then: a row that is almost right keeps its digits, at logits of any size.
struct RowStat {
    float top, log2s, miss;
};

struct GemmArgs {
    const char *a, *b;
    long long pa, pb, la, lb;      // bytes between rows, between planes
    int M, N, K;
    const int* count;              // labelled rows: the extent that COUNT says
    int row0;                      // scores: the first of these rows (b, label, stat ... start there)
    int tiles_m, tiles_n, splits;
    // scores: m = class, n = labelled row
    const void* bias;
    const int* label;
    float *part_m, *part_s, *part_z, *zt;
    long long np;                  // rows of the partial statistics' arrays
    const RowStat* stat;
    const float* coef;             // g_n / max |g| of the finite ones (null: 1)
    float smooth, smooth_share;    // e, e / V
    int class0;                    // first class of the piece
    char* keep;                    // EPI_KEEP: exponentials of the classes below `keeps`, by row
    long long keep_pitch;          // bytes
    int keeps;
    char* dz;
    long long dz_pitch, dz_plane;  // bytes
    // products into a gradient: m = column, n = row of the output
    float* part;                   // [split][N][part_pitch] or null: straight to out
    long long part_pitch;          // elements
    int add;                       // add to what the partial product holds
    char* out;
    long long out_pitch;           // elements
    const int *rowmap, *place;     // output row of row n, or null; rows of the output that no row n has get zeros
    const float *up, *gmax;        // the gradient's factor: *up [/ labelled rows], or *gmax
    int mean, vec;
};

// what every gradient is multiplied by at the end: the upstream gradient (over the labelled rows for a mean), or the largest of the
// rows' upstream gradients, and the inverse of dz's scale
template <class E>
__device__ __forceinline__ float grad_factor(const float* up, const float* gmax, int mean, const int* count) {
    float f = gmax ? *gmax : *up;
    if (mean) f = f / (float)(*count > 1 ? *count : 1);
    return f * (1.f / E::kScale);
}

// four operands of each plane
template <class E>
__device__ __forceinline__ void pack4(const float (&v)[4], uint2 (&r)[E::PLANES]) {
    if constexpr (E::PLANES == 1) {
        typedef typename E::O O4 __attribute__((ext_vector_type(4)));
        O4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (typename E::O)v[j];
        __builtin_memcpy(&r[0], &o, sizeof(uint2));
    } else {
        unsigned short p[4][3];
#pragma unroll
        for (int j = 0; j < 4; ++j) split3(v[j], p[j]);
#pragma unroll
        for (int k = 0; k < 3; ++k) r[k] = make_uint2(p[0][k] | (unsigned)p[1][k] << 16, p[2][k] | (unsigned)p[3][k] << 16);
    }
}
template <class E, bool VEC>
__device__ __forceinline__ void store4(char* dst, const float (&v)[4], int left) {
    typedef typename E::S S;
    S* const p = reinterpret_cast<S*>(dst);
    if (VEC && left >= 4) {
        typedef S S4 __attribute__((ext_vector_type(4)));
        S4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = E::put(v[j]);
        *reinterpret_cast<S4*>(p) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) p[j] = E::put(v[j]);
    }
}

// Tile of a block: BM x BN of the result over WM x WN waves, STAGES stages of the operands (ROW bytes a row) in LDS, BPC blocks per CU.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int BPC_, int ROW_ = 128>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, BPC = BPC_, NW = WM_ * WN_;
    static constexpr int kLds = STAGES_ * (BM_ + BN_) * ROW_;         // ROW: bytes of all planes of a row
    static_assert(kLds * BPC_ <= 160 * 1024, "LDS of a CU");
};

template <int N>
__device__ __forceinline__ void wait_requests() {       // all but the newest N requests of this wave have landed
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One block's tile of a product; `bid` of `8 * ceil(tiles / 8)` blocks.  Block b runs on XCD b % 8: each XCD takes one run of tiles, in
// groups of eight m-tiles by all n-tiles, so that the tiles it works on at one time share operand rows in its L2.
template <class E, bool AKC, bool BKC, class T, int COUNT>
__device__ __forceinline__ void gemm_tile(const GemmArgs& g, unsigned bid, char* smem) {
    constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN;
    constexpr int NW = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
    typedef Operand<E, AKC, BM, NW> OA;
    typedef Operand<E, BKC, BN, NW> OB;
    constexpr int kStage = OA::kBytes + OB::kBytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave % WM, wn = wave / WM;
    const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.splits;
    const int per = (total + 7) >> 3;
    const int t = (bid & 7) * per + (bid >> 3);
    if ((int)(bid >> 3) >= per || t >= total) return;
    const int split = t / tiles, tt = t - split * tiles;
    const int width = 8 * g.tiles_n, grp = tt / width, in = tt - grp * width;
    const int gm = g.tiles_m - grp * 8 < 8 ? g.tiles_m - grp * 8 : 8;
    const int tm = grp * 8 + in % gm, tn = in / gm;
    const int m0 = tm * BM, n0 = tn * BN;
    const int N = COUNT == COUNT_N ? *g.count : g.N, K = COUNT == COUNT_K ? *g.count : g.K;
    if (COUNT == COUNT_N && !g.part && N < g.N) {        // dx of rows n0.. without a label: zeros
        const int wide = g.M - m0 < BM ? g.M - m0 : BM;
        for (int r0 = n0; r0 < n0 + BN; r0 += 64) {
            const unsigned long long none = __ballot(r0 + lane < g.N && g.place[r0 + lane < g.N ? r0 + lane : 0] < 0);
            for (int k = wave; k < 64; k += NW)
                if (none >> k & 1)
                    for (int c = lane; c < wide; c += 64) reinterpret_cast<typename E::S*>(g.out)[(long long)(r0 + k) * g.out_pitch + m0 + c] = E::put(0.f);
        }
    }
    if (n0 >= N) return;
    const int steps = (K + OA::KS - 1) / OA::KS;
    const int s0 = (int)((long long)steps * split / g.splits), s1 = (int)((long long)steps * (split + 1) / g.splits);

    f32x16_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;

    const unsigned lds0 = lds_addr(smem);
    unsigned st_in = 0, st_out = 0;                      // stage the next requests fill, stage the next products read
    auto issue = [&](int s) {
        const unsigned st = lds0 + st_in;
        OA::issue(g.a, g.pa, g.la, m0, g.M, s * OA::KS, K, st, wave, lane);
        OB::issue(g.b, g.pb, g.lb, n0, N, s * OA::KS, K, st + OA::kBytes, wave, lane);
        st_in = st_in + kStage == T::STAGES * kStage ? 0 : st_in + kStage;
    };
    constexpr int kAhead = T::STAGES - 1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (s0 + i < s1) issue(s0 + i);
    for (int s = s0; s < s1; ++s) {
        // stage s has landed for every wave, and every wave has left the stage of s - 1, which the next requests overwrite
        if (kAhead > 1 && s + kAhead <= s1) wait_requests<(kAhead - 1) * (OA::kPer + OB::kPer)>();
        else wait_requests<0>();
        if (s + kAhead < s1) issue(s + kAhead);
        const char* const ia = smem + st_out;
        const char* const ib = ia + OA::kBytes;
        st_out = st_out + kStage == T::STAGES * kStage ? 0 : st_out + kStage;
#pragma unroll
        for (int kk = 0; kk < OA::kSubs; ++kk) sub_step<E, OA, OB, FM, FN>(acc, ia, ib, wm * (BM / WM), wn * (BN / WN), kk, lane);
    }

    // lane: row n = lane & 31 of a fragment; its 16 values are m = 8 (q >> 2) + 4 (lane >> 5) + (q & 3)
    const int half = lane >> 5, l31 = lane & 31;
    const int mw = m0 + wm * (BM / WM), nw = n0 + wn * (BN / WN);
    const float f = g.part ? 1.f : grad_factor<E>(g.up, g.gmax, g.mean, g.count);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = nw + j * 32 + l31;
        if (n >= N) continue;
        const long long row = !g.part && g.rowmap ? g.rowmap[n] : n;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int m = mw + i * 32 + 8 * gq + 4 * half;
                if (m >= g.M) continue;
                if (g.part) {
                    f32x4_t* const p = reinterpret_cast<f32x4_t*>(g.part + ((long long)split * g.N + n) * g.part_pitch + m);
                    f32x4_t v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * gq + e];
                    if (g.add) v += *p;
                    *p = v;
                } else {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * gq + e] * f;
                    char* const dst = g.out + (row * g.out_pitch + m) * E::ES;
                    if (g.vec) store4<E, true>(dst, v, g.M - m);
                    else store4<E, false>(dst, v, g.M - m);
                }
            }
    }
}

// The arguments once more, loaded where the epilogue uses them: taken from the parameter itself they stay in registers through the loop
// over the steps, and two dozen of them spill.
__device__ __forceinline__ GemmArgs args_again() {
    unsigned long long v = (unsigned long long)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(v));
    const __attribute__((address_space(4))) unsigned* const src = reinterpret_cast<const __attribute__((address_space(4))) unsigned*>(v);
    static_assert(sizeof(GemmArgs) % 4 == 0, "copied by dwords");
    GemmArgs r;
    unsigned* const dst = reinterpret_cast<unsigned*>(&r);
#pragma unroll
    for (unsigned i = 0; i < sizeof(GemmArgs) / 4; ++i) dst[i] = src[i];
    return r;
}

// The scores' product: z = W x^T tile by tile, with the statistics (EPI_STATS) or dz (EPI_DZ) as its epilogue; m = class, n = labelled row.
// A tile's reduction is short (the features' width: 16 steps at 1024), so what lies around it counts.  For dz a block stays and walks
// its tiles as one sequence of steps, the first loads of the next tile in flight while the last step of this one is multiplied and its
// dz stored: 16384 x 4096 x 1024 in 151 instead of 164 us.  (Keeping dz in registers to store it during the next tile spills, 203 us.)  The
// statistics lose that way, with their masks kept from spilling too (a training step of 4096 x 32000 x 1024 925 -> 1065 us): a block takes one tile.
template <class E, class T, int EPI>
__global__ __launch_bounds__(T::NW * 64, T::BPC * T::NW / 4) void scores_kernel(const GemmArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN;
    constexpr int NW = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;
    typedef Operand<E, true, BM, NW> OA;
    typedef Operand<E, true, BN, NW> OB;
    constexpr int kStage = OA::kBytes + OB::kBytes;
    constexpr bool kStay = EPI == EPI_DZ;
    typedef typename E::S S;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wm = wave % WM, wn = wave / WM;
    const int half = lane >> 5, l31 = lane & 31;
    const int N = *g.count - g.row0 < g.N ? *g.count - g.row0 : g.N, K = g.K;
    // (XCDs and groups of tiles: gemm_tile)
    const int total = g.tiles_m * g.tiles_n, per = (total + 7) >> 3;
    const int base = (blockIdx.x & 7) * per, stride = gridDim.x >> 3;
    const int end = base + per < total ? base + per : total;
    const int width = 8 * g.tiles_n;
    auto place = [&](int t, int& tm, int& tn) {
        const int grp = t / width, in = t - grp * width;
        const int gm = g.tiles_m - grp * 8 < 8 ? g.tiles_m - grp * 8 : 8;
        tn = in / gm;
        tm = grp * 8 + in - tn * gm;
    };
    auto next = [&](int t, int& tm, int& tn) {            // the block's first tile from t on that has rows; `end`: none
        for (; t < end; t += stride) {
            place(t, tm, tn);
            if (tn * BN < N) return t;
        }
        return end;
    };
    const int steps = (K + OA::KS - 1) / OA::KS;
    const unsigned lds0 = lds_addr(smem);
    unsigned st_in = 0, st_out = 0;
    int ptm = 0, ptn = 0, pt = next(base + (int)(blockIdx.x >> 3), ptm, ptn), ps = 0, ahead = 0;
    int tm = ptm, tn = ptn, t = pt;
    if (t >= end) return;
    auto issue = [&]() {                                  // requests of the sequence's next step, if there is one
        if (pt >= end) return;
        const unsigned st = lds0 + st_in;
        OA::issue(g.a, g.pa, g.la, ptm * BM, g.M, ps * OA::KS, K, st, wave, lane);
        OB::issue(g.b, g.pb, g.lb, ptn * BN, N, ps * OA::KS, K, st + OA::kBytes, wave, lane);
        st_in = st_in + kStage == T::STAGES * kStage ? 0 : st_in + kStage;
        ++ahead;
        if (++ps == steps) {
            ps = 0;
            pt = kStay ? next(pt + stride, ptm, ptn) : end;
        }
    };
    constexpr int kAhead = T::STAGES - 1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) issue();

    while (t < end) {
        f32x16_t acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
        for (int s = 0; s < steps; ++s) {
            // this step's stage has landed for every wave, and every wave has left the stage before, which the next requests overwrite
            // (stores in between only make the count stricter)
            if (kAhead > 1 && ahead == kAhead) wait_requests<(kAhead - 1) * (OA::kPer + OB::kPer)>();
            else wait_requests<0>();
            --ahead;
            issue();
            const char* const ia = smem + st_out;
            const char* const ib = ia + OA::kBytes;
            st_out = st_out + kStage == T::STAGES * kStage ? 0 : st_out + kStage;
#pragma unroll
            for (int kk = 0; kk < OA::kSubs; ++kk) sub_step<E, OA, OB, FM, FN>(acc, ia, ib, wm * (BM / WM), wn * (BN / WN), kk, lane);
        }
        const GemmArgs e = args_again();
        // lane: row n = lane & 31 of a fragment; its 16 values are m = 8 (q >> 2) + 4 (lane >> 5) + (q & 3)
        const int mw = tm * BM + wm * (BM / WM), nw = tn * BN + wn * (BN / WN);
        const bool whole = mw + BM / WM <= e.M;              // every class of this wave's tile is one
        if (e.bias) {
            const S* const bias = reinterpret_cast<const S*>(e.bias) + e.class0;
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int m = mw + i * 32 + 8 * (q >> 2) + 4 * half + (q & 3);
                    const float b = E::get(bias[m < e.M ? m : e.M - 1]);
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j][q] += b;
                }
        }
        if constexpr (EPI != EPI_DZ) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int n = nw + j * 32 + l31;
                const bool live = n < N;
                const long long o = (long long)(tm * WM + wm) * e.np + n;
                const int lab = live ? e.label[n] - mw : -1;
                int left = e.M - mw - 4 * half;              // classes of this lane's 4-runs: 32 i + 8 (q >> 2) + (q & 3) < left
                if (e.part_z) {
                    float zsum = 0.f;
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (whole || i * 32 + 8 * (q >> 2) + (q & 3) < left) zsum += acc[i][j][q];
                    }
                    zsum += __shfl_xor(zsum, 32);
                    if (live && half == 0) e.part_z[o] = zsum;
                }
                if (!whole) {
                    asm volatile("" : "+v"(left));           // (or the compiler forms all masks of all columns ahead, and they spill)
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (i * 32 + 8 * (q >> 2) + (q & 3) >= left) acc[i][j][q] = -INFINITY;
                    }
                }
                if (__ballot(lab >= 0 && lab < BM / WM)) {   // a label of these rows lies in this tile: few do
                    // its logit is handed on by itself and left out of the sum (RowStat)
                    int mine = lab - 4 * half;
                    asm volatile("" : "+v"(mine));
                    float z = 0.f;
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        __builtin_amdgcn_sched_barrier(0);   // (or all the comparisons come first, and their masks spill)
#pragma unroll
                        for (int q = 0; q < 16; ++q) z = mine == i * 32 + 8 * (q >> 2) + (q & 3) ? acc[i][j][q] : z;
                    }
                    if (mine >= 0 && mine < BM / WM && (mine & 4) == 0) e.zt[n] = z;
                    asm volatile("" : "+v"(mine));
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int q = 0; q < 16; ++q) acc[i][j][q] = mine == i * 32 + 8 * (q >> 2) + (q & 3) ? -INFINITY : acc[i][j][q];
                    }
                }
                float top = acc[0][j][0];
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int q = 0; q < 16; ++q) top = fmaxf(top, acc[i][j][q]);
                top = fmaxf(top, __shfl_xor(top, 32));
                // a tile says its largest logit and the sum of exp(z - it); one whose classes are all at -infinity says -infinity, 0
                float all;
                if (EPI == EPI_KEEP && tm * BM < e.keeps) {
                    const float ref = top == -INFINITY ? 0.f : top;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    char* const row = e.keep + (long long)n * e.keep_pitch + (long long)(mw + 4 * half) * E::ES;
                    int end16 = (int)(e.keep_pitch / E::ES) - mw - 4 * half;
                    asm volatile("" : "+v"(end16));
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int gp = 0; gp < 2; ++gp) {
                            __builtin_amdgcn_sched_barrier(0);
                            float v[2][4];
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int c4 = 0; c4 < 4; ++c4) {
                                    v[k][c4] = exp2_fast(fmaf(acc[i][j][8 * gp + 4 * k + c4] - ref, kLog2e, E::kKeepExp));
                                    sum[c4] += v[k][c4];
                                }
                            // (as dz: sixteen bytes a lane; the row is padded to them, and classes behind the last are zeros)
                            if constexpr (E::ES == 4) {
#pragma unroll
                                for (int k = 0; k < 2; ++k)
                                    if (live && i * 32 + 16 * gp + 8 * k < end16)
                                        *reinterpret_cast<float4*>(row + (i * 32 + 16 * gp + 8 * k) * 4) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
                            } else {
                                uint2 a[E::PLANES], b[E::PLANES];
                                pack4<E>(v[0], a);
                                pack4<E>(v[1], b);
                                const auto x = __builtin_amdgcn_permlane32_swap(a[0].x, b[0].x, false, false);
                                const auto y = __builtin_amdgcn_permlane32_swap(a[0].y, b[0].y, false, false);
                                if (live && i * 32 + 16 * gp + 4 * half < end16)
                                    *reinterpret_cast<uint4*>(row + (i * 32 + 16 * gp + 4 * half) * 2) = make_uint4(x[0], y[0], x[1], y[1]);
                            }
                        }
                    all = ((sum[0] + sum[1]) + (sum[2] + sum[3])) * E::kKeepUnit;
                    all += __shfl_xor(all, 32);
                } else {
                    float base = top == -INFINITY ? 0.f : top;
                    if (__ballot(!(fabsf(base) <= 1e38f))) {
                        // base log2 e would leave fp32's range (a tile whose classes a bias of the type's lowest value switches off): such rows
                        // have it subtracted first
                        const float far = fabsf(base) <= 1e38f ? 0.f : base;
#pragma unroll
                        for (int i = 0; i < FM; ++i) {
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int q = 0; q < 16; ++q) acc[i][j][q] -= far;
                        }
                        base = far == 0.f ? base : 0.f;
                    }
                    const float m2 = base * kLog2e;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int q = 0; q < 16; ++q) sum[q & 3] += exp2_fast(fmaf(acc[i][j][q], kLog2e, -m2));
                    all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    all += __shfl_xor(all, 32);
                    // (m2 was rounded: the terms are relative to it, the sum is not)
                    all = top == -INFINITY ? 0.f : all * exp2_fast(-fmaf(base, kLog2e, -m2));
                }
                if (live && half == 0) {
                    e.part_m[o] = top;
                    e.part_s[o] = all;
                }
            }
        } else if constexpr (EPI == EPI_DZ) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int n = nw + j * 32 + l31;
                const bool live = n < N;
                const int nl = live ? n : N - 1;
                const float zmax = e.stat[nl].top, log2s = e.stat[nl].log2s;
                const float c = (e.coef ? e.coef[nl] : 1.f) * E::kScale;
                const float share = -e.smooth_share * c, own = fmaf(-e.stat[nl].miss, c, fmaf(e.smooth, c, share));
                const int lab = e.label[nl] - e.class0 - mw - 4 * half;
                char* const row = e.dz + (long long)n * e.dz_pitch + (long long)(mw + 4 * half) * 2;
                const int left = e.M - mw - 4 * half;
                const int room = (int)(e.dz_pitch / 2) - mw - 4 * half;
                auto emit = [&](auto labelled, auto inside) {
                    int at = lab, to = left, end16 = room;
                    asm volatile("" : "+v"(at), "+v"(to), "+v"(end16));   // (or the compiler forms every mask ahead of the branches, and they spill)
#pragma unroll
                    for (int i = 0; i < FM; ++i)
#pragma unroll
                        for (int gp = 0; gp < 2; ++gp) {
                            if (labelled.value) __builtin_amdgcn_sched_barrier(0);
                            float v[2][4];
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int c4 = 0; c4 < 4; ++c4) {
                                    const int m = i * 32 + 16 * gp + 8 * k + c4;
                                    float d = fmaf(exp2_fast(fmaf(acc[i][j][8 * gp + 4 * k + c4] - zmax, kLog2e, -log2s)), c, share);
                                    if (labelled.value) d = m == at ? own : d;
                                    v[k][c4] = d;
                                }
                            uint2 a[E::PLANES], b[E::PLANES];
                            if (inside.value) {
                                // the half-waves trade runs of four classes: each lane then holds eight in a row, one 16-byte store
                                pack4<E>(v[0], a);
                                pack4<E>(v[1], b);
#pragma unroll
                                for (int p = 0; p < E::PLANES; ++p) {
                                    const auto x = __builtin_amdgcn_permlane32_swap(a[p].x, b[p].x, false, false);
                                    const auto y = __builtin_amdgcn_permlane32_swap(a[p].y, b[p].y, false, false);
                                    if (live) *reinterpret_cast<uint4*>(row + p * e.dz_plane + (i * 32 + 16 * gp + 4 * half) * 2) = make_uint4(x[0], y[0], x[1], y[1]);
                                }
                                continue;
                            }
                            // (the row is padded to 16 bytes: what lies behind the last class is zero, the reduction of dx runs over it; runs
                            // of four start at multiples of eight bytes, so a run is in the row or behind it)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int m = i * 32 + 16 * gp + 8 * k;
                                __builtin_amdgcn_sched_barrier(0);
                                if (!live || m >= end16) continue;
#pragma unroll
                                for (int c4 = 0; c4 < 4; ++c4)
                                    if (m + c4 >= to) v[k][c4] = 0.f;
                                pack4<E>(v[k], a);
#pragma unroll
                                for (int p = 0; p < E::PLANES; ++p) *reinterpret_cast<uint2*>(row + p * e.dz_plane + m * 2) = a[p];
                            }
                        }
                };
                if (!whole) emit(std::true_type{}, std::false_type{});
                else if (__ballot(lab >= -4 && lab < BM / WM)) emit(std::true_type{}, std::true_type{});   // a label of these rows lies in this tile: few do
                else emit(std::false_type{}, std::true_type{});
            }
        }
        if (!kStay) break;
        t = next(t + stride, tm, tn);
    }
}

template <class E, bool AKC, bool BKC, class T, int COUNT>
__global__ __launch_bounds__(T::NW * 64, T::BPC * T::NW / 4) void gemm_kernel(const GemmArgs g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    gemm_tile<E, AKC, BKC, T, COUNT>(g, blockIdx.x, smem);
}
// dx and dW of a piece in one launch: neither has tiles enough to fill the chip evenly, together they do (way_of_grads)
template <class E, class T>
__global__ __launch_bounds__(T::NW * 64, T::BPC * T::NW / 4) void grads_kernel(const GemmArgs x, const GemmArgs w, unsigned xblocks, int x_first) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const unsigned wblocks = gridDim.x - xblocks;
    const bool is_x = x_first ? blockIdx.x < xblocks : blockIdx.x >= wblocks;
    if (is_x) gemm_tile<E, false, true, T, COUNT_N>(x, x_first ? blockIdx.x : blockIdx.x - wblocks, smem);
    else gemm_tile<E, false, false, T, COUNT_K>(w, x_first ? blockIdx.x - xblocks : blockIdx.x, smem);
}

// ------------------------------------------------------------------------------------------------------------------- small kernels
// lse and loss of each labelled row: `places` rows (a power of two) x 1024 / places slices of the tiles' statistics per block: 32 rows
// read whole 128-byte lines, fewer rows are cut into more slices so that there are blocks enough
struct FinishArgs {
    const float *part_m, *part_s, *part_z, *zt;
    long long np;
    int parts, places, row0, rows; // of the labelled rows those from row0 on, `rows` of them (the pointers start there)
    const int *rowmap, *label, *count;
    float smooth, smooth_share;
    RowStat* stat;                 // by place
    float* rows_out;               // by row (reduction none) or null
    float* lossc;                  // by place, unless this is the only block
    float* loss;                   // the only block: the sum, or the mean
    int mean;
};
__global__ __launch_bounds__(1024) void finish_kernel(const FinishArgs a) {
    __shared__ float sm[1024], ss[1024], sz[1024];
    const int i = threadIdx.x & (a.places - 1), sl = threadIdx.x / a.places;
    int slices = 1024 / a.places;
    const int n = blockIdx.x * a.places + i, N = *a.count - a.row0 < a.rows ? *a.count - a.row0 : a.rows;
    float m = -INFINITY, s = 0.f, z = 0.f, zt = 0.f;      // largest logit but the label's; sum of exp(logit - m), the label's left out
    int label = 0, row = 0;
    if (n < N) {
        if (sl == 0) {                 // (asked for early: they are needed behind the last barrier)
            zt = a.zt[n], label = a.label[n];
            if (a.rows_out) row = a.rowmap[n];
        }
#pragma unroll 4
        for (int p = sl; p < a.parts; p += slices) {
            const float pm = a.part_m[(long long)p * a.np + n], ps = a.part_s[(long long)p * a.np + n];
            if (a.part_z) z += a.part_z[(long long)p * a.np + n];
            const float nm = fmaxf(m, pm), ref = nm == -INFINITY ? 0.f : nm;
            s = s * exp2_fast((m - ref) * kLog2e) + ps * exp2_fast((pm - ref) * kLog2e);
            m = nm;
        }
    }
    sm[threadIdx.x] = m, ss[threadIdx.x] = s, sz[threadIdx.x] = z;
    for (; slices > 1; slices >>= 1) {
        __syncthreads();
        if (sl < slices / 2) {
            const int o = threadIdx.x + slices / 2 * a.places;
            const float pm = sm[o], nm = fmaxf(m, pm), ref = nm == -INFINITY ? 0.f : nm;
            s = s * exp2_fast((m - ref) * kLog2e) + ss[o] * exp2_fast((pm - ref) * kLog2e);
            z += sz[o];
            m = nm;
            sm[threadIdx.x] = m, ss[threadIdx.x] = s, sz[threadIdx.x] = z;
        }
    }
    __syncthreads();
    float loss = 0.f;
    if (sl == 0 && n < N) {
        const float top = fmaxf(m, zt), rest = s * exp2_fast((m - top) * kLog2e), own = exp2_fast((zt - top) * kLog2e), sum = rest + own;
        loss = zt >= m ? log1pf(rest) * own : (m - zt) + logf(sum);      // (own is 1 there, or a NaN)
        if (a.smooth > 0.f) loss = (1.f - a.smooth) * loss + (a.smooth * (top + logf(sum)) - a.smooth_share * z);
        if (label < 0) loss = NAN;             // a label that is no class
        a.stat[n] = {top, label < 0 ? NAN : log2_fast(sum), rest / sum};
        if (a.rows_out) a.rows_out[row] = loss;
        if (a.lossc) a.lossc[n] = loss;
    }
    if (!a.loss) return;
    sm[threadIdx.x] = loss;
    __syncthreads();
    if (threadIdx.x) return;
    double all = 0;
    for (int k = 0; k < a.places; ++k) all += (double)sm[k];
    *a.loss = (float)(a.mean ? all / (N > 1 ? N : 1) : all);
}

__global__ __launch_bounds__(1024) void loss_sum_kernel(const float* __restrict__ lossc, const int* __restrict__ count, int mean, float* __restrict__ loss) {
    __shared__ double sh[16];
    const int N = *count;
    double s = 0;
    for (int i = threadIdx.x; i < N; i += 1024) s += (double)lossc[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) s += sh[w];
    *loss = (float)(mean ? s / (N > 1 ? N : 1) : s);
}

// reduction none: gmax = max |g| over the labelled rows whose g is finite (1 where all of those are zero), coef = g / gmax.  A g that is not
// finite stays with its row: its dz, hence its dx and the sums over rows, dW and db, are not finite; the other rows' dx do not see it.
__global__ __launch_bounds__(1024) void coef_kernel(const float* __restrict__ up, const int* __restrict__ rowmap, const int* __restrict__ count,
                                                    float* __restrict__ coef, float* __restrict__ gmax) {
    __shared__ float sh[16];
    const int N = *count;
    float top = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        const float v = fabsf(up[rowmap[i]]);
        top = v > top && v < INFINITY ? v : top;             // (comparisons with a NaN are false)
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
    __syncthreads();
    top = sh[0];
    for (int w = 1; w < 16; ++w) top = fmaxf(top, sh[w]);
    if (top == 0.f) top = 1.f;
    if (threadIdx.x == 0) *gmax = top;
    for (int i = threadIdx.x; i < N; i += 1024) coef[i] = up[rowmap[i]] / top;
}

// sum of the splits of a product, times the gradient's factor, rounded once
struct JoinArgs {
    const float* part;
    long long part_pitch, part_rows;   // part: [split][part_rows][part_pitch]
    int rows, width, splits;
    char* out;
    long long out_pitch;               // elements
    const int *place, *count;          // dx: row -> row of part, -1: zeros; or null
    const float *up, *gmax;
    int mean, vec;
};
template <class E>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
    const float f = grad_factor<E>(a.up, a.gmax, a.mean, a.count);
    const int q = (a.width + 3) >> 2;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)a.rows * q; i += (long long)gridDim.x * 256) {
        const int row = (int)(i / q), m = (int)(i - (long long)row * q) * 4;
        const int n = a.place ? a.place[row] : row;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
        if (n >= 0) {
            const float* const p = a.part + (long long)n * a.part_pitch + m;
#pragma unroll 8
            for (int k = 0; k < a.splits; ++k) s += *reinterpret_cast<const f32x4_t*>(p + (long long)k * a.part_rows * a.part_pitch);
        }
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = n >= 0 ? s[e] * f : 0.f;
        char* const dst = a.out + ((long long)row * a.out_pitch + m) * E::ES;
        if (a.vec) store4<E, true>(dst, v, a.width - m);
        else store4<E, false>(dst, v, a.width - m);
    }
}

// db of a piece: columns of dz summed over the labelled rows, blockIdx.y's share of them -> part[y][class].  A thread takes 16 bytes of
// a row, 32 threads 512 bytes, eight rows at a time.
constexpr int kBiasRows = 64;          // shares at most
constexpr int kBiasCols = 256;         // classes of a block
template <class E>
__global__ __launch_bounds__(256) void bias_part_kernel(const char* __restrict__ dz, long long pitch, long long plane, int classes,
                                                        const int* __restrict__ count, float* __restrict__ part, typename E::S* __restrict__ db,
                                                        const float* up, const float* gmax, int mean) {
    constexpr int V = 8;
    __shared__ float sh[8][32 * V + 1];
    const int N = *count, c = (blockIdx.x * 32 + (threadIdx.x & 31)) * V, w = threadIdx.x >> 5;
    const int r0 = (int)((long long)N * blockIdx.y / gridDim.y), r1 = (int)((long long)N * (blockIdx.y + 1) / gridDim.y);
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.f;
    if (c < classes) {                 // (rows are padded to 16 bytes)
#pragma unroll 4
        for (int r = r0 + w; r < r1; r += 8) {
            typedef typename E::O OV __attribute__((ext_vector_type(V)));
            float t[V];
#pragma unroll
            for (int p = E::PLANES - 1; p >= 0; --p) {
                const OV v = *reinterpret_cast<const OV*>(dz + p * plane + (long long)r * pitch + (long long)c * 2);
#pragma unroll
                for (int e = 0; e < V; ++e) t[e] = p == E::PLANES - 1 ? (float)v[e] : t[e] + (float)v[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += t[e];
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sh[w][(threadIdx.x & 31) * V + e] = s[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
        const int col = blockIdx.x * 32 * V + i;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += sh[k][i];
        if (col >= classes) continue;
        if (db) db[col] = E::put(t * grad_factor<E>(up, gmax, mean, count));       // the only share
        else part[(long long)blockIdx.y * classes + col] = t;
    }
}
// dz of a piece from the exponentials that the forward kept: dz = c (e 2^((tile's largest - top) log2 e - log2s) - share), the label's from
// its RowStat.  A wave takes 512 classes, 16 bytes a lane, and 4, 8 or 16 rows (layout), four at a time, so that it also has their sum, which
// becomes db: the block adds its four waves', in order.  Memory bounds it: 128 MB to 128 MB in 48-53 us, 5-5.3 TB/s, where forming the scores of
// 1024 features again took 150.  (32 rows a wave: 37 instead of 31 us at 1383 x 25088.)
constexpr int kKeptCols = 512;
struct KeptArgs {
    const char* e;                 // the piece's first class
    long long e_pitch;
    const float* part_m;           // [row piece][part][np]
    long long np;
    int parts, part_shift, stat_rows;
    const RowStat* stat;
    const float* coef;
    const int *label, *count;
    float smooth, smooth_share;
    int class0, classes, col_blocks, rows;   // rows: of a wave, a multiple of four
    char* dz;
    long long dz_pitch, dz_plane;
    float* bpart;                  // [block of rows][classes] or null
};
template <class E>
__global__ __launch_bounds__(256) void kept_kernel(const KeptArgs a) {
    __shared__ float sh[4][8][64];
    typedef typename E::S S4 __attribute__((ext_vector_type(E::ES == 4 ? 4 : 8)));     // 16 bytes
    constexpr int L = E::ES == 4 ? 2 : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int bx = blockIdx.x % a.col_blocks, by = blockIdx.x / a.col_blocks;
    const int N = *a.count, c0 = bx * kKeptCols + lane * 8, n0 = (by * 4 + wave) * a.rows;
    const bool mine = c0 * 2 < a.dz_pitch;
    const int part = (a.class0 + (mine ? c0 : 0)) >> a.part_shift;
    float sum[8] = {};
    constexpr int U = 4;
    for (int k = n0; k < n0 + a.rows && k < N; k += U) {
        S4 e[U][L];
        float pm[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int n = k + u < N ? k + u : N - 1;
#pragma unroll
            for (int l = 0; l < L; ++l)            // (read once: dz stays in the caches)
                e[u][l] = __builtin_nontemporal_load(reinterpret_cast<const S4*>(a.e + n * a.e_pitch + (mine ? c0 * E::ES : 0) + (mine ? l * 16 : 0)));
            pm[u] = a.part_m[((long long)(n / a.stat_rows) * a.parts + part) * a.np + n % a.stat_rows];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int n = k + u;
            if (n >= N) break;
            const RowStat st = a.stat[n];
            const float c = (a.coef ? a.coef[n] : 1.f) * E::kScale, share = -a.smooth_share * c;
            const float f = exp2_fast(fmaf(pm[u] - st.top, kLog2e, -st.log2s - E::kKeepExp)) * c, own = fmaf(-st.miss, c, fmaf(a.smooth, c, share));
            const int at = a.label[n] - a.class0 - c0;
            float d[2][4];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float v = fmaf((float)e[u][q * L / 8][q % (8 / L)], f, share);
                v = q == at ? own : c0 + q < a.classes ? v : 0.f;
                sum[q] += v;
                d[q / 4][q % 4] = v;
            }
            uint2 lo[E::PLANES], hi[E::PLANES];
            pack4<E>(d[0], lo);
            pack4<E>(d[1], hi);
#pragma unroll
            for (int p = 0; p < E::PLANES; ++p)
                if (mine) *reinterpret_cast<uint4*>(a.dz + p * a.dz_plane + n * a.dz_pitch + c0 * 2) = make_uint4(lo[p].x, lo[p].y, hi[p].x, hi[p].y);
        }
    }
    if (!a.bpart) return;
#pragma unroll
    for (int q = 0; q < 8; ++q) sh[wave][q][lane] = sum[q];
    __syncthreads();
    for (int i = threadIdx.x; i < kKeptCols; i += 256) {
        const int c = bx * kKeptCols + i;
        if (c < a.classes) a.bpart[(long long)by * a.classes + c] = (sh[0][i & 7][i >> 3] + sh[1][i & 7][i >> 3]) + (sh[2][i & 7][i >> 3] + sh[3][i & 7][i >> 3]);
    }
}

// db of a piece from its shares: 32 classes a block, 32 threads each, every one adds up each 32nd share, then the first their sums in order.
// (Shares grow with the rows, 4096 of them at 262144; classes of a piece may be 256: with one thread a class db took 250 of a call's 1394 us at
// 262144 rows x 128 x 1024 classes, so 52.)
constexpr int kJoinCols = 32;
template <class E>
__global__ __launch_bounds__(1024) void bias_join_kernel(const float* __restrict__ part, int shares, int classes, typename E::S* __restrict__ db,
                                                         const float* up, const float* gmax, int mean, const int* count) {
    __shared__ float sh[1024 / kJoinCols][kJoinCols];
    const int lane = threadIdx.x % kJoinCols, w = threadIdx.x / kJoinCols;
    const float f = grad_factor<E>(up, gmax, mean, count);
    for (int c0 = blockIdx.x * kJoinCols; c0 < classes; c0 += gridDim.x * kJoinCols) {
        const int c = c0 + lane;
        float s = 0.f;
        if (c < classes) {
#pragma unroll 8
            for (int k = w; k < shares; k += 1024 / kJoinCols) s += part[(long long)k * classes + c];
        }
        sh[w][lane] = s;
        __syncthreads();
        if (w == 0 && c < classes) {
#pragma unroll
            for (int k = 1; k < 1024 / kJoinCols; ++k) s += sh[k][lane];
            db[c] = E::put(s * f);
        }
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------------------------------------------------- host side
int type_bytes(int t) { return t == Y6_F32 ? 4 : 2; }
long long up_to(long long v, long long m) { return (v + m - 1) / m * m; }
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// ---- tiles.  kBig: 256 x 256, eight waves, one block per CU.  kMid: 128 x 128, four waves, two blocks per CU: a quarter of the tile for
// what kBig leaves unfilled, and its epilogue hides behind the other block.  kSmall: 64 x 64 with three stages in flight: 64 rows x 1000 classes x
// 512 in 6.0 us against kMid's 9.1, one row x 32000 classes x 1024 in 12.1 against 14.8.  The three planes of fp32 fill LDS sooner: one block
// of 128 x 128 per CU.
typedef Tile<256, 256, 2, 4, 2, 1> BigScores;     // waves 2 x 4: a lane's row has 128 classes (32000 x 4096 x 1024 statistics 262 us, 4 x 2: 300)
typedef Tile<256, 256, 4, 2, 2, 1> BigGrads;      // dx, dW: 4 x 2: 1.20 PFLOP/s, 2 x 4: 1.15 (8192 x 8192 x 2048)
typedef Tile<128, 128, 2, 2, 2, 2> Mid;           // dx, dW 1.04 PFLOP/s; the same statistics 280 us
typedef Tile<64, 64, 2, 2, 4, 2> Small;
typedef Tile<128, 128, 2, 4, 3, 1, 192> MidSplit;     // eight waves of 64 x 32: 4096 x 8192 x 2048 with gradients 2.93 ms, four of 64 x 64: 3.21
typedef Tile<64, 64, 2, 2, 3, 2, 192> SmallSplit;
enum { kBig, kMid, kSmall, kTiles };
constexpr int kSide[kTiles] = {256, 128, 64};
constexpr int kSlots[2][kTiles] = {{256, 512, 512}, {1, 256, 512}};
constexpr int kWavesM[kTiles] = {BigScores::WM, Mid::WM, Small::WM};
static_assert(MidSplit::WM == Mid::WM && SmallSplit::WM == Small::WM, "parts of the statistics");
// microseconds of one step of a block (64 values of the reduction, of fp32 32), alone on its CU and beside another, and of its first loads
// and its epilogue (measured)
constexpr double kStepAlone[2][kTiles] = {{1.85, 0.75, 0.38}, {1e9, 1.35, 0.5}};
constexpr double kStepFull[2][kTiles] = {{1.85, 1.05, 0.5}, {1e9, 1.4, 1.05}};
constexpr double kEnds[kTiles] = {4.0, 2.0, 1.5};
constexpr double kBytesPerUs = 4e6;

double block_us(int tile, bool fp32, long long steps, long long blocks) {
    return (blocks <= 256 ? kStepAlone : kStepFull)[fp32][tile] * steps + kEnds[tile];
}
// the tile for M x N x `steps` without splits: the one whose rounds of blocks take least
int way_of_scores(bool fp32, long long m, long long n, long long steps) {
    int best = kMid;
    double least = 1e300;
    for (int t = fp32 ? kMid : kBig; t < kTiles; ++t) {
        const long long blocks = (long long)ceil_div(m, kSide[t]) * ceil_div(n, kSide[t]);
        const double us = ceil_div(blocks, kSlots[fp32][t]) * block_us(t, fp32, steps, blocks);
        if (us < least) least = us, best = t;
    }
    return best;
}
struct GradWay {
    int tile, split_x, split_w;
    double us;
};
// Tile and splits of a piece's dx (width x rows, reduction `classes`) and dW (width x classes, reduction `rows`) in one launch: the long
// blocks go first, the short ones fill up behind them; splits cost the traffic of their partial products.
GradWay way_of_grads(bool fp32, bool dx, bool dw, long long rows, long long width, long long classes, int pieces) {
    const int ks = fp32 ? 32 : 64;
    const long long kx = ceil_div(classes, ks), kw = ceil_div(rows, ks);
    GradWay best = {kMid, 1, 1, 1e300};
    for (int t = fp32 ? kMid : kBig; t < kTiles; ++t)
        for (int sx = 1; sx <= (dx ? 32 : 1) && (sx == 1 || kx / sx >= 4); sx *= 2)
            for (int sw = 1; sw <= (dw ? 32 : 1) && (sw == 1 || kw / sw >= 4); sw *= 2) {
                const long long wide = ceil_div(width, kSide[t]);
                const long long bx = dx ? wide * ceil_div(rows, kSide[t]) * sx : 0, bw = dw ? wide * ceil_div(classes, kSide[t]) * sw : 0;
                double ux = block_us(t, fp32, ceil_div(kx, sx), bx + bw), uw = block_us(t, fp32, ceil_div(kw, sw), bx + bw);
                long long nl = bx, ns = bw;
                if (uw > ux) {
                    const double u = ux;
                    ux = uw, uw = u, nl = bw, ns = bx;
                }
                const long long p = kSlots[fp32][t], q = nl / p, r = nl % p;
                double us;
                const long long fill = r ? (p - r) * (long long)(ux / uw) : 0;
                if (ns <= fill) us = (q + (r ? 1 : 0)) * ux;
                else us = (q + (r ? 1 : 0)) * ux + ceil_div(ns - fill, p) * uw;
                if (dx && (sx > 1 || pieces > 1)) us += (pieces > 1 ? 2.0 : 1.0) * rows * width * 4 * sx / kBytesPerUs;
                if (dx && sx > 1 && pieces == 1) us += 4 + 1.0 * rows * width * 4 * sx / kBytesPerUs;
                if (dw && sw > 1) us += 4 + 2.0 * classes * width * 4 * sw / kBytesPerUs;
                if (us < best.us) best = {t, sx, sw, us};
            }
    return best;
}

struct Layout {
    size_t xc, wc, rowmap, place, label, count, stat, kept;                           // what the backward takes over from the forward
    size_t exps, kept_m, kept_all;                                                    // and, if it comes, these
    size_t seg, part_m, part_s, part_z, zt, lossc;                                    // forward's workspace
    size_t coef, gmax, dz, accx, accw, bpart;                                         // backward's
    size_t bytes;
    long long cpitch, np;              // bytes between rows of the gathered features, of the weight's copy; rows
    int planes, scores, parts, places, stat_rows, piece, pieces, shares;
    int keeps, kept_scores, kept_rows; // classes whose exponentials are kept (whole pieces), by tiles of this kind; rows of a kept_kernel wave
    long long keep_pitch;              // bytes
    GradWay grads;
    long long px, pw;
    bool copy_w;                       // the weight is used from a copy: padded, or its planes
};

Layout layout(const y6_linear_ce_desc* d, bool backward) {
    Layout L = {};
    const int es = type_bytes(d->dtype);
    const bool fp32 = d->dtype == Y6_F32;
    const long long n = d->rows, v = d->classes, w = d->width;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    };
    L.planes = fp32 ? 3 : 1;
    L.cpitch = up_to(w * 2, 16);
    L.copy_w = (d->flags & Y6_CE_COPY_WEIGHT) || fp32 || (w * es) % 16 != 0 || (d->w_pitch * es) % 16 != 0 || (uintptr_t)d->weight % 16 != 0;
    L.xc = take((size_t)n * L.cpitch * L.planes);
    L.wc = take(L.copy_w ? (size_t)v * L.cpitch * L.planes : 0);
    L.rowmap = take((size_t)n * 4);
    L.place = take((size_t)n * 4);
    L.label = take((size_t)n * 4);
    L.stat = take((size_t)n * sizeof(RowStat));
    L.count = take(4);
    L.kept = at;
    const long long steps = ceil_div(w, fp32 ? 32 : 64);
    // the backward's pieces: of equal size, whole tiles, of about kPieceBytes of dz or, where the blocks of the gradients' products come
    // out that much more evenly, twice that: the caches then hold less of it (8192 x 131072 x 1024: 7.24 ms, with 256 MB 7.47; 4096 x
    // 32000: 967 us, in one piece of 262 MB 942)
    auto cut = [&](long long bytes, int* count, int* size) {
        const long long pieces = (long long)(((size_t)n * v * 2 * L.planes + bytes - 1) / bytes);
        const long long piece = up_to((v + pieces - 1) / pieces, 256);
        *size = (int)(piece < v ? piece : v);
        *count = ceil_div(v, *size);
    };
    cut(kPieceBytes, &L.pieces, &L.piece);
    if (L.pieces > 1) {
        int count, size;
        cut(2 * kPieceBytes, &count, &size);
        auto us = [&](int count, int size) {
            return (count - 1) * way_of_grads(fp32, true, true, n, w, size, count).us + way_of_grads(fp32, true, true, n, w, v - (count - 1ll) * size, count).us;
        };
        if (1.05 * us(count, size) < us(L.pieces, L.piece)) L.pieces = count, L.piece = size;
    }
    const long long piece = L.piece;
    // the forward's tiles and statistics
    L.kept_scores = way_of_scores(fp32, v, n, steps);
    L.parts = ceil_div(v, kSide[L.kept_scores]) * kWavesM[L.kept_scores];
    long long rows = (long long)(kPartBytes / ((size_t)L.parts * 8)) / 256 * 256;
    if (rows < 256) rows = 256;
    L.stat_rows = (int)(rows < n ? rows : n);
    L.np = up_to(L.stat_rows, 64);
    if (!(d->flags & Y6_CE_RECOMPUTE) && w >= kKeepWidth[fp32] && v >= kKeepClasses[fp32] && n * v >= kKeepScores[fp32]) {
        const long long most = (long long)(kKeepBytes / ((size_t)n * piece * es));
        L.keeps = (int)(most >= L.pieces ? v : most * piece);
    }
    // (a wave of kept_kernel takes 16 rows, fewer where four blocks a CU would not come together: 1024 x 4001 in fp32 22 us with 16)
    L.kept_rows = 16;
    while (L.kept_rows > 4 && (long long)ceil_div(n, 4 * L.kept_rows) * ceil_div(L.piece, kKeptCols) < 1024) L.kept_rows /= 2;
    L.keep_pitch = up_to((long long)L.keeps, 8) * es;
    L.exps = take((size_t)n * L.keep_pitch);
    L.kept_m = take(L.keeps ? (size_t)ceil_div(n, L.stat_rows) * L.parts * L.np * 4 : 0);
    L.kept_all = at;
    at = 0;
    if (!backward) {
        L.seg = take(n > kCountRows ? ((size_t)ceil_div(n, kGatherRows) + ceil_div(n, kTotalRows)) * 4 : 0);
        L.scores = L.kept_scores;
        // one block for all rows, which then also adds up the loss, where that is 16 rounds of its threads at most
        L.places = 1;
        while (L.places < n && L.places < 128) L.places *= 2;
        if (L.places < n || (long long)L.places * L.parts > 16 * 1024) L.places = n >= 8192 ? 32 : n >= 64 ? 8 : 1;
        L.part_m = take(d->saved && L.keeps ? 0 : (size_t)L.parts * L.np * 4);
        L.part_s = take((size_t)L.parts * L.np * 4);
        L.part_z = take(d->smoothing > 0.f ? (size_t)L.parts * L.np * 4 : 0);
        L.zt = take((size_t)n * 4);
        L.lossc = take((size_t)n * 4);
    } else {
        L.scores = way_of_scores(fp32, piece, n, steps);
        L.grads = way_of_grads(fp32, d->dx != nullptr, d->dw != nullptr, n, w, piece, L.pieces);
        L.px = L.pw = up_to(w, 4);
        L.shares = n <= 256 ? 1 : n < kBiasRows * 64 ? ceil_div(n, 64) : kBiasRows;
        L.coef = take((size_t)n * 4);
        L.gmax = take(4);
        L.dz = take((size_t)n * up_to(piece * 2, 16) * L.planes);
        L.accx = take(d->dx && (L.pieces > 1 || L.grads.split_x > 1) ? (size_t)L.grads.split_x * n * L.px * 4 : 0);
        L.accw = take(d->dw && L.grads.split_w > 1 ? (size_t)L.grads.split_w * piece * L.pw * 4 : 0);
        const int kept_shares = L.keeps ? ceil_div(n, 4 * L.kept_rows) : 0;
        L.bpart = take(d->dbias ? (size_t)(L.shares > kept_shares ? L.shares : kept_shares) * piece * 4 : 0);
    }
    L.bytes = at;
    return L;
}

// A launch has less than 2^32 threads: gather_kernel's 1024 for 16 rows, scores_kernel's 256 for 64 classes of few rows.
constexpr long long kMaxThreads = (1ll << 32) - 1;
constexpr long long kMaxRows = kMaxThreads / kGatherThreads * kGatherRows, kMaxClasses = kMaxThreads / 256 / 8 * 8 * kSide[kSmall];

int check_desc(const y6_linear_ce_desc* d, const char* what) {
    Y6_REQUIRE(d, "%s: null argument", what);
    Y6_REQUIRE(d->dtype == Y6_F16 || d->dtype == Y6_BF16 || d->dtype == Y6_F32, "%s: dtype %d (fp16, bf16 or fp32)", what, d->dtype);
    Y6_REQUIRE(d->rows >= 1 && d->rows <= kMaxRows && d->classes >= 1 && d->classes <= kMaxClasses && d->width >= 1 && d->width <= (1 << 20),
               "%s: %lld rows x %d wide, %d classes", what, (long long)d->rows, d->width, d->classes);
    Y6_REQUIRE(d->x && d->weight && d->target, "%s: null argument", what);
    Y6_REQUIRE(d->x_pitch >= 0 && d->w_pitch >= d->width && d->w_pitch <= (1 << 21), "%s: pitches %lld, %lld", what, (long long)d->x_pitch, (long long)d->w_pitch);
    Y6_REQUIRE(d->reduction == Y6_REDUCE_NONE || d->reduction == Y6_REDUCE_SUM || d->reduction == Y6_REDUCE_MEAN, "%s: reduction %d", what, d->reduction);
    Y6_REQUIRE(d->smoothing >= 0.f && d->smoothing <= 1.f, "%s: label smoothing %g", what, (double)d->smoothing);
    const uintptr_t es = type_bytes(d->dtype);
    Y6_REQUIRE(((uintptr_t)d->x | (uintptr_t)d->weight | (uintptr_t)d->bias | (uintptr_t)d->dx | (uintptr_t)d->dw | (uintptr_t)d->dbias) % es == 0,
               "%s: a tensor is not aligned to its elements", what);
    return Y6_OK;
}

struct Run {
    const y6_linear_ce_desc* d;
    const Layout& L;
    char *keep, *ws;
    hipStream_t s;
    template <class T>
    T* kept(size_t o) const { return reinterpret_cast<T*>(keep + o); }
    template <class T>
    T* at(size_t o) const { return reinterpret_cast<T*>(ws + o); }
};

template <class E>
int launch_gather(const Run& r) {
    const y6_linear_ce_desc* d = r.d;
    GatherArgs a = {};
    a.x = (const char*)d->x, a.pitch = d->x_pitch * E::ES, a.target = d->target, a.ignore = d->ignore_index;
    a.rows = (int)d->rows, a.width = d->width, a.classes = d->classes;
    a.vec = (E::ES == 4 || (d->width * E::ES) % 16 == 0) && a.pitch % 16 == 0 && (uintptr_t)d->x % 16 == 0;
    a.xc = r.kept<char>(r.L.xc), a.cpitch = r.L.cpitch, a.plane = d->rows * r.L.cpitch;
    a.rowmap = r.kept<int>(r.L.rowmap), a.place = r.kept<int>(r.L.place), a.label = r.kept<int>(r.L.label), a.count = r.kept<int>(r.L.count);
    const int segs = ceil_div(d->rows, kGatherRows);
    if (d->rows > kCountRows) {
        const int totals = ceil_div(d->rows, kTotalRows);
        int* const total = r.at<int>(r.L.seg) + segs;
        a.seg = r.at<int>(r.L.seg), a.total = total, a.scanned = totals > kTotals;
        hipLaunchKernelGGL(count_kernel, dim3(totals), dim3(256), 0, r.s, d->target, (long long)d->ignore_index, a.rows, r.at<int>(r.L.seg), segs, total);
        Y6_LAUNCH_CHECK();
        if (a.scanned) {
            hipLaunchKernelGGL(scan_kernel, dim3(1), dim3(1024), 0, r.s, total, totals);
            Y6_LAUNCH_CHECK();
        }
    }
    if (d->reduction == Y6_REDUCE_NONE) a.loss_rows = d->loss;
    hipLaunchKernelGGL(gather_kernel<E::ES>, dim3(segs), dim3(kGatherThreads), 0, r.s, a);
    Y6_LAUNCH_CHECK();
    if (r.L.copy_w) {
        const long long blocks = (d->classes * (r.L.cpitch / (E::ES == 4 ? 8 : 16)) + 255) / 256;
        const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
        const int vec = (d->w_pitch * E::ES) % 16 == 0 && (uintptr_t)d->weight % 16 == 0;
        if (E::ES == 4)
            hipLaunchKernelGGL(split_kernel, grid, dim3(256), 0, r.s, (const char*)d->weight, d->w_pitch * E::ES, d->classes, d->width, vec, r.kept<char>(r.L.wc),
                               r.L.cpitch, d->classes * r.L.cpitch);
        else
            hipLaunchKernelGGL(pad_kernel, grid, dim3(256), 0, r.s, (const char*)d->weight, d->w_pitch * E::ES, d->classes, d->width, r.kept<char>(r.L.wc), r.L.cpitch);
        Y6_LAUNCH_CHECK();
    }
    return Y6_OK;
}

// (raising a kernel's LDS limit is idempotent: threads that get here together all do it)
int raise_lds(const void* kern, int lds, std::atomic<unsigned long long>& raised) {
    if (lds <= 64 * 1024) return Y6_OK;
    int dev = 0;
    Y6_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !(raised.load(std::memory_order_acquire) >> dev & 1)) {
        Y6_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        if (dev < 64) raised.fetch_or(1ull << dev, std::memory_order_release);
    }
    return Y6_OK;
}
template <class T>
int set_tiles(GemmArgs& g, unsigned* blocks) {
    g.tiles_m = ceil_div(g.M, T::BM), g.tiles_n = ceil_div(g.N, T::BN);
    if (g.splits < 1) g.splits = 1;
    const long long total = (long long)g.tiles_m * g.tiles_n * g.splits;
    Y6_REQUIRE((total + 7) / 8 * 8 * (T::NW * 64) <= kMaxThreads, "linear_ce: %lld tiles", total);
    *blocks = (unsigned)((total + 7) / 8 * 8);
    return Y6_OK;
}
template <class E, bool AKC, bool BKC, class T, int COUNT>
int launch_tile(GemmArgs& g, hipStream_t s) {
    static std::atomic<unsigned long long> raised{0};
    auto* const kern = gemm_kernel<E, AKC, BKC, T, COUNT>;
    unsigned blocks = 0;
    int rc = set_tiles<T>(g, &blocks);
    if (rc == Y6_OK) rc = raise_lds((const void*)kern, T::kLds, raised);
    if (rc != Y6_OK) return rc;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(T::NW * 64), T::kLds, s, g);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}
template <class E, class T, int EPI>
int launch_scores_tile(GemmArgs& g, hipStream_t s) {
    static std::atomic<unsigned long long> raised{0};
    auto* const kern = scores_kernel<E, T, EPI>;
    unsigned blocks = 0;
    int rc = set_tiles<T>(g, &blocks);
    if (rc == Y6_OK) rc = raise_lds((const void*)kern, T::kLds, raised);
    if (rc != Y6_OK) return rc;
    if (EPI == EPI_DZ && blocks > 256u * T::BPC) blocks = 256u * T::BPC;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(T::NW * 64), T::kLds, s, g);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}
template <class E, int EPI>
int launch_scores(int tile, GemmArgs& g, hipStream_t s) {
    if constexpr (E::PLANES == 3) {
        return tile == kSmall ? launch_scores_tile<E, SmallSplit, EPI>(g, s) : launch_scores_tile<E, MidSplit, EPI>(g, s);
    } else {
        return tile == kSmall ? launch_scores_tile<E, Small, EPI>(g, s) : tile == kMid ? launch_scores_tile<E, Mid, EPI>(g, s) : launch_scores_tile<E, BigScores, EPI>(g, s);
    }
}
template <class E, class T>
int launch_grads_tile(GemmArgs* x, GemmArgs* w, hipStream_t s) {
    if (!w) return launch_tile<E, false, true, T, COUNT_N>(*x, s);
    if (!x) return launch_tile<E, false, false, T, COUNT_K>(*w, s);
    static std::atomic<unsigned long long> raised{0};
    auto* const kern = grads_kernel<E, T>;
    unsigned bx = 0, bw = 0;
    int rc = set_tiles<T>(*x, &bx);
    if (rc == Y6_OK) rc = set_tiles<T>(*w, &bw);
    if (rc != Y6_OK) return rc;
    Y6_REQUIRE(((long long)bx + bw) * (T::NW * 64) <= kMaxThreads, "linear_ce: %lld tiles", (long long)bx + bw);
    rc = raise_lds((const void*)kern, T::kLds, raised);
    if (rc != Y6_OK) return rc;
    hipLaunchKernelGGL(kern, dim3(bx + bw), dim3(T::NW * 64), T::kLds, s, *x, *w, bx, x->K / x->splits >= w->K / w->splits ? 1 : 0);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}
template <class E>
int launch_grads(int tile, GemmArgs* x, GemmArgs* w, hipStream_t s) {
    if constexpr (E::PLANES == 3) {
        return tile == kSmall ? launch_grads_tile<E, SmallSplit>(x, w, s) : launch_grads_tile<E, MidSplit>(x, w, s);
    } else {
        return tile == kSmall ? launch_grads_tile<E, Small>(x, w, s) : tile == kMid ? launch_grads_tile<E, Mid>(x, w, s) : launch_grads_tile<E, BigGrads>(x, w, s);
    }
}

#define Y6_TRY(expr)                     \
    do {                                 \
        const int _rc = (expr);          \
        if (_rc != Y6_OK) return _rc;    \
    } while (0)

template <class E>
int forward(const Run& r) {
    const y6_linear_ce_desc* d = r.d;
    const Layout& L = r.L;
    Y6_TRY(launch_gather<E>(r));
    GemmArgs g = {};
    g.a = L.copy_w ? r.kept<char>(L.wc) : (const char*)d->weight;
    g.pa = L.copy_w ? L.cpitch : d->w_pitch * E::ES;
    g.pb = L.cpitch;
    g.la = d->classes * L.cpitch, g.lb = d->rows * L.cpitch;
    g.M = d->classes, g.K = d->width;
    g.count = r.kept<int>(L.count), g.bias = d->bias;
    g.part_m = r.at<float>(L.part_m), g.part_s = r.at<float>(L.part_s), g.part_z = d->smoothing > 0.f ? r.at<float>(L.part_z) : nullptr;
    g.np = L.np;
    const bool keeps = d->saved && L.keeps;
    g.keeps = L.keeps, g.keep_pitch = L.keep_pitch;
    FinishArgs f = {};
    f.part_m = g.part_m, f.part_s = g.part_s, f.part_z = g.part_z, f.np = L.np, f.parts = L.parts, f.places = L.places;
    f.count = g.count;
    f.smooth = d->smoothing, f.smooth_share = d->smoothing / d->classes;
    f.mean = d->reduction == Y6_REDUCE_MEAN ? 1 : 0;
    const bool sums = d->reduction != Y6_REDUCE_NONE, alone = d->rows <= L.places && L.stat_rows == d->rows;
    for (long long n0 = 0; n0 < d->rows; n0 += L.stat_rows) {
        g.row0 = f.row0 = (int)n0;
        g.N = f.rows = (int)(d->rows - n0 < L.stat_rows ? d->rows - n0 : L.stat_rows);
        g.b = r.kept<char>(L.xc) + n0 * L.cpitch;
        g.label = f.label = r.kept<int>(L.label) + n0;
        g.zt = r.at<float>(L.zt) + n0, f.zt = g.zt;
        if (keeps) {
            g.part_m = r.kept<float>(L.kept_m) + n0 / L.stat_rows * (L.parts * L.np), f.part_m = g.part_m;
            g.keep = r.kept<char>(L.exps) + n0 * L.keep_pitch;
        }
        Y6_TRY((keeps ? launch_scores<E, EPI_KEEP>(L.scores, g, r.s) : launch_scores<E, EPI_STATS>(L.scores, g, r.s)));
        f.rowmap = r.kept<int>(L.rowmap) + n0;
        f.stat = r.kept<RowStat>(L.stat) + n0;
        if (!sums) f.rows_out = d->loss;
        else if (alone) f.loss = d->loss;
        else f.lossc = r.at<float>(L.lossc) + n0;
        hipLaunchKernelGGL(finish_kernel, dim3(ceil_div(g.N, L.places)), dim3(1024), 0, r.s, f);
        Y6_LAUNCH_CHECK();
    }
    if (sums && !alone) {
        hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, r.s, r.at<float>(L.lossc), f.count, f.mean, d->loss);
        Y6_LAUNCH_CHECK();
    }
    return Y6_OK;
}

template <class E>
int backward(const Run& r) {
    const y6_linear_ce_desc* d = r.d;
    const Layout& L = r.L;
    const int* const count = r.kept<int>(L.count);
    const int* const place = r.kept<int>(L.place);
    const float *gmax = nullptr, *coef = nullptr;
    if (d->reduction == Y6_REDUCE_NONE) {
        hipLaunchKernelGGL(coef_kernel, dim3(1), dim3(1024), 0, r.s, d->grad_out, r.kept<int>(L.rowmap), count, r.at<float>(L.coef), r.at<float>(L.gmax));
        Y6_LAUNCH_CHECK();
        gmax = r.at<float>(L.gmax), coef = r.at<float>(L.coef);
    }
    const int mean = d->reduction == Y6_REDUCE_MEAN ? 1 : 0;
    const char* const w = L.copy_w ? r.kept<char>(L.wc) : (const char*)d->weight;
    const long long wp = L.copy_w ? L.cpitch : d->w_pitch * E::ES, wl = d->classes * L.cpitch, xl = d->rows * L.cpitch;
    char* const dz = r.at<char>(L.dz);
    const bool accx = L.pieces > 1 || L.grads.split_x > 1;
    const int split_x = L.grads.split_x, split_w = L.grads.split_w;
    for (int p = 0; p < L.pieces; ++p) {
        const int v0 = p * L.piece, vn = d->classes - v0 < L.piece ? d->classes - v0 : L.piece;
        GemmArgs g = {};
        g.a = w + v0 * wp, g.pa = wp, g.la = wl, g.b = r.kept<char>(L.xc), g.pb = L.cpitch, g.lb = xl;
        g.M = vn, g.N = (int)d->rows, g.K = d->width, g.count = count;
        g.label = r.kept<int>(L.label), g.bias = d->bias, g.class0 = v0;
        g.stat = r.kept<RowStat>(L.stat), g.coef = coef;
        g.smooth = d->smoothing, g.smooth_share = d->smoothing / d->classes;
        g.dz = dz, g.dz_pitch = up_to((long long)vn * 2, 16), g.dz_plane = d->rows * g.dz_pitch;
        const bool kept = v0 < L.keeps;
        int shares = L.shares;
        if (kept) {
            KeptArgs k = {};
            k.e = r.kept<char>(L.exps) + (long long)v0 * E::ES, k.e_pitch = L.keep_pitch;
            k.part_m = r.kept<float>(L.kept_m), k.np = L.np, k.parts = L.parts, k.stat_rows = L.stat_rows;
            k.part_shift = __builtin_ctz(kSide[L.kept_scores] / kWavesM[L.kept_scores]);
            k.stat = g.stat, k.coef = coef, k.label = g.label, k.count = count, k.smooth = g.smooth, k.smooth_share = g.smooth_share;
            k.col_blocks = ceil_div(g.dz_pitch, kKeptCols * 2);
            k.class0 = v0, k.classes = vn, k.dz = dz, k.dz_pitch = g.dz_pitch, k.dz_plane = g.dz_plane;
            k.rows = L.kept_rows, shares = ceil_div(d->rows, 4 * k.rows);
            if (d->dbias) k.bpart = r.at<float>(L.bpart);
            hipLaunchKernelGGL(kept_kernel<E>, dim3((unsigned)(k.col_blocks * shares)), dim3(256), 0, r.s, k);
            Y6_LAUNCH_CHECK();
        }
        if (!kept) Y6_TRY((launch_scores<E, EPI_DZ>(L.scores, g, r.s)));
        if (d->dbias) {
            auto* const db = (typename E::S*)d->dbias + v0;
            if (!kept) {
            hipLaunchKernelGGL(bias_part_kernel<E>, dim3(ceil_div(vn, kBiasCols), L.shares), dim3(256), 0, r.s, dz, g.dz_pitch, g.dz_plane, vn, count,
                               r.at<float>(L.bpart), L.shares == 1 ? db : nullptr, d->grad_out, gmax, mean);
            Y6_LAUNCH_CHECK();
            }
            if (kept || shares > 1) {
                hipLaunchKernelGGL(bias_join_kernel<E>, dim3(vn < 65536 * kJoinCols ? ceil_div(vn, kJoinCols) : 65536), dim3(1024), 0, r.s, r.at<float>(L.bpart), shares, vn, db, d->grad_out, gmax,
                                   mean, count);
                Y6_LAUNCH_CHECK();
            }
        }
        GemmArgs x = {}, y = {};
        x.a = w + v0 * wp, x.pa = wp, x.la = wl, x.b = dz, x.pb = g.dz_pitch, x.lb = g.dz_plane;
        x.M = d->width, x.N = (int)d->rows, x.K = vn, x.count = count, x.splits = split_x;
        x.up = d->grad_out, x.gmax = gmax, x.mean = mean;
        if (accx) {
            x.part = r.at<float>(L.accx), x.part_pitch = L.px, x.add = p > 0;
        } else {
            x.out = (char*)d->dx, x.out_pitch = d->width, x.rowmap = r.kept<int>(L.rowmap), x.place = place;
            x.vec = d->width % 4 == 0 && (uintptr_t)d->dx % (4 * E::ES) == 0;
        }
        y.a = r.kept<char>(L.xc), y.pa = L.cpitch, y.la = xl, y.b = dz, y.pb = g.dz_pitch, y.lb = g.dz_plane;
        y.M = d->width, y.N = vn, y.K = (int)d->rows, y.count = count, y.splits = split_w;
        y.up = d->grad_out, y.gmax = gmax, y.mean = mean;
        char* const dw = (char*)d->dw + (long long)v0 * d->width * E::ES;
        const int vec = d->width % 4 == 0 && (uintptr_t)d->dw % (4 * E::ES) == 0;
        if (split_w > 1) y.part = r.at<float>(L.accw), y.part_pitch = L.pw;
        else y.out = dw, y.out_pitch = d->width, y.vec = vec;
        if (d->dx || d->dw) Y6_TRY(launch_grads<E>(L.grads.tile, d->dx ? &x : nullptr, d->dw ? &y : nullptr, r.s));
        if (d->dw && split_w > 1) {
            JoinArgs j = {};
            j.part = y.part, j.part_pitch = L.pw, j.part_rows = vn, j.rows = vn, j.width = d->width, j.splits = split_w;
            j.out = dw, j.out_pitch = d->width, j.count = count, j.up = d->grad_out, j.gmax = gmax, j.mean = mean, j.vec = vec;
            const long long need = ((long long)vn * ((d->width + 3) / 4) + 255) / 256;
            hipLaunchKernelGGL(join_kernel<E>, dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, r.s, j);
            Y6_LAUNCH_CHECK();
        }
    }
    if (d->dx && accx) {
        JoinArgs j = {};
        j.part = r.at<float>(L.accx), j.part_pitch = L.px, j.part_rows = d->rows, j.rows = (int)d->rows, j.width = d->width, j.splits = split_x;
        j.out = (char*)d->dx, j.out_pitch = d->width, j.place = place, j.count = count;
        j.up = d->grad_out, j.gmax = gmax, j.mean = mean;
        j.vec = d->width % 4 == 0 && (uintptr_t)d->dx % (4 * E::ES) == 0;
        const long long need = (d->rows * ((d->width + 3) / 4) + 255) / 256;
        hipLaunchKernelGGL(join_kernel<E>, dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, r.s, j);
        Y6_LAUNCH_CHECK();
    }
    return Y6_OK;
}

}  // namespace

// ====================================================================== C ABI
extern "C" size_t y6_linear_ce_saved_bytes(const y6_linear_ce_desc* d) {
    if (check_desc(d, "linear_ce_saved_bytes") != Y6_OK) return 0;
    return layout(d, false).kept_all;
}

extern "C" size_t y6_linear_ce_workspace_bytes(const y6_linear_ce_desc* d, int backward_pass) {
    if (check_desc(d, "linear_ce_workspace_bytes") != Y6_OK) return 0;
    const Layout L = layout(d, backward_pass != 0);
    return L.bytes + (backward_pass || d->saved ? 0 : L.kept);
}

static int check_buffers(const y6_linear_ce_desc* d, const Layout& L, size_t need, const char* what) {
    Y6_REQUIRE(d->workspace && d->workspace_bytes >= need && (uintptr_t)d->workspace % 16 == 0, "%s: workspace of %zu bytes, %zu needed", what,
               d->workspace_bytes, need);
    Y6_REQUIRE(!d->saved || (d->saved_bytes >= L.kept_all && (uintptr_t)d->saved % 16 == 0), "%s: saved holds %zu bytes, %zu needed", what, d->saved_bytes, L.kept_all);
    return Y6_OK;
}

extern "C" int y6_linear_ce_forward(const y6_linear_ce_desc* d, void* stream) {
    Y6_CLEAR_STALE_ERROR();
    Y6_TRY(check_desc(d, "linear_ce_forward"));
    Y6_REQUIRE(d->loss, "linear_ce_forward: null argument");
    const Layout L = layout(d, false);
    Y6_TRY(check_buffers(d, L, L.bytes + (d->saved ? 0 : L.kept), "linear_ce_forward"));
    const Run r = {d, L, d->saved ? (char*)d->saved : (char*)d->workspace + L.bytes, (char*)d->workspace, (hipStream_t)stream};
    return d->dtype == Y6_F16 ? forward<Half>(r) : d->dtype == Y6_BF16 ? forward<Brain>(r) : forward<Single>(r);
}

extern "C" int y6_linear_ce_backward(const y6_linear_ce_desc* d, void* stream) {
    Y6_CLEAR_STALE_ERROR();
    Y6_TRY(check_desc(d, "linear_ce_backward"));
    Y6_REQUIRE(d->saved && d->grad_out, "linear_ce_backward: null argument");
    if (!d->dx && !d->dw && !d->dbias) return Y6_OK;
    const Layout L = layout(d, true);
    Y6_TRY(check_buffers(d, L, L.bytes, "linear_ce_backward"));
    const Run r = {d, L, (char*)d->saved, (char*)d->workspace, (hipStream_t)stream};
    return d->dtype == Y6_F16 ? backward<Half>(r) : d->dtype == Y6_BF16 ? backward<Brain>(r) : backward<Single>(r);
}
