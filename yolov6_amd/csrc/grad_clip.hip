// grad_clip.hip - the global norm of many gradient tensors, their clipping, and the clipped SGD step over the parameter arena.
//
//   norm = (sum_i g_i^2)^(1/2) | sum_i |g_i| | max_i |g_i|   over all elements of all tensors
//   c    = min(1, max_norm / (norm + 1e-6))                  g_i <- c g_i
//
// Bound by HBM: the norm has to be known before the first element is written, so every gradient is read twice and written once
// (the second reading meets the 256 MB last-level cache where the gradients fit it).  Two launches for up to kTable tensors: partial
// sums, then the scaling, whose blocks each add the partial sums again in the same fixed order (at most kJoin of them, out of L2: a
// third launch to add them once costs more).  No atomics: the same gradients give the same bits.
//
// Measured: 489 fp32 tensors of 29.5 M elements (118 MB).  The norm's two launches (330 and 159 tensors) 19 and 10 us, 4.1 TB/s although the data
// lies in the last-level cache: a thread asks for 64 bytes, converts and adds them, and only then asks for more.  The scaling's two 34 and 19 us
// where they write (236 MB read and written, 4.4 TB/s), 4-5 each where the factor is 1 and they read no gradient.  The call: the norm alone
// 33 us, clipped 103, not clipped 57-67.  112 M parameters stepped with a clipped gradient 549 us, 2.8 GB at 5.1 TB/s, what a copy of 1 GB
// reaches (the norm's part 449 MB in 120 us, 3.7 TB/s); 40 tensors of at most 5000 elements 14 us, two launches and their host side.
//
// Squares and sums are doubles: the square of an fp32 / bf16 gradient leaves the range of a float (1e20, 1e-23), the sum of 1e8
// of them its precision, and the conversions hide behind the loads.  No sum of fp32 squares reaches infinity in double: the
// norm is non-finite exactly when a gradient is, which is the overflow check of the loss scaler for free.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.hpp"

namespace {

constexpr int kTable = 330;            // entries per launch: the table rides in the kernel's arguments (no upload, safe to capture)
constexpr int kThreads = 256;
constexpr int kChunk = 16384;          // bytes a block takes of one tensor at a time: four 16-byte loads in flight per thread
constexpr int kBlocks = 1024;          // four blocks per CU: 64 KB of loads in flight on each
constexpr int kJoin = 4096;            // partial sums that every block adds by itself; more are added by one block in between
constexpr long long kEntry = 1ll << 30;                // elements of one entry; a larger tensor is several

// 12 bytes an entry, 4 KB in all: 489 gradients (YOLOv6-L) are two launches of each kernel, not four
struct Table {
    unsigned long long at[kTable];     // the address, its type in the upper two bits
    unsigned n[kTable];                // elements
    int count;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

// An entry as the loads see it: its address rounded down to 16 bytes, the first and the last byte from there
struct Entry {
    char* base;
    unsigned head, type;
    unsigned long long end;
};
__host__ __device__ __forceinline__ Entry entry(unsigned long long at, unsigned n) {
    Entry e;
    e.type = (unsigned)(at >> 62);
    const unsigned long long p = at & ((1ull << 62) - 1);
    e.head = (unsigned)(p & 15);
    e.base = (char*)(p - e.head);
    e.end = e.head + (unsigned long long)n * (e.type == Y6_F32 ? 4 : 2);
    return e;
}
__host__ __device__ __forceinline__ unsigned chunks_of(unsigned long long at, unsigned n) {
    return (unsigned)((entry(at, n).end + kChunk - 1) / kChunk);
}

union Vec {
    uint4 v;
    float f[4];
    _Float16 h[8];
    unsigned short s[8];
};

__device__ __forceinline__ float bf16_value(unsigned short s) { return __uint_as_float((unsigned)s << 16); }
__device__ __forceinline__ unsigned short bf16_round(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40);          // NaN stays NaN
    return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);                          // to nearest, ties to even
}

// the 16 bytes at `off`; what lies outside the tensor reads as zero and is not touched
template <int TYPE>
__device__ __forceinline__ Vec load_vec(const char* base, unsigned long long off, unsigned head, unsigned long long end) {
    constexpr int ES = TYPE == Y6_F32 ? 4 : 2;
    Vec r;
    if (off >= head && off + 16 <= end) {
        r.v = *reinterpret_cast<const uint4*>(base + off);
        return r;
    }
    r.v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 16 / ES; ++e) {
        const unsigned long long o = off + e * ES;
        if (o >= head && o < end) {
            if (ES == 4) r.f[e] = *reinterpret_cast<const float*>(base + o);
            else r.s[e] = *reinterpret_cast<const unsigned short*>(base + o);
        }
    }
    return r;
}
template <int TYPE>
__device__ __forceinline__ void store_vec(char* base, unsigned long long off, unsigned head, unsigned long long end, const Vec& r) {
    constexpr int ES = TYPE == Y6_F32 ? 4 : 2;
    if (off >= head && off + 16 <= end) {
        *reinterpret_cast<uint4*>(base + off) = r.v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 16 / ES; ++e) {
        const unsigned long long o = off + e * ES;
        if (o >= head && o < end) {
            if (ES == 4) *reinterpret_cast<float*>(base + o) = r.f[e];
            else *reinterpret_cast<unsigned short*>(base + o) = r.s[e];
        }
    }
}
template <int TYPE>
__device__ __forceinline__ float vec_get(const Vec& r, int e) {
    return TYPE == Y6_F32 ? r.f[e] : TYPE == Y6_F16 ? (float)r.h[e] : bf16_value(r.s[e]);
}

// a NaN stays: comparisons with it are false
template <int NORM>
__device__ __forceinline__ double join(double a, double b) {
    if (NORM == Y6_NORM_INF) return (b > a || b != b) ? b : a;
    return a + b;
}
template <int NORM>
__device__ __forceinline__ double block_join(double v, double* sh) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = join<NORM>(v, __shfl_down(v, d));
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) sh[wave] = v;
    __syncthreads();
    double r = sh[0];
    for (int w = 1; w < kThreads / 64; ++w) r = join<NORM>(r, sh[w]);
    return r;                          // every thread has it
}
template <int NORM>
__device__ __forceinline__ double add_parts(const double* parts, int n, double* sh) {
    double s = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) s = join<NORM>(s, parts[i]);
    s = block_join<NORM>(s, sh);
    return NORM == Y6_NORM_L2 ? sqrt(s) : s;
}
__device__ __forceinline__ double any_norm(int norm, const double* parts, int n, double* sh) {
    return norm == Y6_NORM_L2 ? add_parts<Y6_NORM_L2>(parts, n, sh) : norm == Y6_NORM_L1 ? add_parts<Y6_NORM_L1>(parts, n, sh)
                                                                                         : add_parts<Y6_NORM_INF>(parts, n, sh);
}
// min(1, max_norm / (norm + 1e-6)); a NaN norm stays one
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.f : (float)c;
}

template <int NORM, int TYPE>
__device__ __forceinline__ double chunk_part(const char* base, unsigned long long at, unsigned head, unsigned long long end) {
    Vec r[kChunk / 16 / kThreads];
#pragma unroll
    for (int i = 0; i < kChunk / 16 / kThreads; ++i) {
        const unsigned long long off = at + (unsigned long long)(i * kThreads + threadIdx.x) * 16;
        r[i].v = make_uint4(0, 0, 0, 0);
        if (off < end) r[i] = load_vec<TYPE>(base, off, head, end);
    }
    double a = 0;
#pragma unroll
    for (int i = 0; i < kChunk / 16 / kThreads; ++i)
#pragma unroll
        for (int e = 0; e < (TYPE == Y6_F32 ? 4 : 8); ++e) {
            const double g = (double)vec_get<TYPE>(r[i], e);
            if (NORM == Y6_NORM_L2) a = fma(g, g, a);
            else a = join<NORM>(a, fabs(g));
        }
    return a;
}
template <int TYPE>
__device__ __forceinline__ void chunk_scale(char* base, unsigned long long at, unsigned head, unsigned long long end, float c) {
    Vec r[kChunk / 16 / kThreads];
#pragma unroll
    for (int i = 0; i < kChunk / 16 / kThreads; ++i) {
        const unsigned long long off = at + (unsigned long long)(i * kThreads + threadIdx.x) * 16;
        if (off < end) r[i] = load_vec<TYPE>(base, off, head, end);
    }
#pragma unroll
    for (int i = 0; i < kChunk / 16 / kThreads; ++i) {
        const unsigned long long off = at + (unsigned long long)(i * kThreads + threadIdx.x) * 16;
        if (off >= end) continue;
#pragma unroll
        for (int e = 0; e < (TYPE == Y6_F32 ? 4 : 8); ++e) {
            const float v = vec_get<TYPE>(r[i], e) * c;          // one rounding to the gradient's type
            if (TYPE == Y6_F32) r[i].f[e] = v;
            else if (TYPE == Y6_F16) r[i].h[e] = (_Float16)v;
            else r[i].s[e] = bf16_round(v);
        }
        store_vec<TYPE>(base, off, head, end, r[i]);
    }
}

// f(entry, byte offset of the chunk) for each of the block's chunks; all blocks together move over the tensors as one window.  Every block
// adds up the entries' chunks for itself (two entries a thread).
template <class F>
__device__ __forceinline__ void for_chunks(const Table& tb, F f) {
    static_assert(kTable <= 2 * kThreads, "two entries a thread");
    __shared__ unsigned first[2 * kThreads + 1], wave_sum[kThreads / 64];
    const int i = threadIdx.x * 2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned c0 = i < tb.count ? chunks_of(tb.at[i], tb.n[i]) : 0, c1 = i + 1 < tb.count ? chunks_of(tb.at[i + 1], tb.n[i + 1]) : 0;
    unsigned sum = c0 + c1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned v = __shfl_up(sum, d);
        if (lane >= d) sum += v;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sum += wave_sum[w];
    first[i + 1] = sum - c1;
    first[i + 2] = sum;
    if (threadIdx.x == 0) first[0] = 0;
    __syncthreads();
    const unsigned total = first[2 * kThreads];
    int lo = 0;
    for (unsigned c = blockIdx.x; c < total; c += gridDim.x) {
        int hi = tb.count;             // first[lo] <= c < first[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= c) lo = mid;
            else hi = mid;
        }
        const int t = __builtin_amdgcn_readfirstlane(lo);
        f(entry(tb.at[t], tb.n[t]), (unsigned long long)(c - first[lo]) * kChunk);
    }
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void grad_part_kernel(const Table tb, double* __restrict__ parts) {
    __shared__ double sh[kThreads / 64];
    double a = 0;
    for_chunks(tb, [&](const Entry& e, unsigned long long at) {
        a = join<NORM>(a, e.type == Y6_F32   ? chunk_part<NORM, Y6_F32>(e.base, at, e.head, e.end)
                          : e.type == Y6_F16 ? chunk_part<NORM, Y6_F16>(e.base, at, e.head, e.end)
                                             : chunk_part<NORM, Y6_BF16>(e.base, at, e.head, e.end));
    });
    a = block_join<NORM>(a, sh);
    if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

// the sum of the partial sums back to parts[n], or the norm itself
__global__ __launch_bounds__(kThreads) void grad_join_kernel(int norm, double* parts, int n, float* out) {
    __shared__ double sh[kThreads / 64];
    const double v = any_norm(norm, parts, n, sh);
    if (threadIdx.x) return;
    if (out) *out = (float)v;
    else parts[n] = norm == Y6_NORM_L2 ? v * v : v;
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(const Table tb, int norm, const double* __restrict__ parts, int nparts, double max_norm,
                                                              float* __restrict__ out) {
    __shared__ double sh[kThreads / 64];
    const double v = any_norm(norm, parts, nparts, sh);
    if (out && blockIdx.x == 0 && threadIdx.x == 0) *out = (float)v;
    const float c = clip_factor(v, max_norm);
    if (c == 1.f) return;              // nothing to clip: x * 1 is x, bit for bit
    for_chunks(tb, [&](const Entry& e, unsigned long long at) {
        if (e.type == Y6_F32) chunk_scale<Y6_F32>(e.base, at, e.head, e.end, c);
        else if (e.type == Y6_F16) chunk_scale<Y6_F16>(e.base, at, e.head, e.end, c);
        else chunk_scale<Y6_BF16>(e.base, at, e.head, e.end, c);
    });
}

struct ClipSgd {
    float* p;
    const float* g;
    float* m;
    const uint8_t* group;
    size_t n;
    float lr[4], wd[4];
    float mom, grad_mul;
    int nesterov, first, nparts;
    const float* scale;
    int32_t* found_inf;
    const double* parts;
    double max_norm;
    float* out;
};

__device__ __forceinline__ float decayed(float d, float wd, float p) {
#pragma clang fp contract(off)
    return d + wd * p;
}

// sgd_grouped_kernel's step (train.hip) with the clipping factor in the gradient's multiplier: the clipped gradients are never
// written.  Four elements per thread and request.
__global__ __launch_bounds__(kThreads) void sgd_clipped_kernel(const ClipSgd a) {
    __shared__ double sh[kThreads / 64];
    const float inv = (a.scale ? 1.f / *a.scale : 1.f) * a.grad_mul;
    const double sum = add_parts<Y6_NORM_L2>(a.parts, a.nparts, sh);
    const double norm = sum * fabs((double)inv);
    if (a.out && blockIdx.x == 0 && threadIdx.x == 0) *a.out = (float)norm;
    if (a.found_inf) {
        // (a flag that another check set before counts too; whoever reads it after block 0's write returns either way)
        const bool skip = *a.found_inf != 0;
        if (!(sum < INFINITY)) {
            if (blockIdx.x == 0 && threadIdx.x == 0) *a.found_inf = 1;
            return;
        }
        if (skip) return;
    }
    const float mul = inv * clip_factor(norm, a.max_norm);
    auto one = [&](float& p, float g, float& m, int k) {
        if (k > 2) return;
        // (the roundings spelled out: those sgd_grouped_kernel is compiled to, so that a factor of 1 gives its bits)
        float d = g * mul;
        if (a.wd[k] != 0.f) d = decayed(d, a.wd[k], p);
        float b = d;
        if (a.mom != 0.f) {
            b = a.first ? d : fmaf(a.mom, m, d);
            m = b;
            if (a.nesterov) b = fmaf(a.mom, b, d);
        }
        p = fmaf(-a.lr[k], b, p);
    };
    const size_t n4 = a.n / 4;
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n4; i += (size_t)gridDim.x * kThreads) {
        const uchar4 k = reinterpret_cast<const uchar4*>(a.group)[i];
        float4 p = reinterpret_cast<const float4*>(a.p)[i];
        const float4 g = reinterpret_cast<const float4*>(a.g)[i];
        float4 m = a.mom != 0.f ? reinterpret_cast<const float4*>(a.m)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        one(p.x, g.x, m.x, k.x);
        one(p.y, g.y, m.y, k.y);
        one(p.z, g.z, m.z, k.z);
        one(p.w, g.w, m.w, k.w);
        reinterpret_cast<float4*>(a.p)[i] = p;
        if (a.mom != 0.f) reinterpret_cast<float4*>(a.m)[i] = m;
    }
    if (blockIdx.x == 0 && threadIdx.x < (a.n & 3)) {
        const size_t i = n4 * 4 + threadIdx.x;
        float m = a.mom != 0.f ? a.m[i] : 0.f;
        one(a.p[i], a.g[i], m, a.group[i]);
        if (a.mom != 0.f) a.m[i] = m;
    }
}

int elem_bytes(int type) { return type == Y6_F32 ? 4 : 2; }

int check_list(const y6_grad_list* l, const char* what) {
    Y6_REQUIRE(l, "%s: null argument", what);
    Y6_REQUIRE(l->count >= 0 && (l->count == 0 || (l->grads_host && l->numels_host && l->dtypes_host)), "%s: null argument", what);
    Y6_REQUIRE(l->norm_type == Y6_NORM_L2 || l->norm_type == Y6_NORM_L1 || l->norm_type == Y6_NORM_INF, "%s: unknown norm %d", what, l->norm_type);
    for (int i = 0; i < l->count; ++i) {
        const int t = l->dtypes_host[i];
        Y6_REQUIRE(t == Y6_F32 || t == Y6_F16 || t == Y6_BF16, "%s: tensor %d has dtype %d (fp16, bf16 or fp32)", what, i, t);
        Y6_REQUIRE((uintptr_t)l->grads_host[i] >> 62 == 0 && l->numels_host[i] >= 0 && l->numels_host[i] < (1ll << 40), "%s: tensor %d has %lld elements", what, i, (long long)l->numels_host[i]);
        Y6_REQUIRE(l->numels_host[i] == 0 || l->grads_host[i], "%s: tensor %d is null", what, i);
        Y6_REQUIRE((uintptr_t)l->grads_host[i] % elem_bytes(t) == 0, "%s: tensor %d is not aligned to its elements", what, i);
    }
    return Y6_OK;
}

// The next entries of the list from element `from` of tensor `i` on (empty tensors left out); moves i and from.  Returns the chunks.
unsigned fill_table(const y6_grad_list* l, int& i, long long& from, Table& tb) {
    unsigned long long chunks = 0;
    for (tb.count = 0; i < l->count && tb.count < kTable;) {
        const long long left = l->numels_host[i] - from;
        if (left <= 0) {
            ++i, from = 0;
            continue;
        }
        const int type = l->dtypes_host[i];
        const unsigned n = (unsigned)(left < kEntry ? left : kEntry);
        const unsigned long long at = ((unsigned long long)(uintptr_t)l->grads_host[i] + (unsigned long long)from * elem_bytes(type)) | (unsigned long long)type << 62;
        tb.at[tb.count] = at;          // (the types are 0, 1 and 3)
        tb.n[tb.count] = n;
        ++tb.count;
        chunks += chunks_of(at, n);
        from += n;
    }
    return (unsigned)chunks;           // 330 entries of at most 2^18 + 1
}
int table_blocks(unsigned chunks) { return chunks < (unsigned)kBlocks ? (int)chunks : kBlocks; }
// tables of a list of so many tensors and elements, at most
size_t tables_for(size_t tensors, unsigned long long elements) { return (tensors + elements / kEntry) / kTable + 1; }

int launch_part(int norm, const Table& tb, int blocks, double* parts, hipStream_t s) {
    const dim3 g(blocks), b(kThreads);
    if (norm == Y6_NORM_L2) hipLaunchKernelGGL(grad_part_kernel<Y6_NORM_L2>, g, b, 0, s, tb, parts);
    else if (norm == Y6_NORM_L1) hipLaunchKernelGGL(grad_part_kernel<Y6_NORM_L1>, g, b, 0, s, tb, parts);
    else hipLaunchKernelGGL(grad_part_kernel<Y6_NORM_INF>, g, b, 0, s, tb, parts);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}

// partial sums of the whole list -> parts[0 .. *n)
int list_parts(const y6_grad_list* l, double* parts, size_t cap, int* n, hipStream_t s) {
    Table tb;
    *n = 0;
    int i = 0;
    long long from = 0;
    while (const unsigned chunks = fill_table(l, i, from, tb)) {
        const int blocks = table_blocks(chunks);
        Y6_REQUIRE((size_t)*n + blocks + 1 <= cap, "grad_norm: workspace too small");
        const int rc = launch_part(l->norm_type, tb, blocks, parts + *n, s);
        if (rc != Y6_OK) return rc;
        *n += blocks;
    }
    return Y6_OK;
}

}  // namespace

// ====================================================================== C ABI
extern "C" size_t y6_grad_norm_workspace_bytes(int count, int64_t elements) {
    return (tables_for(count > 0 ? (size_t)count : 0, elements > 0 ? (unsigned long long)elements : 0) * kBlocks + 1) * sizeof(double);
}

extern "C" int y6_grad_norm(const y6_grad_list* l, void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    Y6_CLEAR_STALE_ERROR();
    int rc = check_list(l, "grad_norm");
    if (rc != Y6_OK) return rc;
    Y6_REQUIRE(norm && workspace, "grad_norm: null argument");
    hipStream_t s = (hipStream_t)stream;
    int n = 0;
    rc = list_parts(l, (double*)workspace, workspace_bytes / sizeof(double), &n, s);
    if (rc != Y6_OK) return rc;
    hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(kThreads), 0, s, l->norm_type, (double*)workspace, n, norm);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}

extern "C" int y6_grad_clip(const y6_grad_list* l, double max_norm, void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    Y6_CLEAR_STALE_ERROR();
    int rc = check_list(l, "grad_clip");
    if (rc != Y6_OK) return rc;
    Y6_REQUIRE(norm && workspace, "grad_clip: null argument");
    Y6_REQUIRE(max_norm >= 0, "grad_clip: max_norm %g is negative or not a number", max_norm);
    try {                              // two tensors over the same memory would be scaled by two blocks at once
        std::vector<std::pair<uintptr_t, uintptr_t>> span;
        span.reserve((size_t)l->count);
        for (int i = 0; i < l->count; ++i)
            if (l->numels_host[i])
                span.emplace_back((uintptr_t)l->grads_host[i], (uintptr_t)l->grads_host[i] + (size_t)l->numels_host[i] * elem_bytes(l->dtypes_host[i]));
        std::sort(span.begin(), span.end());
        for (size_t i = 1; i < span.size(); ++i)
            Y6_REQUIRE(span[i].first >= span[i - 1].second, "grad_clip: two gradients share memory");
    } catch (const std::bad_alloc&) {
        y6_set_error("grad_clip: out of host memory");
        return Y6_ENOMEM;
    }
    hipStream_t s = (hipStream_t)stream;
    double* parts = (double*)workspace;
    int n = 0;
    rc = list_parts(l, parts, workspace_bytes / sizeof(double), &n, s);
    if (rc != Y6_OK) return rc;
    if (n == 0) {
        hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(kThreads), 0, s, l->norm_type, parts, 0, norm);
        Y6_LAUNCH_CHECK();
        return Y6_OK;
    }
    if (n > kJoin) {
        hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(kThreads), 0, s, l->norm_type, parts, n, (float*)nullptr);
        Y6_LAUNCH_CHECK();
        parts += n;
        n = 1;
    }
    Table tb;
    int i = 0;
    long long from = 0;
    while (const unsigned chunks = fill_table(l, i, from, tb)) {
        hipLaunchKernelGGL(grad_scale_kernel, dim3(table_blocks(chunks)), dim3(kThreads), 0, s, tb, l->norm_type, parts, n, max_norm, norm);
        Y6_LAUNCH_CHECK();
    }
    return Y6_OK;
}

extern "C" int y6_sgd_step_clipped(float* param, const float* grad, float* momentum_buf, const uint8_t* group, size_t n, const float* lr3,
                                   const float* wd3, float momentum, int nesterov, int first_step, float grad_mul, const float* scale,
                                   int32_t* found_inf, double max_norm, void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    Y6_CLEAR_STALE_ERROR();
    Y6_REQUIRE(param && grad && group && lr3 && wd3 && workspace && (momentum == 0.f || momentum_buf), "sgd_step_clipped: null argument");
    Y6_REQUIRE(max_norm >= 0, "sgd_step_clipped: max_norm %g is negative or not a number", max_norm);
    Y6_REQUIRE(((uintptr_t)param | (uintptr_t)grad | (uintptr_t)momentum_buf) % 16 == 0 && (uintptr_t)group % 4 == 0,
               "sgd_step_clipped: the arena is not aligned to 16 bytes");
    Y6_REQUIRE(n < ((size_t)1 << 40), "sgd_step_clipped: %zu elements", n);
    hipStream_t s = (hipStream_t)stream;
    if (n == 0) {                      // the norm of nothing is 0, as y6_grad_norm's
        if (!norm) return Y6_OK;
        hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(kThreads), 0, s, Y6_NORM_L2, (double*)workspace, 0, norm);
        Y6_LAUNCH_CHECK();
        return Y6_OK;
    }
    void* const grads[1] = {(void*)grad};
    const int64_t numels[1] = {(int64_t)n};
    const int32_t types[1] = {Y6_F32};
    y6_grad_list l = {grads, numels, types, 1, Y6_NORM_L2};
    ClipSgd a;
    int rc = list_parts(&l, (double*)workspace, workspace_bytes / sizeof(double), &a.nparts, s);
    if (rc != Y6_OK) return rc;
    a.p = param, a.g = grad, a.m = momentum_buf, a.group = group, a.n = n;
    for (int i = 0; i < 3; ++i) {
        a.lr[i] = lr3[i];
        a.wd[i] = wd3[i];
    }
    a.lr[3] = a.wd[3] = 0.f;
    a.mom = momentum, a.grad_mul = grad_mul, a.nesterov = nesterov, a.first = first_step;
    a.scale = scale, a.found_inf = found_inf, a.parts = (const double*)workspace, a.max_norm = max_norm, a.out = norm;
    const size_t need = (n / 4 + kThreads - 1) / kThreads;
    const int blocks = need < 1 ? 1 : need > 2048 ? 2048 : (int)need;
    hipLaunchKernelGGL(sgd_clipped_kernel, dim3(blocks), dim3(kThreads), 0, s, a);
    Y6_LAUNCH_CHECK();
    return Y6_OK;
}
