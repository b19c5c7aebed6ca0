// Operators of a paged key/value cache for sm_100a: tables from request lengths, rotary positions, writing
// new tokens into the pages, and the attention of one new token per request over them.  The interface, with
// the formulas, is include/fa_paged_sm100.h.
//
// All of them are bound by memory or, for the small calls of a decoding step, by the latency of a launch:
// none comes near the tensor pipe's rate (the attention does 4 flops per byte and query head of a group).
//
// Every kernel is launched chained to the kernel before it in the stream (programmatic stream serialization)
// and executes griddepcontrol.wait before it first touches memory, so "the kernel before has finished" covers
// all kernels before it.  Behind that wait nothing is read through the read-only path: no `__ldg`, no
// `__restrict__` arguments (the compiler may move such loads ahead of the wait).
#include <atomic>
#include <climits>
#include <cmath>
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fa_paged_sm100.h"

namespace fa_paged {

// ------------------------------------------------------------------------------------------------
// PTX wrappers
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// Lets the next kernel of the stream become resident / waits until the kernel before has finished.  The rotary
// and attention kernels do not announce the next one early: resident CTAs of the next take their places SM by SM as theirs
// leave, which spread the next call unevenly (48 requests, 16 heads of 64, an earlier form of the kernel: 53 us a call
// with it, 40 without).
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait_prior_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16 bytes; volatile, so that it stays where it is written: ahead of the work it is meant to overlap.
__device__ __forceinline__ uint4 ld_v4(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// 16 bytes from global to shared memory; the rest of them is zero where `bytes` is less (0: nothing is read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// The address of another cluster CTA's copy of a shared-memory location, and loads from there.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Transposes the 8 x 8 matrix of 16-bit elements that the warp's registers hold.
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The page size, as a divisor of numbers below 2^31:  x / size = x * mul >> shift,  shift = 31 + ceil(log2(size)),
// mul = ceil(2^shift / size).  (mul is off by less than 1, so the product is by less than x < 2^31, a quotient by less
// than 1 / size.)
struct PageSize {
    unsigned size, mul, shift;
};
static PageSize page_size_of(int size) {
    unsigned s = 31;
    while ((1ULL << (s - 31)) < static_cast<unsigned long long>(size)) ++s;
    return PageSize{static_cast<unsigned>(size), static_cast<unsigned>(((1ULL << s) + size - 1) / size), s};
}
__device__ __forceinline__ unsigned page_of(unsigned token, const PageSize& ps) {
    return static_cast<unsigned>((static_cast<unsigned long long>(token) * ps.mul) >> ps.shift);
}
// Pages of so many tokens.
__device__ __forceinline__ unsigned pages_of(unsigned tokens, const PageSize& ps) {
    const unsigned whole = page_of(tokens, ps);
    return whole + (whole * ps.size != tokens);
}

__device__ __forceinline__ long long load_int(const void* p, int is64, long long i) {
    return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// Inclusive prefix sum over the CTA (any multiple of 32 threads up to 1024); `scratch` holds 32 values and is
// free again once the CTA has passed its next barrier.
__device__ __forceinline__ long long block_scan(long long v, long long* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    long long before = lane < warp && lane < warps ? scratch[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    return v + before;
}

// The same of two values at once.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long (*scratch)[32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
            a += x;
            b += y;
        }
    }
    if (lane == 31) {
        scratch[0][warp] = a;
        scratch[1][warp] = b;
    }
    __syncthreads();
    long long x = lane < warp && lane < warps ? scratch[0][lane] : 0, y = lane < warp && lane < warps ? scratch[1][lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    a += x;
    b += y;
}

// ------------------------------------------------------------------------------------------------
// Tables from request lengths
// ------------------------------------------------------------------------------------------------
// A block-wide prefix sum over the requests (tokens, and pages needed), kept in shared memory; then every thread
// takes four consecutive tokens at a time, finds the request of the first by bisection and walks on from there.
// What is read and written is a few bytes per token: the time is that of a launch and of a chain of dependent
// reads (lengths, free list, table).  Small calls are one CTA; from kTableTokens on it is a cluster of eight, each
// of which works out the (cheap) sums for itself and takes an eighth of the tokens and pages.  A cluster and not
// a grid, because lens and free_head may be updated in place: they are written behind a cluster barrier, when
// every CTA has read them.  Replayed from a graph: 256 decoding requests 3.5 us (8.0 with a warp per request for its
// pages, four tokens a thread and divisions); 48 prompts, 79,000 tokens and 5,000 pages: 10.5 us; called from Python both
// take the host's 10 us.  With one CTA the prompts took 70 us.
constexpr int kTableThreads = 512, kTableClusterThreads = 1024;      // of the one CTA, of each of the eight
constexpr int kTableCluster = 8;
constexpr int kFewPages = 4;           // that the thread of a request hands out by itself
constexpr long long kTableTokens = 4096;       // both the host's 10 us up to 8,000 tokens; 16,000: 12.2 us against 16.5

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

struct ExtendParams {
    int* table;
    long long table_stride;
    const int* lens;
    const int* new_lens;
    const int* free_pages;
    const int* free_head;
    int* lens_out;
    int* head_out;
    long long* slots;
    int* positions;
    int* cu;
    PageSize page;
    int batch, width, num_free;
    long long num_tokens;
};


__global__ void __launch_bounds__(kTableClusterThreads) paged_extend_kernel(const ExtendParams p) {
    extern __shared__ int s_table[];
    int* s_cu = s_table;                    // batch + 1: first token of each request
    int* s_len = s_cu + p.batch + 1;        // batch: length before
    int* s_src = s_len + p.batch;           // batch: index of its first new page in the free list, -1: refused
    __shared__ long long s_scan[2][32];
    __shared__ long long s_before[2];
    __shared__ int s_head;
    pdl_launch_dependents();
    const int tid = threadIdx.x, threads = blockDim.x;
    const unsigned rank = cluster_rank(), ranks = cluster_size();
    pdl_wait_prior_grid();
    const int head = min(max(p.free_head[0], 0), p.num_free);
    const long long avail = p.num_free - head;
    if (tid == 0) {
        s_cu[0] = 0;
        s_head = head;
        s_before[0] = s_before[1] = 0;
    }
    __syncthreads();
    bool many = false;                      // some request gets more than a few pages
    for (int base = 0; base < p.batch; base += threads) {
        const int b = base + tid;
        const bool in = b < p.batch;
        const unsigned len = in ? max(p.lens[b], 0) : 0, add = in ? max(p.new_lens[b], 0) : 0;
        const unsigned have = pages_of(len, p.page);
        unsigned want = have;
        const bool counted = len + add <= static_cast<unsigned>(INT_MAX);
        if (counted) want = pages_of(len + add, p.page);
        const bool fits = counted && want <= static_cast<unsigned>(p.width);
        const unsigned need = fits ? want - have : 0;
        long long tokens = add, pages = need;
        block_scan2(tokens, pages, s_scan);
        tokens += s_before[0];
        pages += s_before[1];
        const bool granted = fits && (need == 0 || pages <= avail);
        if (in) {
            s_cu[b + 1] = static_cast<int>(min(tokens, static_cast<long long>(INT_MAX)));
            s_len[b] = static_cast<int>(len);
            const int src = head + static_cast<int>(pages) - static_cast<int>(need);
            s_src[b] = !granted ? -1 : need > 0 ? src : 0;
            // a few pages: here and now
            if (granted && need > 0 && need <= kFewPages && b % ranks == rank) {
                int* row = p.table + b * p.table_stride + have;
                for (unsigned i = 0; i < need; ++i) row[i] = p.free_pages[src + i];
            }
        }
        many |= in && granted && need > kFewPages;
        // pages are given to a first part of those that need some: the last prefix sum there is their number
        const int given = __reduce_max_sync(0xffffffffu, in && granted && need > 0 ? head + static_cast<int>(pages) : 0);
        if ((tid & 31) == 0 && given > 0) atomicMax(&s_head, given);
        __syncthreads();
        if (tid == threads - 1) {
            s_before[0] = tokens;
            s_before[1] = pages;
        }
        __syncthreads();
    }
    cluster_arrive();                       // lens and free_head have been read
    if (__syncthreads_or(many)) {
        // many pages: one warp per request
        const int warps = ranks * (threads / 32);
        for (int b = rank * (threads / 32) + (tid >> 5); b < p.batch; b += warps) {
            if (s_src[b] < 0) continue;
            const unsigned len = s_len[b], add = s_cu[b + 1] - s_cu[b];
            const int have = pages_of(len, p.page), want = pages_of(len + add, p.page);
            if (want - have <= kFewPages) continue;
            int* row = p.table + b * p.table_stride;
            for (int i = have + (tid & 31); i < want; i += 32) row[i] = p.free_pages[s_src[b] + i - have];
        }
    }
    // slots and positions; a page that is new is read from the free list, not from the row just written
    const long long total = s_cu[p.batch];
    const bool vec = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) & 15u) == 0;
    const int each = p.num_tokens <= static_cast<long long>(ranks) * threads ? 1 : 4;     // tokens that a thread takes at a time
    for (long long t0 = each * (static_cast<long long>(rank) * threads + tid); t0 < p.num_tokens;
         t0 += static_cast<long long>(each) * ranks * threads) {
        const int* from[4];                              // where the page of each token is named
        unsigned row[4];
        int pos[4];
        int b = 0, hi = p.batch;                         // s_cu[b] <= t0 < s_cu[hi]
        if (t0 < total)
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (s_cu[mid] <= t0) b = mid;
                else hi = mid;
            }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const long long t = t0 + e;
            from[e] = nullptr;
            row[e] = 0;
            pos[e] = 0;
            if (e < each && t < total) {
                while (s_cu[b + 1] <= t) ++b;
                pos[e] = static_cast<int>(s_len[b] + (t - s_cu[b]));
                if (s_src[b] >= 0) {
                    const unsigned have = pages_of(s_len[b], p.page), at = page_of(pos[e], p.page);
                    from[e] = at < have ? p.table + b * p.table_stride + at : p.free_pages + s_src[b] + (at - have);
                    row[e] = static_cast<unsigned>(pos[e]) - at * p.page.size;
                }
            }
        }
        int page[4];
        long long slot[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) page[e] = from[e] != nullptr ? *from[e] : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) slot[e] = from[e] != nullptr ? static_cast<long long>(page[e]) * p.page.size + row[e] : -1;
        if (vec && each == 4 && t0 + 4 <= p.num_tokens) {
            *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
            *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
            *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < each && t0 + e < p.num_tokens) {
                    p.slots[t0 + e] = slot[e];
                    p.positions[t0 + e] = pos[e];
                }
        }
    }
    cluster_wait();
    for (int b = rank * threads + tid; b < p.batch; b += ranks * threads) {
        p.cu[b + 1] = s_cu[b + 1];
        p.lens_out[b] = s_len[b] + (s_src[b] >= 0 ? s_cu[b + 1] - s_cu[b] : 0);
    }
    if (rank == 0 && tid == 0) {
        p.cu[0] = 0;
        p.head_out[0] = s_head;
    }
}

struct ShrinkParams {
    const int* table;
    long long table_stride;
    int* lens;
    const int* keep;
    int* free_pages;
    int* free_head;
    PageSize page;
    int batch, width, num_free;
};

__global__ void __launch_bounds__(kTableThreads) paged_shrink_kernel(const ShrinkParams p) {
    extern __shared__ int s_table[];
    int* s_from = s_table;                  // first page released
    int* s_count = s_from + p.batch;        // pages released (0 for a refused request)
    int* s_to = s_count + p.batch;          // where they go in the free list
    __shared__ long long s_scan[32];
    __shared__ long long s_before;
    __shared__ int s_head;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int tid = threadIdx.x;
    const int head = min(max(p.free_head[0], 0), p.num_free);
    if (tid == 0) {
        s_head = head;
        s_before = 0;
    }
    __syncthreads();
    for (int base = 0; base < p.batch; base += kTableThreads) {
        const int b = base + tid;
        const bool in = b < p.batch;
        const unsigned len = in ? max(p.lens[b], 0) : 0;
        const unsigned keep = in ? min(static_cast<unsigned>(max(p.keep[b], 0)), len) : 0;
        const unsigned most = p.width;
        const unsigned from = min(pages_of(keep, p.page), most), upto = min(pages_of(len, p.page), most);
        const unsigned count = upto - from;
        const long long sum = s_before + block_scan(count, s_scan);
        const bool granted = count == 0 || sum <= head;
        if (in) {
            s_from[b] = static_cast<int>(from);
            s_count[b] = granted ? static_cast<int>(count) : 0;
            s_to[b] = granted ? head - static_cast<int>(sum) : 0;
            if (granted) p.lens[b] = static_cast<int>(keep);
        }
        const int low = __reduce_min_sync(0xffffffffu, in && granted && count > 0 ? head - static_cast<int>(sum) : INT_MAX);
        if ((tid & 31) == 0) atomicMin(&s_head, low);
        __syncthreads();
        if (tid == kTableThreads - 1) s_before = sum;
        __syncthreads();
    }
    for (int b = tid >> 5; b < p.batch; b += kTableThreads / 32) {
        const int* row = p.table + b * p.table_stride + s_from[b];
        for (int i = tid & 31; i < s_count[b]; i += 32) p.free_pages[s_to[b] + i] = row[i];
    }
    if (tid == 0) p.free_head[0] = s_head;
}

// ------------------------------------------------------------------------------------------------
// Rotary positions, and writing new tokens into the pages
// ------------------------------------------------------------------------------------------------
// A CTA takes 1, 2, 4 or 8 tokens: the angles of their positions are worked out once, in shared memory, and serve
// all heads of queries and keys.  A thread takes 16 elements of a head, always the same ones of the same token, so
// the 8 pairs' cos and sin stay in registers; the first kRotaryBatch heads' loads are in flight while the angles
// are worked out.  Tokens per CTA: as many as keep a thread at kRotaryBatch heads at most, so that all of a CTA's
// loads are in flight together - unless that leaves SMs without a CTA.  Bound by memory: 4 x 2048 tokens with 16 + 4
// heads of 128 take 15.6 to 16.9 us, 5.0 to 5.4 TB/s of 6.5 both ways; 8100 tokens with 32 + 8 + 8 heads into the pages
// 37.9 us, 5.3 TB/s; 64 tokens 7.1 us a call, the host's time.  Measured and left: four heads a thread (fewer CTAs,
// 17.2 us), CTAs that stay and load pieces ahead by cp.async (19.9), loads through shared memory (16.4).
constexpr int kRotaryThreads = 128;
constexpr int kRotaryBatch = 3;
constexpr int kRotaryTokens = 8;
constexpr int kRotaryWaves = 4;       // CTAs per SM that there have to be
// (One token a CTA: 21.7 us instead of 15.7 for 20 heads of 128, 19.4 instead of 11.9 for 8100 tokens with 12.)

struct Rows {                     // heads of one token: where they are read and where they go
    const uint16_t* in;
    uint16_t* out;
    long long in_outer, in_head, in_token;     // element strides
    long long out_outer, out_head, out_token;
    int heads;
};

struct RotaryParams {
    Rows rows[3];                 // queries and keys, which turn, and values, which do not
    const double* freqs;
    const void* positions;
    long long position_outer;
    int positions_64, rot;        // rot = 0: nothing turns
    float mscale, sign;
    int tokens, per_cta;          // tokens of one outer index; tokens of a CTA
    // grid.x: tokens, grid.y: outer.  In the append form rows 1 and 2 go to the cache: out_token is
    // the stride of a token in its page and out_outer that of a page.
    const void* slots;            // NULL: not the append form
    int slots_64, page_size;
    long long num_slots;
};

// How a head's elements are paired, and so which 16 a thread takes.
enum Pairing {
    kHalves,          // (i, i + rot / 2), rot a multiple of 16: 8 elements and the 8 they are paired with
    kNeighbours,      // (2i, 2i + 1): 16 consecutive ones
    kRaggedHalves     // (i, i + rot / 2) with any rot: 16 consecutive ones, turned in shared memory, where pair c is the
                      // head's thread c % kParts's.  (4 x 2048 tokens, 16 + 4 heads of 128, rot 20: 17.7 us; 38.7 with
                      // each element's partner read from global memory, 36.7 from shared memory: 8 threads at 1 bank.)
};

template <int D, bool BF16, int PAIRING>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
    __shared__ __align__(16) float2 s_turn[kRotaryTokens * D / 2];     // (cos, sin) * mscale of each pair
    const int tid = threadIdx.x;
    constexpr int kParts = D / 16;
    const int part = tid % kParts, mine = tid / kParts % p.per_cta, start = tid / kParts / p.per_cta;
    const int step = kRotaryThreads / kParts / p.per_cta;
    const long long outer = blockIdx.y, token0 = static_cast<long long>(blockIdx.x) * p.per_cta, token = token0 + mine;
    const int pairs = p.rot / 2;
    const float2* turn = s_turn + mine * (D / 2);
    __shared__ __align__(16) uint16_t s_head[PAIRING == kRaggedHalves ? kRotaryThreads / kParts : 1][D + 8];  // a head per team
    const unsigned team = ((1u << kParts) - 1) << (tid % 32 / kParts * kParts);      // the lanes that share a head
    const int col_a = PAIRING == kHalves ? (part * 16 < p.rot ? part * 8 : part * 16) : part * 16;
    const int col_b = PAIRING == kHalves && part * 16 < p.rot ? col_a + pairs : col_a + 8;
    const bool turned = part * 16 < p.rot;     // some of my elements turn
    const int h0 = p.rows[0].heads, h1 = h0 + p.rows[1].heads, total = token < p.tokens ? h1 + p.rows[2].heads : 0;
    auto source = [&](int head) {
        const int which = head < h0 ? 0 : head < h1 ? 1 : 2;
        const Rows& r = p.rows[which];
        return r.in + outer * r.in_outer + token * r.in_token + (head - (which == 0 ? 0 : which == 1 ? h0 : h1)) * r.in_head;
    };
    pdl_wait_prior_grid();

    uint4 a[kRotaryBatch], b[kRotaryBatch];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < kRotaryBatch; ++i) {
            const int head = first + i * step;
            if (head < total) {
                const uint16_t* in = source(head);
                a[i] = ld_v4(in + col_a);
                b[i] = ld_v4(in + col_b);
            }
        }
    };
    load(start);
    long long page = 0, row = 0;
    bool kept = true;
    if (p.slots != nullptr && token < p.tokens) {
        const long long slot = load_int(p.slots, p.slots_64, token);
        kept = slot >= 0 && slot < p.num_slots;
        if (slot <= UINT_MAX) {                // the usual case: no division in 64 bits
            page = static_cast<unsigned>(slot) / static_cast<unsigned>(p.page_size);
            row = static_cast<unsigned>(slot) - static_cast<unsigned>(page) * p.page_size;
        } else {
            page = slot / p.page_size;
            row = slot - page * p.page_size;
        }
    }
    float2 t[8];
    if (p.rot > 0) {
        constexpr int kLanes = kRotaryThreads / (D / 2);          // tokens worked on at a time, one pair a thread
        const int i = tid % (D / 2);
        for (int at = tid / (D / 2); at < p.per_cta; at += kLanes) {
            if (i >= pairs || token0 + at >= p.tokens) continue;
            const double pos = static_cast<double>(load_int(p.positions, p.positions_64, outer * p.position_outer + token0 + at));
            const double turns = pos * p.freqs[i] * 0.15915494309189533577;      // 1 / (2 pi)
            float s, c;
            sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
            s_turn[at * (D / 2) + i] = make_float2(c * p.mscale, s * p.mscale * p.sign);
        }
        __syncthreads();
        if (PAIRING != kRaggedHalves && turned)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(&turn[part * 8 + 2 * i]);
                t[2 * i] = make_float2(x.x, x.y);
                t[2 * i + 1] = make_float2(x.z, x.w);
            }
    }
    for (int first = start; first < total; first += kRotaryBatch * step) {
        if (first != start) load(first);
#pragma unroll
        for (int i = 0; i < kRotaryBatch; ++i) {
            const int head = first + i * step;
            if (head >= total) break;
            uint32_t* wa = reinterpret_cast<uint32_t*>(&a[i]);
            uint32_t* wb = reinterpret_cast<uint32_t*>(&b[i]);
            if constexpr (PAIRING == kRaggedHalves) {
                if (p.rot > 0 && head < h1) {
                    uint16_t* all = s_head[tid / kParts];
                    uint4* mine_of_all = reinterpret_cast<uint4*>(all + part * 16);
                    mine_of_all[0] = a[i];
                    mine_of_all[1] = b[i];
                    __syncwarp(team);
                    for (int c = part; c < pairs; c += kParts) {
                        const float2 x = unpack2<BF16>(all[c] | static_cast<uint32_t>(all[c + pairs]) << 16), cs = turn[c];
                        const uint32_t y = pack2<BF16>(x.x * cs.x - x.y * cs.y, x.y * cs.x + x.x * cs.y);
                        all[c] = static_cast<uint16_t>(y);
                        all[c + pairs] = static_cast<uint16_t>(y >> 16);
                    }
                    __syncwarp(team);
                    a[i] = mine_of_all[0];
                    b[i] = mine_of_all[1];
                }
            } else if (turned && head < h1) {
                if constexpr (PAIRING == kHalves) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 x = unpack2<BF16>(wa[e]), y = unpack2<BF16>(wb[e]);
                        const float2 t0 = t[2 * e], t1 = t[2 * e + 1];
                        wa[e] = pack2<BF16>(x.x * t0.x - y.x * t0.y, x.y * t1.x - y.y * t1.y);
                        wb[e] = pack2<BF16>(y.x * t0.x + x.x * t0.y, y.y * t1.x + x.y * t1.y);
                    }
                } else if constexpr (PAIRING == kNeighbours) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t& w = e < 4 ? wa[e] : wb[e - 4];
                        const float2 x = unpack2<BF16>(w);
                        if (part * 8 + e < pairs) w = pack2<BF16>(x.x * t[e].x - x.y * t[e].y, x.y * t[e].x + x.x * t[e].y);
                    }
                }
            }
            const int which = head < h0 ? 0 : head < h1 ? 1 : 2;
            const Rows& r = p.rows[which];
            uint16_t* out = r.out + (head - (which == 0 ? 0 : which == 1 ? h0 : h1)) * r.out_head;
            if (p.slots != nullptr && which > 0) {
                if (!kept) continue;
                out += page * r.out_outer + row * r.out_token;
            } else {
                out += outer * r.out_outer + token * r.out_token;
            }
            *reinterpret_cast<uint4*>(out + col_a) = a[i];
            *reinterpret_cast<uint4*>(out + col_b) = b[i];
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Attention of one new token per request over the pages
// ------------------------------------------------------------------------------------------------
// Mathematics: one pass over the keys with a running reference m, a sum l and an accumulator o per query head, in
// fp32 and in powers of two: x = log2(e) * score, p = 2^(x - m), l = sum p, o = sum p v.  m goes by a maximum that
// moves only when a score exceeds it by more than 8 (o / l does not depend on m).  Parts of a
// key range are joined by  o = sum_i 2^(m_i - m) o_i  and likewise l.
//
// Bound: memory.  A key of a KV head costs 4 * head_dim bytes and 4 * head_dim flops per query head of the
// group, so even 32 heads a group stay far from the tensor pipe's balance (250 flops a byte).  What matters is
// to keep enough loads in flight on every SM, whatever the lengths are, and, for short histories, that little has to
// happen one after the other.
//
// Work: the requests' key ranges, per KV head, are cut in tiles of kTile keys and laid one behind the other -
// request, then KV head, then row block, then tile - and every CTA takes an equal, consecutive share of that
// sequence.  The end of a unit costs what one to four tiles do, so in a long sequence it counts as so many places: 16
// requests with 32 heads on one key head 37.1 -> 34.0 us, with 16 heads 27.1 -> 24.8; 300 of up to 300 keys 54.3 -> 50.6;
// 8 of up to 7001 with a bias 21.9 -> 21.2 (half or twice as many places are worse by 0.1 to 0.9).  The lengths are on
// the device only, so each CTA works out the sums itself.  A share may begin or end inside a unit (one request and KV
// head): then it leaves a partial result (o, m, l) in the workspace and paged_join_kernel joins the parts.  At most one
// such part at either end of a share.
//
// Inside a CTA four warps take the keys of a tile, kKeys each, and stream on their own: each has its own ring
// of stages in shared memory, fills it by cp.async across tile, unit and request borders and never waits
// for another warp before a unit ends; then the four results are joined through shared memory.
//
// Products: with few query rows the keys are the rows of the mma: S^T (16 keys x 8 heads) = K Q^T and
// O^T (16 of d x 8 heads) += V^T P^T.  Eight heads to a tile waste half of what sixteen would, and the
// accumulators are half as many.  K and V come through ldmatrix (V transposed); P^T moves from the accumulator
// layout to the operand's by movmatrix.  mma.sync is enough up to 8 heads a tile: the tensor pipe is busy for 15 % of
// the time, and tcgen05, with 128 keys as its rows, would want P^T in shared memory.  With 16 and 32 heads it is not:
// registers leave room for eight warps an SM, too few to hide the products' latencies.
//
// Precision: a weight p is the sum of two 16-bit numbers (hi + lo), two products instead of one; a single
// 16-bit weight would add as much error as the rounding of the output.  Sums take the fp32 weight.
//
// Measured (calls back to back; memory's rate is 6.54 TB/s): one request of 131072 keys, 32 + 8 heads of 128: 89 us,
// 6.03 TB/s; 32 requests of up to 4096: 62.0, 5.7 TB/s; 48 requests of a window of 1024, 16 heads of 64, capped: 38.2,
// 5.2 TB/s; 8 requests of up to 7001 with a bias: 21.2, 3.9 TB/s; one of 333: 7.1, the host's time.  Of what is above
// the bytes' time, 2 us are the launch and the way to the first load, 2 the first loads' latency, 1.3 the end of a
// unit, 3 to 4 the joining kernel.  32 heads on one key head: 34 against 14 for the bytes - eight warps an SM with 96
// products a step each do not hide their latencies.
// Measured and left: warps that share a tile and exchange P, so that accumulators are small (two barriers a tile: 109
// us for the 131072 keys); bulk copies of a row per lane (issued one by one, 137); joining by the last CTA to
// finish, by tickets (25.9 us for the bias, 89 for the 32 heads); two to four times as many shares (64, 67, 71 us for
// the 32 requests).
constexpr int kWarps = 4;
constexpr int kAttnThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kLongShare = 4;          // tiles of a share from which on the end of a unit counts
constexpr float kGrowth = 8.f;         // how far (in powers of two) a score may exceed the maximum that m goes by
// m lies so far below that maximum.  Weights in fp16 vanish below 2^-25: with p up to 2^14 instead of 2^8, a hundred
// thousand keys of such weights together stay below the rounding of the output.  (bf16 has fp32's exponents.)
template <bool BF16>
constexpr float kHeadroom = BF16 ? 0.f : 6.f;

template <int D, int NT>
struct AttnCfg {
    static constexpr int kKeys = 2048 / D;                 // keys of one warp's step: K and V are 4 KB each
    static constexpr int kTile = kKeys * kWarps;
    static constexpr int kStageBytes = kKeys * D * 2 * 2;
    // Stages and CTAs per SM: what shared memory and registers allow.  24 to 32 KB in flight per warp and three stages
    // read 6.0 of 6.5 TB/s in the longest call; at 64, more warps hide the softmax, twice the work per byte (35 us against
    // 77 with two CTAs).
    static constexpr int kStages = NT > 2 || D == 64 ? 2 : 3;
    static constexpr int kCtas = D == 64 && NT == 1 ? 3 : 2;
    static constexpr int kUnitEnd = (NT > 2 ? 2 : 1) * (D == 64 ? 1 : 2);      // tiles that the end of a unit counts as
    static constexpr int kRingBytes = kStageBytes * kStages * kWarps;
    static constexpr int kJoinBytes = kWarps * 8 * D * 4;
    // The query rows of a unit: in registers up to 16 heads; 32 would not fit beside the accumulators and stay in
    // shared memory, in the buffer that joins the warps' results when the unit ends.
    static constexpr bool kQueryInSmem = NT > 2;
    static constexpr int kSmem = kRingBytes + kJoinBytes;
    static_assert(!kQueryInSmem || NT * 8 * D * 2 <= kJoinBytes, "the query rows fit the join buffer");
};
constexpr int attn_tile(int d) { return 2048 / d * kWarps; }

struct AttnParams {
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    const uint16_t* k;
    const uint16_t* v;
    const int* table;
    const int* lens;
    const float* slopes;
    long long q_batch, q_head, table_stride;
    long long k_page, k_head, k_row, v_page, v_head, v_row;
    int batch, heads, heads_k, group, row_blocks, width, num_pages, window;
    int cluster;                  // n > 0: unit u is done by the n CTAs from n u on, a cluster; 0: equal shares
    PageSize page;
    // x, in powers of two, is s * scale2, or capped
    float scale2, cap2, inner;
    int cap_series;
    // workspace
    struct CutInfo* cuts;         // one per unit, or one per CTA where there are more units than CTAs
    int cuts_by_unit;
    float* parts;                 // two per CTA: rows * D of o, then rows (m, l)
    long long part_floats;
};

// A unit that is cut in parts: those of `count` shares from `first` on; count = 0: nothing to join.
struct CutInfo {
    int unit, first, count, pad;
};

struct Range {
    int lo, hi;                   // visible keys [lo, hi)
    int tile_lo, tile_hi;
};
template <int TILE>
__device__ __forceinline__ Range key_range(const AttnParams& p, int len) {
    const int most = p.width * static_cast<int>(p.page.size);
    Range r;
    r.hi = min(max(len, 0), most);
    r.lo = p.window > 0 ? max(0, r.hi - p.window) : 0;
    r.tile_lo = r.lo / TILE;
    r.tile_hi = max(r.tile_lo + 1, (r.hi + TILE - 1) / TILE);     // a request without a key still takes one
    return r;
}

// Share c of `shares` equal ones of `total` tiles begins at floor(c * total / shares).
__device__ __forceinline__ long long share_begin(long long c, long long total, int shares) {
    if (total < (1LL << 22)) return static_cast<unsigned>(c * total) / static_cast<unsigned>(shares);   // shares < 2^10
    return c * total / shares;
}
// The share that tile `at` belongs to.
__device__ __forceinline__ int share_of(long long at, long long total, int shares) {
    if (total < (1LL << 22)) return static_cast<unsigned>((at + 1) * shares - 1) / static_cast<unsigned>(total);
    return static_cast<int>(((at + 1) * shares - 1) / total);
}

// The capped score  cap2 * tanh(y),  y = scale s / cap, with z = s * inner = 2 log2(e) y:  tanh(y) = 1 - 2 / (1 + 2^z).
// The three steps' errors (2^-22 each) stay whole where the difference is small: a score is off by up to cap * 2^-21.
__device__ __forceinline__ float capped(const AttnParams& p, float s) {
    return fmaf(-2.f * p.cap2, rcp_approx(1.f + exp2_approx(s * p.inner)), p.cap2);
}
// The same for caps above kSeriesCap, where that would show: |y| < 1/4 takes the odd series of tanh, of which the first
// term left out, 1382/155925 y^10, is 2^-26.8 of the first; from there on the difference is 0.245 at least, and the score is
// off by 2^-18.9 of itself.  (Up to a cap of 64 the way above loses 2^-15 at most, and keeps its results.)  48 requests,
// window 1024, 16 heads of 64: 38.3 us this way, 38.2 the other.
constexpr float kSeriesCap = 64.f;
__device__ __forceinline__ float capped_by_series(const AttnParams& p, float s) {
    constexpr double k2 = 0.12011325347955035;        // (ln(2) / 2)^2: y^2 = k2 z^2
    constexpr float a1 = -1. / 3. * k2, a2 = 2. / 15. * k2 * k2, a3 = -17. / 315. * k2 * k2 * k2, a4 = 62. / 2835. * k2 * k2 * k2 * k2;
    const float z = s * p.inner, u = z * z, x = s * p.scale2;
    const float odd = fmaf(x * u, fmaf(u, fmaf(u, fmaf(u, a4, a3), a2), a1), x);
    return fabsf(z) < 0.72f ? odd : capped(p, s);     // 0.25 * 2 log2(e) = 0.7213
}

template <bool BF16>
__device__ __forceinline__ uint2 pack4(float4 x) { return make_uint2(pack2<BF16>(x.x, x.y), pack2<BF16>(x.z, x.w)); }
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void store_lse(const AttnParams& p, long long head, float sum, float top) {
    if (p.lse != nullptr) p.lse[head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Joins the parts that the CTAs of a cluster have in their shared memory: rows * D of o, then rows (m, l).  Every CTA
// takes its share of the elements and reads all the parts.
template <int D, bool BF16, int ROWS>
__device__ __forceinline__ void join_cluster(const AttnParams& p, const float* part) {
    const int tid = threadIdx.x, rank = static_cast<int>(cluster_rank()), unit = blockIdx.x / p.cluster;
    const int per_request = p.heads_k * p.row_blocks;
    const int b = unit / per_request, u = unit - b * per_request, hk = u / p.row_blocks, row0 = (u - hk * p.row_blocks) * ROWS;
    const int rows = min(ROWS, p.group - row0);
    const long long head0 = static_cast<long long>(b) * p.heads + hk * p.group + row0;
    const uint32_t mine = smem_u32(part);
    cluster_arrive();
    cluster_wait();                  // the parts are there
    for (int i = (rank * kAttnThreads + tid) * 4; i < rows * D; i += p.cluster * kAttnThreads * 4) {
        const int row = i / D;
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < p.cluster; ++c) {
            const uint32_t theirs = cluster_addr(mine, c);
            const float2 ml = ld_cluster_v2(theirs + (ROWS * D + 2 * row) * 4);
            if (ml.y == 0.f) continue;                   // nothing seen; its o may never have been written
            const float4 x = ld_cluster_v4(theirs + i * 4);
            const float now = fmaxf(top, ml.x), f = exp2_approx(top - now), g = exp2_approx(ml.x - now);
            sum = sum * f + ml.y * g;
            acc.x = acc.x * f + x.x * g, acc.y = acc.y * f + x.y * g, acc.z = acc.z * f + x.z * g, acc.w = acc.w * f + x.w * g;
            top = now;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
        *reinterpret_cast<uint2*>(p.out + head0 * D + i) = pack4<BF16>(acc);
        if (i % D == 0) store_lse(p, head0 + row, sum, top);
    }
    cluster_arrive();
    cluster_wait();                  // and have been read
}

// ALONE: every warp takes whole units, every so-manieth, by itself - for many short ones.  Else the four warps of a CTA
// take the keys of a tile together.
template <int D, bool BF16, int NT, bool CAP, bool ALONE>
__global__ void __launch_bounds__(kAttnThreads, AttnCfg<D, NT>::kCtas) paged_attention_kernel(const AttnParams p) {
    using C = AttnCfg<D, NT>;
    constexpr int MT = C::kKeys / 16, KK = D / 16, DT = D / 16, KEYS = C::kKeys, STAGES = C::kStages;
    constexpr int ROWS = NT * 8;
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ long long s_scan[kWarps], s_at, s_total;
    __shared__ int s_request, s_len;
    __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
    struct Step { int b, unit, rel, last; uint32_t mask; int pad[3]; };     // last: 1 ends the share, 2 ends its unit
    __shared__ Step s_step[kWarps][STAGES];
    pdl_wait_prior_grid();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_request = p.heads_k * p.row_blocks, share = blockIdx.x;

    // ---- my share; the loader's place: request, unit within the request, tile
    constexpr int TILE = ALONE ? KEYS : C::kTile;    // keys of a place in the sequence
    int lb, lu, lt, left;                            // left: places of the share (ALONE: of the unit) still to be loaded
    int gap = 0;                                     // places that the end of a unit counts as
    Range lr;
    // ALONE: the unit that is loaded, the step to the next, all of them, and the next one's length, asked for ahead
    int unit = share * kWarps + warp, next_len = 0;
    const int stride = static_cast<int>(gridDim.x) * kWarps, units = p.batch * per_request;
    auto begin_unit = [&](int len) {
        lb = unit / per_request;
        lu = unit - lb * per_request;
        lr = key_range<TILE>(p, len);
        lt = lr.tile_lo;
        left = lr.tile_hi - lt;
        if (units - unit > stride) next_len = p.lens[(unit + stride) / per_request];
    };
    if constexpr (ALONE) {
        if (unit >= units) return;
        begin_unit(p.lens[unit / per_request]);
    } else     if (p.cluster > 0) {
        const int rank = static_cast<int>(cluster_rank()), mine = share / p.cluster;
        lb = mine / per_request;
        lu = mine - lb * per_request;
        lr = key_range<C::kTile>(p, p.lens[lb]);
        const int tiles = lr.tile_hi - lr.tile_lo;       // 8 CTAs at most, of ten tiles
        lt = lr.tile_lo + tiles * rank / p.cluster;
        left = lr.tile_lo + tiles * (rank + 1) / p.cluster - lt;
    } else {
        long long total, begin, at;                  // places: all of them, the share's first, the request's first
        int len;
        auto count = [&](long long tiles) {          // the share, now that the number of tiles is known
            gap = tiles >= static_cast<long long>(kLongShare) * gridDim.x ? C::kUnitEnd : 0;
            total = tiles + static_cast<long long>(gap) * units;
            const int shares = total < gridDim.x ? static_cast<int>(total) : static_cast<int>(gridDim.x);
            if (share >= shares) return false;       // fewer tiles than CTAs, so the cuts are told by unit
            begin = share_begin(share, total, shares);
            left = static_cast<int>(share_begin(share + 1, total, shares) - begin);
            return true;
        };
        if (p.batch <= 32) {
            // every warp by itself: a request per lane, no barrier
            len = lane < p.batch ? p.lens[lane] : 0;
            const Range r = key_range<C::kTile>(p, len);
            const int tiles = lane < p.batch ? r.tile_hi - r.tile_lo : 0;    // 32 of them: below 2^31
            int upto = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            if (!count(static_cast<long long>(__shfl_sync(0xffffffffu, upto, 31)) * per_request)) return;
            at = (static_cast<long long>(upto - tiles) + gap * lane) * per_request;
            lb = __popc(__ballot_sync(0xffffffffu, lane < p.batch && at <= begin)) - 1;
            len = __shfl_sync(0xffffffffu, len, lb);
            at = __shfl_sync(0xffffffffu, at, lb);
        } else {
            const int chunk = (p.batch + kAttnThreads - 1) / kAttnThreads;
            const int b_lo = min(tid * chunk, p.batch), b_hi = min(b_lo + chunk, p.batch);
            long long mine = 0;
            for (int b = b_lo; b < b_hi; ++b) {
                const Range r = key_range<C::kTile>(p, p.lens[b]);
                mine += static_cast<long long>(r.tile_hi - r.tile_lo) * per_request;
            }
            const long long upto = block_scan(mine, s_scan);
            if (tid == kAttnThreads - 1) s_total = upto;
            __syncthreads();
            if (!count(s_total)) return;
            long long from = upto - mine + static_cast<long long>(gap) * b_lo * per_request;
            if (begin >= from && begin < upto + static_cast<long long>(gap) * b_hi * per_request) {
                for (int b = b_lo; b < b_hi; ++b) {
                    const int length = p.lens[b];
                    const Range r = key_range<C::kTile>(p, length);
                    const long long n = static_cast<long long>(r.tile_hi - r.tile_lo + gap) * per_request;
                    if (begin < from + n) {
                        s_request = b;
                        s_len = length;
                        s_at = from;
                        break;
                    }
                    from += n;
                }
            }
            __syncthreads();
            lb = s_request;
            len = s_len;
            at = s_at;
        }
        if (tid == 0) s_total = total;               // (read again by this thread only)
        lr = key_range<C::kTile>(p, len);
        const unsigned off = static_cast<unsigned>(begin - at);     // below (tiles + gap) * per_request: 32 bits, checked
        const unsigned places = lr.tile_hi - lr.tile_lo + gap;
        lu = off / places;
        const int place = off - lu * places;
        lt = lr.tile_lo + place;
        if (lt >= lr.tile_hi) {                      // at the end of a unit: the share begins with the next one
            left -= places - place;
            if (++lu == per_request) {
                lu = 0;
                if (++lb < p.batch) lr = key_range<C::kTile>(p, p.lens[lb]);
            }
            lt = lr.tile_lo;
        }
        if (left <= 0) {                             // (and has nothing of it)
            if (tid == 0 && !p.cuts_by_unit) p.cuts[share].count = 0;
            return;
        }
    }
    bool from_begin = lt == lr.tile_lo;              // this part of a unit contains its first key

    const uint32_t ring_u = smem_u32(s_ring) + warp * (C::kStageBytes * STAGES);
    float* join = reinterpret_cast<float*>(s_ring + C::kRingBytes);
    const uint32_t join_u = smem_u32(join);

    constexpr int CH = D / 8;                        // 16-byte chunks of a row
    constexpr int RPI = 32 / CH;                     // rows that one instruction of the warp loads
    const int lrow = lane / CH, lcol = (lane % CH) * 8;

    // The query rows of a unit: to registers, or - where they go through shared memory - on their way to the L1.  Asked
    // for ahead of the loads of keys, behind which they would wait: when the launch begins, and when a unit ends.
    uint32_t qf[C::kQueryInSmem ? 1 : NT][C::kQueryInSmem ? 1 : KK][2];
    auto ask_queries = [&](int b, int unit) {
        const int hk = p.row_blocks == 1 ? unit : unit / p.row_blocks, row0 = (unit - hk * p.row_blocks) * ROWS;
        const uint16_t* qrow = p.q + b * p.q_batch + (static_cast<long long>(hk) * p.group + row0) * p.q_head;
        if constexpr (C::kQueryInSmem) {
            constexpr int LINES = D / 64;
            if (tid < ROWS * LINES && row0 + tid / LINES < p.group)
                asm volatile("prefetch.global.L1 [%0];" ::"l"(qrow + (tid / LINES) * p.q_head + (tid % LINES) * 64));
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = n * 8 + lane / 4;
#pragma unroll
                for (int k = 0; k < KK; ++k) {
                    const uint16_t* x = qrow + r * p.q_head + k * 16 + (lane % 4) * 2;
                    qf[n][k][0] = row0 + r < p.group ? *reinterpret_cast<const uint32_t*>(x) : 0u;
                    qf[n][k][1] = row0 + r < p.group ? *reinterpret_cast<const uint32_t*>(x + 8) : 0u;
                }
            }
        }
    };
    ask_queries(lb, lu);

    // The page of my key of the step at (lb, lt); looked up one step ahead, so that its latency is not waited for.
    // `found`: the key is visible; `row_in`: its row in the page.
    int page = 0, row_in = 0;
    bool found = false;
    auto look_up = [&]() {
        const int key = lt * TILE + (ALONE ? 0 : warp * KEYS) + (lane % KEYS);
        found = key >= lr.lo && key < lr.hi;
        if (found) {
            const int at = page_of(key, p.page);
            page = p.table[lb * p.table_stride + at];
            row_in = key - at * static_cast<int>(p.page.size);
        }
    };
    look_up();

    if (!ALONE && left == 0) {                       // a cluster that has more CTAs than the unit tiles
        for (int r = tid; r < ROWS; r += kAttnThreads)
            *reinterpret_cast<float2*>(s_ring + (ROWS * D + 2 * r) * 4) = make_float2(-INFINITY, 0.f);
        join_cluster<D, BF16, ROWS>(p, reinterpret_cast<const float*>(s_ring));
        return;
    }
    float o[DT][NT][4], m[NT][2], l[NT][2];
    bool fresh = true;               // a unit begins
    int stage = 0, ahead = STAGES - 1;               // steps to load before the first is waited for
    for (;;) {
        // ---- load the step that is STAGES - 1 ahead
        __syncwarp();                // every lane has read the stage that is filled
        if (left > 0) {
            const uint32_t mask = __ballot_sync(0xffffffffu, found && page >= 0 && page < p.num_pages);
            const int hk = p.row_blocks == 1 ? lu : lu / p.row_blocks;
            const uint16_t* kb = p.k + hk * p.k_head + lcol;
            const uint16_t* vb = p.v + hk * p.v_head + lcol;
            const int load_stage = ahead > 0 ? STAGES - 1 - ahead : stage == 0 ? STAGES - 1 : stage - 1;
            const uint32_t dst = ring_u + load_stage * C::kStageBytes;
            const bool ok = (mask >> (lane % KEYS)) & 1u;
            const long long ko = ok ? page * p.k_page + row_in * p.k_row : 0, vo = ok ? page * p.v_page + row_in * p.v_row : 0;
#pragma unroll(NT > 2 ? 4 : KEYS / RPI)
            for (int i = 0; i < KEYS / RPI; ++i) {
                const int row = i * RPI + lrow;
                const long long kro = __shfl_sync(0xffffffffu, ko, row), vro = __shfl_sync(0xffffffffu, vo, row);
                const uint32_t bytes = (mask >> row) & 1u ? 16u : 0u;
                const uint32_t at = dst + row * (D * 2) + (((lane % CH) ^ (row & 7)) << 4);
                cp_async16(at, kb + kro, bytes);
                cp_async16(at + KEYS * D * 2, vb + vro, bytes);
            }
            if (lane == 0) {
                Step& st = s_step[warp][load_stage];
                st.b = lb;
                st.unit = lu;
                st.rel = lt * TILE + (ALONE ? 0 : warp * KEYS) - (lr.hi - 1);
                st.mask = KEYS == 32 ? mask : mask & 0xffffu;
                if constexpr (ALONE) st.last = left > 1 ? 0 : units - unit > stride ? 2 : 3;
                else st.last = (left <= (lt + 1 == lr.tile_hi ? 1 + gap : 1) ? 1 : 0) | (lt + 1 == lr.tile_hi ? 2 : 0);
            }
            if constexpr (ALONE) {
                ++lt;
                if (--left == 0 && units - unit > stride) {
                    unit += stride;
                    begin_unit(next_len);
                }
                if (left > 0) look_up();
            } else {
                left -= lt + 1 == lr.tile_hi ? 1 + gap : 1;
                if (left > 0) {
                    if (++lt == lr.tile_hi) {
                        if (++lu == per_request) {
                            lu = 0;
                            ++lb;
                            lr = key_range<C::kTile>(p, p.lens[lb]);
                        }
                        lt = lr.tile_lo;
                    }
                    look_up();
                }
            }
        }
        cp_async_commit();
        if (ahead > 0) {
            --ahead;
            continue;
        }
        __syncwarp();
        const Step st = s_step[warp][stage];
        const int hk = p.row_blocks == 1 ? st.unit : st.unit / p.row_blocks;
        const int row0 = (st.unit - hk * p.row_blocks) * ROWS;               // first query head in the group
        if (fresh) {
            fresh = false;
            if constexpr (C::kQueryInSmem) {
                const uint16_t* qrow = p.q + st.b * p.q_batch + (static_cast<long long>(hk) * p.group + row0) * p.q_head;
                // all four warps are here: the unit before has been joined, and the first begins with the launch
                for (int i = tid; i < ROWS * CH; i += kAttnThreads) {
                    const int r = i / CH, c = i % CH;
                    const uint4 x = row0 + r < p.group ? ld_v4(qrow + r * p.q_head + c * 8) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(join) + r * (D * 2) + ((c ^ (r & 7)) << 4)) = x;
                }
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m[n][e] = -INFINITY;
                    l[n][e] = 0.f;
                }
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][n][e] = 0.f;
            }
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t kaddr = ring_u + stage * C::kStageBytes, vaddr = kaddr + KEYS * D * 2;
        // ---- S^T = K Q^T
        float s[MT][NT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < KK; ++k) {
            uint32_t qs[NT][2];
            if constexpr (C::kQueryInSmem) {
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t x[4];
                    const int r = n * 8 + (lane & 7) + ((lane >> 4) << 3);
                    ldmatrix_x4(x, join_u + r * (D * 2) + (((k * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
                    qs[n][0] = x[0], qs[n][1] = x[1], qs[n + 1][0] = x[2], qs[n + 1][1] = x[3];
                }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t a[4];
                const int row = t * 16 + (lane & 15);
                ldmatrix_x4(a, kaddr + row * (D * 2) + (((k * 2 + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (C::kQueryInSmem) mma16816<BF16>(s[t][n], a, qs[n][0], qs[n][1]);
                    else mma16816<BF16>(s[t][n], a, qf[n][k][0], qf[n][k][1]);
                }
            }
        }
        // ---- scores in powers of two
        if (CAP && p.cap_series) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][n][e] = capped_by_series(p, s[t][n][e]);
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][n][e] = CAP ? capped(p, s[t][n][e]) : s[t][n][e] * p.scale2;
        }
        if (p.slopes != nullptr) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = row0 + n * 8 + (lane % 4) * 2 + r;
                    const float slope = row < p.group ? p.slopes[hk * p.group + row] * kLog2e : 0.f;
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int e = r; e < 4; e += 2)
                            s[t][n][e] = fmaf(slope, static_cast<float>(st.rel + t * 16 + lane / 4 + (e >> 1) * 8), s[t][n][e]);
                }
        }
        if (st.mask != (KEYS == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool seen = (st.mask >> (t * 16 + lane / 4 + (e >> 1) * 8)) & 1u;
#pragma unroll
                    for (int n = 0; n < NT; ++n) s[t][n][e] = seen ? s[t][n][e] : -INFINITY;
                }
        }
        float top[NT][2];
        bool grown = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = fmaxf(s[0][n][r], s[0][n][r + 2]);
#pragma unroll
                for (int t = 1; t < MT; ++t) x = fmaxf(x, fmaxf(s[t][n][r], s[t][n][r + 2]));
                top[n][r] = x;
                grown |= x > m[n][r] + (kGrowth + kHeadroom<BF16>);
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x = top[n][r];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float now = fmaxf(m[n][r], x - kHeadroom<BF16>);
                    const float f = exp2_approx(m[n][r] - finite_ref(now));
                    m[n][r] = now;
                    l[n][r] *= f;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        o[t][n][r] *= f;
                        o[t][n][r + 2] *= f;
                    }
                }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float r0 = finite_ref(m[n][0]), r1 = finite_ref(m[n][1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p0 = exp2_approx(s[t][n][2 * h] - r0);
                    const float p1 = exp2_approx(s[t][n][2 * h + 1] - r1);
                    l[n][0] += p0;
                    l[n][1] += p1;
                    const uint32_t w = pack2<BF16>(p0, p1);
                    const float2 back = unpack2<BF16>(w);
                    hi[n][h] = movmatrix(w);
                    lo[n][h] = movmatrix(pack2<BF16>(p0 - back.x, p1 - back.y));
                }
            }
            const int row = t * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                uint32_t a[4];
                ldmatrix_x4_trans(a, vaddr + row * (D * 2) + (((dt * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816<BF16>(o[dt][n], a, hi[n][0], hi[n][1]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816<BF16>(o[dt][n], a, lo[n][0], lo[n][1]);
            }
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (st.last == 0) continue;

        if constexpr (ALONE) {
            // ---- the unit ends: this warp has all of it
            if ((st.last & 1) == 0) {
                const Step& next = s_step[warp][stage];
                ask_queries(next.b, next.unit);
            }
            const long long head0 = static_cast<long long>(st.b) * p.heads + hk * p.group;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = l[0][r];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int row = (lane % 4) * 2 + r;
                if (row >= p.group) continue;
                const float inv = x == 0.f ? 0.f : 1.f / x;
                uint16_t* const out = p.out + (head0 + row) * D + lane / 4;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) out[t * 16 + h * 8] = static_cast<uint16_t>(pack2<BF16>(o[t][0][r + 2 * h] * inv, 0.f));
                if (lane < 4) store_lse(p, head0 + row, x, m[0][r]);
            }
            if ((st.last & 1) != 0) break;
            fresh = true;
            continue;
        }
        // ---- the unit ends, or the share does: the four warps' results become one.  Each warp scales its own to the
        // maximum of the four; what is left is a sum, eight heads at a time through shared memory.
        if (!C::kQueryInSmem && (st.last & 1) == 0) {
            const Step& next = s_step[warp][stage];
            ask_queries(next.b, next.unit);
        }
        const bool whole = p.cluster <= 1 && from_begin && (st.last & 2) != 0;
        const int rows = min(p.group - row0, ROWS);
        const long long head0 = static_cast<long long>(st.b) * p.heads + hk * p.group + row0;
        // a cluster's parts stay in shared memory, where the loads, all done, have been
        float* const part = p.cluster > 1 ? reinterpret_cast<float*>(s_ring)
                                          : p.parts + (2 * static_cast<long long>(share) + (from_begin ? 1 : 0)) * p.part_floats;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = l[n][r];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (lane < 4) {
                    s_m[warp][n * 8 + lane * 2 + r] = m[n][r];
                    s_l[warp][n * 8 + lane * 2 + r] = x;
                }
            }
        __syncthreads();             // (and, with the query rows in shared memory: they are not needed any more)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n * 8 >= rows) break;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = n * 8 + (lane % 4) * 2 + r;
                const float most = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
                const float f = exp2_approx(m[n][r] - finite_ref(most));
                if (row < rows)
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            join[(warp * 8 + (lane % 4) * 2 + r) * D + ((t * 16 + h * 8 + lane / 4) ^ ((lane % 4) * 8))] = o[t][n][r + 2 * h] * f;
            }
            __syncthreads();
            const int mine = min(8, rows - n * 8) * D / 4;
            for (int i = tid; i < mine; i += kAttnThreads) {
                const int r = i / (D / 4), d = i % (D / 4) * 4, row = n * 8 + r;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                float most = -INFINITY, weight = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(&join[(w * 8 + r) * D + (d ^ ((r >> 1) * 8))]);
                    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
                    most = fmaxf(most, s_m[w][row]);
                }
#pragma unroll
                for (int w = 0; w < kWarps; ++w) weight = fmaf(s_l[w][row], exp2_approx(s_m[w][row] - finite_ref(most)), weight);
                if (whole) {
                    const float inv = weight == 0.f ? 0.f : 1.f / weight;
                    sum.x *= inv, sum.y *= inv, sum.z *= inv, sum.w *= inv;
                    *reinterpret_cast<uint2*>(p.out + (head0 + row) * D + d) = pack4<BF16>(sum);
                    if (d == 0) store_lse(p, head0 + row, weight, most);
                } else {
                    *reinterpret_cast<float4*>(part + row * D + d) = sum;
                    if (d == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * row) = make_float2(most, weight);
                }
            }
            __syncthreads();
        }
        if (tid == 0 && p.cluster == 0 && (p.cuts_by_unit ? from_begin : (st.last & 1) != 0)) {
            CutInfo cut{st.b * per_request + st.unit, share, 0, 0};
            if (from_begin && !whole) {              // the last part here: it ends with the share
                const Range r = key_range<C::kTile>(p, p.lens[st.b]);
                const int shares = s_total < gridDim.x ? static_cast<int>(s_total) : static_cast<int>(gridDim.x);
                const int done = (st.rel + r.hi - 1) / C::kTile - r.tile_lo + 1;
                const long long unit_end = share_begin(share + 1, s_total, shares) - done + (r.tile_hi - r.tile_lo);
                cut.count = share_of(unit_end - 1, s_total, shares) - share + 1;
            }
            p.cuts[p.cuts_by_unit ? cut.unit : share] = cut;
        }
        if ((st.last & 1) != 0) break;
        fresh = true;
        from_begin = true;
    }
    cp_async_wait<0>();
    if (!ALONE && p.cluster > 1) join_cluster<D, BF16, ROWS>(p, reinterpret_cast<const float*>(s_ring));
}

// Joins the parts of the units that several shares worked on.  CTA (x, y): the unit of cut x, rows from
// y * rows_per_cta on; the CTA's warps are shared out evenly among its rows, take a row's parts in turn, four at a time
// with all their loads in flight, and are joined through shared memory.  Bound by the latency of two dependent
// loads: 4.1 to 4.9 us with cold caches, of which 2 are the launch; 7.4 for 16 units of 18 parts and 32 rows.
constexpr int kJoinThreads = 512;      // at most

template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads, 2) paged_join_kernel(const AttnParams p, int rows, int rows_per_cta) {
    constexpr int kJoinWarps = kJoinThreads / 32, V = D / 64, U = 4;      // V: pairs of elements of a lane
    __shared__ float2 s_o[kJoinWarps][D / 2];
    __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = static_cast<int>(blockDim.x / 32) / rows_per_cta, member = warp % team, row = blockIdx.y * rows_per_cta + warp / team;
    pdl_wait_prior_grid();
    const int4 cut = *reinterpret_cast<const int4*>(p.cuts + blockIdx.x);
    const int count = cut.z;
    if (count == 0) return;
    float top = -INFINITY, sum = 0.f;
    float2 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float2(0.f, 0.f);
    // (a row behind the group's last holds nothing, and is not stored below)
    for (int i0 = member; i0 < count; i0 += U * team) {
        float2 ml[U], x[U][V];
#pragma unroll
        for (int c = 0; c < U; ++c) {
            const int i = i0 + c * team;
            ml[c] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int v = 0; v < V; ++v) x[c][v] = make_float2(0.f, 0.f);
            if (i < count && row < rows) {
                const float* part = p.parts + (2 * static_cast<long long>(cut.y + i) + (i == 0 ? 1 : 0)) * p.part_floats;
                ml[c] = *reinterpret_cast<const float2*>(part + rows * D + 2 * row);
#pragma unroll
                for (int v = 0; v < V; ++v) x[c][v] = *reinterpret_cast<const float2*>(part + row * D + v * 64 + lane * 2);
            }
        }
        float now = top;
#pragma unroll
        for (int c = 0; c < U; ++c) now = fmaxf(now, ml[c].x);
        const float ref = finite_ref(now), f = exp2_approx(top - ref);
        sum *= f;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v].x *= f, acc[v].y *= f;
#pragma unroll
        for (int c = 0; c < U; ++c) {
            const float g = exp2_approx(ml[c].x - ref);
            sum = fmaf(g, ml[c].y, sum);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                acc[v].x = fmaf(g, x[c][v].x, acc[v].x);
                acc[v].y = fmaf(g, x[c][v].y, acc[v].y);
            }
        }
        top = now;
    }
    if (lane == 0) {
        s_m[warp] = top;
        s_l[warp] = sum;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) s_o[warp][v * 32 + lane] = acc[v];
    __syncthreads();
    const int per_request = p.heads_k * p.row_blocks;
    const int b = cut.x / per_request, u = cut.x - b * per_request, hk = u / p.row_blocks, row0 = (u - hk * p.row_blocks) * rows;
    if (member != 0 || row >= rows || row0 + row >= p.group) return;
    for (int w = 1; w < team; ++w) {
        const float now = fmaxf(top, s_m[warp + w]), ref = finite_ref(now);
        const float f = exp2_approx(top - ref), g = exp2_approx(s_m[warp + w] - ref);
        sum = sum * f + s_l[warp + w] * g;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 x = s_o[warp + w][v * 32 + lane];
            acc[v].x = acc[v].x * f + x.x * g;
            acc[v].y = acc[v].y * f + x.y * g;
        }
        top = now;
    }
    const long long head = static_cast<long long>(b) * p.heads + hk * p.group + row0 + row;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v)
        *reinterpret_cast<uint32_t*>(p.out + head * D + v * 64 + lane * 2) = pack2<BF16>(acc[v].x * inv, acc[v].y * inv);
    if (lane == 0) store_lse(p, head, sum, top);
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
constexpr int kMaxDevices = 64;
static std::atomic<unsigned long long> g_launches{0};
static std::atomic<int> g_sm_count[kMaxDevices];       // 0: not asked yet, -1: not compute capability 10.x

struct DeviceGuard {
    int prev = -1;
    bool switched = false;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) {
            err = cudaSetDevice(dev);
            switched = err == cudaSuccess;
        }
    }
    ~DeviceGuard() {
        if (switched) cudaSetDevice(prev);
    }
};

static int cuda_failed() {
    cudaGetLastError();                                // do not leave the error for the caller's next call
    return FA_PAGED_ERR_CUDA;
}

// SMs of the device, or a negative error code.
static int sm_count(int device) {
    int n = g_sm_count[device].load(std::memory_order_relaxed);
    if (n == 0) {
        int major = 0;
        if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess ||
            cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
            return cuda_failed();
        if (major != 10) n = -1;
        g_sm_count[device].store(n, std::memory_order_relaxed);
    }
    return n > 0 ? n : FA_PAGED_ERR_ARCH;
}

template <typename Kern, typename... Args>
static int launch_cluster(Kern kern, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return cuda_failed();
    ++g_launches;
    return FA_PAGED_OK;
}
template <typename Kern, typename... Args>
static int launch_chained(Kern kern, dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    return launch_cluster(kern, grid, threads, smem, 1, stream, args...);
}

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device.
template <typename Kern>
static int allow_smem(Kern kern, int bytes, std::atomic<unsigned long long>& done, int device) {
    const unsigned long long bit = 1ULL << device;
    if (done.load(std::memory_order_acquire) & bit) return FA_PAGED_OK;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return cuda_failed();
    done.fetch_or(bit, std::memory_order_release);
    return FA_PAGED_OK;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static bool stride8(long long s) { return s >= 0 && s % 8 == 0; }

static int check_device(int device) { return device >= 0 && device < kMaxDevices ? FA_PAGED_OK : FA_PAGED_ERR_SHAPE; }

static int check_cache(const FaPagedCache& c) {
    if (c.num_pages < 0 || c.heads_k <= 0 || c.page_size <= 0) return FA_PAGED_ERR_SHAPE;
    if (c.head_dim != 64 && c.head_dim != 128) return FA_PAGED_ERR_HEAD_DIM;
    if (c.num_pages > 0 && (c.k == nullptr || c.v == nullptr)) return FA_PAGED_ERR_NULL;
    if (!aligned16(c.k) || !aligned16(c.v) || !stride8(c.k_page_stride) || !stride8(c.k_head_stride) ||
        !stride8(c.k_row_stride) || !stride8(c.v_page_stride) || !stride8(c.v_head_stride) || !stride8(c.v_row_stride))
        return FA_PAGED_ERR_ALIGN;
    return FA_PAGED_OK;
}

static int check_rotary(const FaRotarySpec& r, int head_dim) {
    if (r.freqs == nullptr || r.positions == nullptr) return FA_PAGED_ERR_NULL;
    if (r.rot_dim < 2 || r.rot_dim > head_dim || r.rot_dim % 2 != 0) return FA_PAGED_ERR_ROTARY;
    if (!std::isfinite(r.mscale)) return FA_PAGED_ERR_ROTARY;
    return FA_PAGED_OK;
}

static void fill_rotary(RotaryParams* p, const FaRotarySpec& r) {
    p->freqs = r.freqs;
    p->positions = r.positions;
    p->positions_64 = r.positions_64 != 0;
    p->rot = r.rot_dim;
    p->mscale = r.mscale;
    p->sign = r.adjoint ? -1.f : 1.f;
}

template <int D, bool BF16>
static int launch_rotary(RotaryParams p, bool interleaved, long long tokens, int outer, int sms, cudaStream_t stream) {
    constexpr int kHeadsAtOnce = kRotaryThreads / (D / 16);
    const long long heads = static_cast<long long>(p.rows[0].heads) + p.rows[1].heads + p.rows[2].heads;
    p.tokens = static_cast<int>(tokens);
    p.per_cta = 1;
    while (p.per_cta < kRotaryTokens && 2 * heads * p.per_cta <= kRotaryBatch * kHeadsAtOnce &&
           tokens * outer >= 2LL * p.per_cta * kRotaryWaves * sms)
        p.per_cta *= 2;
    const dim3 grid(static_cast<unsigned>((tokens + p.per_cta - 1) / p.per_cta), static_cast<unsigned>(outer));
    if (interleaved) return launch_chained(rotary_kernel<D, BF16, kNeighbours>, grid, kRotaryThreads, 0, stream, p);
    if (p.rot % 16 == 0) return launch_chained(rotary_kernel<D, BF16, kHalves>, grid, kRotaryThreads, 0, stream, p);
    return launch_chained(rotary_kernel<D, BF16, kRaggedHalves>, grid, kRotaryThreads, 0, stream, p);
}

static int launch_rotary(const RotaryParams& p, bool interleaved, long long tokens, int outer, int head_dim, int dtype,
                         int sms, cudaStream_t stream) {
    const bool bf16 = dtype == FA_PAGED_BF16;
    if (head_dim == 128)
        return bf16 ? launch_rotary<128, true>(p, interleaved, tokens, outer, sms, stream)
                    : launch_rotary<128, false>(p, interleaved, tokens, outer, sms, stream);
    return bf16 ? launch_rotary<64, true>(p, interleaved, tokens, outer, sms, stream)
                : launch_rotary<64, false>(p, interleaved, tokens, outer, sms, stream);
}

// Short units, as far as the table's width and the window show it (the lengths are on the device; a request of 333 keys
// takes 5.7 us of GPU time under a table of 368 and 6.3 under one of 8192, called from Python 7 and 9): each is done by a
// cluster of 1 to 8 CTAs that join their parts through their shared memory.  No sums
// over the lengths, no partial results in memory, no second kernel (which costs the host 2.7 us, too).  Up to so many
// tiles for a CTA: 4, and 6 more as the clusters fill the GPU, where equal shares of all keys have no SMs to win.  GPU
// time with clusters and with equal shares, 4 KV heads of 128: one request of 300 keys 5.9 and 6.5 us, of 2000 (4 tiles
// a CTA) 7.9 and 6.9, of 3000 9.7 and 7.2; 4 requests of 2500 (5) 9.1 and 9.3, of 4000 12.0 and 10.0; 8 of 4000 (8) 15.0
// and 15.5; 16 of 2000 (8) 14.8 and 16.1, of 3000 (12) 19.4 and 19.0.
constexpr int kUnitTiles = 4, kUnitTilesFull = 6;
constexpr int kMostCluster = 8;
// Many short units: one warp each, nothing to join (up to 8 heads; more keep four warps busy at the end of a unit as
// well).  Up to so many keys that the table or the window could hold, and in proportion fewer where there are fewer units
// than 3 per CTA, three quarters of the warps.  Against equal shares, 32 KV heads of 128: 128 requests of up to 30 keys
// 13.5 and 46.6 us, of 200 50.7 and 60.7, of 400 94.4 and 91.5; 32 requests of 400 29.4 and 30.0; 16 requests (512 units)
// of 200 14.9 and 15.0, of 400 26.4 and 20.0.  At 64: 128 requests of 30 7.2 and 29.5, of 400 48.5 and 49.8, of 700 80.9
// and 78.8.
constexpr int kAloneKeys = 384, kAloneUnits = 3;

struct AttnPlan {
    int grid, nt, row_blocks;
    int cluster;
    bool alone;
    long long part_floats;
    int cuts, rows_per_cta, join_warps;       // of the joining kernel
    size_t cut_bytes, bytes;
};

static float score_inner(const FaPagedAttentionArgs* a) {
    return a->softcap > 0.f ? static_cast<float>(2.0 * 1.4426950408889634 * a->scale / a->softcap) : 0.f;
}

static int check_attention(const FaPagedAttentionArgs* a) {
    if (a == nullptr) return FA_PAGED_ERR_NULL;
    if (a->struct_size != sizeof(FaPagedAttentionArgs)) return FA_PAGED_ERR_ABI;
    int rc = check_device(a->device);
    if (rc != FA_PAGED_OK) return rc;
    if (a->dtype != FA_PAGED_FP16 && a->dtype != FA_PAGED_BF16) return FA_PAGED_ERR_DTYPE;
    rc = check_cache(a->cache);
    if (rc != FA_PAGED_OK) return rc;
    if (a->batch < 0 || a->heads < 0 || a->table_width < 0 || a->heads % a->cache.heads_k != 0 || a->table_stride < 0)
        return FA_PAGED_ERR_SHAPE;
    // key numbers are 32 bits, with room for the last tile; so are the units
    if (static_cast<long long>(a->table_width) * a->cache.page_size > INT_MAX - 1024 ||
        static_cast<long long>(a->batch) * a->heads > INT_MAX)
        return FA_PAGED_ERR_SHAPE;
    if (a->window < 0 || !std::isfinite(a->scale) || !std::isfinite(a->softcap) || a->scale < 0.f || a->softcap < 0.f)
        return FA_PAGED_ERR_SCORE;
    if (!std::isfinite(a->scale * kLog2e) || !std::isfinite(a->softcap * kLog2e) || !std::isfinite(score_inner(a)))
        return FA_PAGED_ERR_SCORE;
    if (!aligned16(a->q) || !aligned16(a->out) || !stride8(a->q_batch_stride) || !stride8(a->q_head_stride))
        return FA_PAGED_ERR_ALIGN;
    return FA_PAGED_OK;
}

template <int D>
static int make_attn_plan(const FaPagedAttentionArgs* a, int sms, AttnPlan* plan) {
    const int group = a->heads / a->cache.heads_k;
    // Query heads of a tile: as many as the group has.  16 requests of 16384 keys on one key head: 8 heads 23.9 us (with
    // tiles of 16: 25.1), 12 heads 26.1 (of 8, twice: 32.5; of 32: 30.8), 16 heads 27.1 (32.9; 31.2), 32 heads 37.1 (of 16,
    // twice: 41.0).
    plan->nt = group <= 8 ? 1 : group <= 16 ? 2 : 4;
    plan->row_blocks = (group + plan->nt * 8 - 1) / (plan->nt * 8);
    const long long capacity = static_cast<long long>(a->table_width) * a->cache.page_size;
    const long long tiles = (capacity + attn_tile(D) - 1) / attn_tile(D);
    const long long most = static_cast<long long>(a->batch) * a->cache.heads_k * plan->row_blocks * (tiles > 0 ? tiles : 1);
    const long long resident = static_cast<long long>(D == 64 && plan->nt == 1 ? AttnCfg<64, 1>::kCtas : AttnCfg<D, 2>::kCtas) * sms;
    // tiles of one request, and of one share, are counted in 32 bits
    if (tiles * a->cache.heads_k * plan->row_blocks > INT_MAX || most / resident >= INT_MAX) return FA_PAGED_ERR_SHAPE;
    // with many units, equal shares beat whole units: no last round
    const long long units = static_cast<long long>(a->batch) * a->cache.heads_k * plan->row_blocks;
    const long long seen = a->window > 0 && a->window < capacity ? a->window / attn_tile(D) + 2 : tiles;      // of one unit, at most
    int cluster = 1;
    while (cluster < kMostCluster && 2 * cluster <= seen && 2 * cluster * units <= resident) cluster *= 2;
    const long long most_keys = a->window > 0 && a->window < capacity ? a->window : capacity;
    if (plan->nt == 1 && units > resident &&
        most_keys * kAloneUnits * resident <= kAloneKeys * (units < kAloneUnits * resident ? units : kAloneUnits * resident)) {
        plan->alone = true;
        plan->cluster = 1;                             // (nothing is cut)
        plan->grid = static_cast<int>((units + kWarps - 1) / kWarps < resident ? (units + kWarps - 1) / kWarps : resident);
        return FA_PAGED_OK;
    }
    const long long ctas = units * cluster;
    if (seen <= 1 || (ctas <= resident && seen <= cluster * (kUnitTiles + kUnitTilesFull * ctas / resident))) {
        plan->cluster = cluster;
        plan->grid = static_cast<int>(ctas);
        return FA_PAGED_OK;
    }
    plan->grid = static_cast<int>(most < resident ? most : resident);
    plan->part_floats = plan->nt * 8 * (D + 2);
    plan->cuts = static_cast<int>(units < plan->grid ? units : plan->grid);
    // Few parts per unit: one CTA does all rows (up to 16) with eight warps at most.  Many: sixteen warps, and a CTA per
    // row as long as they all run at once, four to an SM.  (Sixteen warps a row cost 32 requests of 8 KV heads 0.5 us
    // and 768 units of one row 2.5; four parts a warp are one round of loads.)
    const int rows = group < plan->nt * 8 ? group : plan->nt * 8;
    plan->rows_per_cta = 1;
    if (plan->grid / units < 4) {
        while (plan->rows_per_cta < 16 && plan->rows_per_cta < rows) plan->rows_per_cta *= 2;
        plan->join_warps = plan->rows_per_cta == 1 ? 4 : plan->rows_per_cta <= 8 ? 8 : 16;
    } else {
        while (plan->rows_per_cta < 16 && static_cast<long long>(plan->cuts) * ((rows + plan->rows_per_cta - 1) / plan->rows_per_cta) > 4LL * sms)
            plan->rows_per_cta *= 2;
        plan->join_warps = 16;
    }
    plan->cut_bytes = (plan->cuts * sizeof(CutInfo) + 255) / 256 * 256;
    plan->bytes = plan->cut_bytes + 2 * plan->grid * plan->part_floats * sizeof(float);
    return FA_PAGED_OK;
}

static int attn_plan(const FaPagedAttentionArgs* a, AttnPlan* plan) {
    const int rc = check_attention(a);
    if (rc != FA_PAGED_OK) return rc;
    *plan = AttnPlan{};
    if (a->batch == 0 || a->heads == 0) return FA_PAGED_OK;
    const int sms = sm_count(a->device);
    if (sms < 0) return sms;
    return a->cache.head_dim == 128 ? make_attn_plan<128>(a, sms, plan) : make_attn_plan<64>(a, sms, plan);
}

template <int D, bool BF16, int NT, bool CAP, bool ALONE>
static int launch_attention(const AttnParams& p, const AttnPlan& plan, int device, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    constexpr int smem = AttnCfg<D, NT>::kSmem;
    int rc = allow_smem(paged_attention_kernel<D, BF16, NT, CAP, ALONE>, smem, done, device);
    if (rc != FA_PAGED_OK) return rc;
    rc = launch_cluster(paged_attention_kernel<D, BF16, NT, CAP, ALONE>, dim3(plan.grid), kAttnThreads, smem, plan.cluster, stream, p);
    if (rc != FA_PAGED_OK || plan.cluster > 0) return rc;
    const int rows = p.group < NT * 8 ? p.group : NT * 8;
    const dim3 grid(plan.cuts, (rows + plan.rows_per_cta - 1) / plan.rows_per_cta);
    return launch_chained(paged_join_kernel<D, BF16>, grid, plan.join_warps * 32, 0, stream, p, NT * 8, plan.rows_per_cta);
}

template <int D, bool BF16, int NT>
static int launch_attention(const AttnParams& p, const AttnPlan& plan, bool cap, int device, cudaStream_t stream) {
    if constexpr (NT == 1) {
        if (plan.alone)
            return cap ? launch_attention<D, BF16, NT, true, true>(p, plan, device, stream)
                       : launch_attention<D, BF16, NT, false, true>(p, plan, device, stream);
    }
    return cap ? launch_attention<D, BF16, NT, true, false>(p, plan, device, stream)
               : launch_attention<D, BF16, NT, false, false>(p, plan, device, stream);
}

template <int D, bool BF16>
static int dispatch_attention(const AttnParams& p, const AttnPlan& plan, bool cap, int device, cudaStream_t stream) {
    switch (plan.nt) {
        case 1: return launch_attention<D, BF16, 1>(p, plan, cap, device, stream);
        case 2: return launch_attention<D, BF16, 2>(p, plan, cap, device, stream);
        default: return launch_attention<D, BF16, 4>(p, plan, cap, device, stream);
    }
}

static int attention(const FaPagedAttentionArgs* a, void* workspace, size_t bytes, cudaStream_t stream) {
    AttnPlan plan;
    const int rc = attn_plan(a, &plan);
    if (rc != FA_PAGED_OK || plan.grid == 0) return rc;
    if (a->q == nullptr || a->out == nullptr || a->lens == nullptr || (a->table_width > 0 && a->block_table == nullptr))
        return FA_PAGED_ERR_NULL;
    if (plan.bytes > 0 && (workspace == nullptr || bytes < plan.bytes || !aligned16(workspace))) return FA_PAGED_ERR_WORKSPACE;
    DeviceGuard guard(a->device);
    if (guard.err != cudaSuccess) return cuda_failed();
    const FaPagedCache& c = a->cache;
    AttnParams p = {};
    p.q = static_cast<const uint16_t*>(a->q);
    p.out = static_cast<uint16_t*>(a->out);
    p.lse = a->lse;
    // (a cache without pages: nothing is read, but what is copied as zeros names an address)
    p.k = static_cast<const uint16_t*>(c.num_pages > 0 ? c.k : a->q);
    p.v = static_cast<const uint16_t*>(c.num_pages > 0 ? c.v : a->q);
    p.table = a->block_table;
    p.lens = a->lens;
    p.slopes = a->slopes;
    p.q_batch = a->q_batch_stride, p.q_head = a->q_head_stride, p.table_stride = a->table_stride;
    p.k_page = c.k_page_stride, p.k_head = c.k_head_stride, p.k_row = c.k_row_stride;
    p.v_page = c.v_page_stride, p.v_head = c.v_head_stride, p.v_row = c.v_row_stride;
    p.batch = a->batch, p.heads = a->heads, p.heads_k = c.heads_k, p.group = a->heads / c.heads_k;
    p.row_blocks = plan.row_blocks, p.width = a->table_width, p.page = page_size_of(c.page_size), p.num_pages = c.num_pages;
    p.window = a->window;
    const bool cap = a->softcap > 0.f;
    p.scale2 = a->scale * kLog2e;
    p.cap2 = a->softcap * kLog2e;
    p.inner = score_inner(a);
    p.cap_series = a->softcap > kSeriesCap;
    p.cluster = plan.cluster;
    p.cuts = static_cast<CutInfo*>(workspace);
    p.cuts_by_unit = plan.cuts < plan.grid;
    p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.cut_bytes);
    p.part_floats = plan.part_floats;
    const bool bf16 = a->dtype == FA_PAGED_BF16;
    if (c.head_dim == 128)
        return bf16 ? dispatch_attention<128, true>(p, plan, cap, a->device, stream)
                    : dispatch_attention<128, false>(p, plan, cap, a->device, stream);
    return bf16 ? dispatch_attention<64, true>(p, plan, cap, a->device, stream)
                : dispatch_attention<64, false>(p, plan, cap, a->device, stream);
}

static int rotary(const FaRotaryArgs* a, cudaStream_t stream) {
    if (a == nullptr) return FA_PAGED_ERR_NULL;
    if (a->struct_size != sizeof(FaRotaryArgs)) return FA_PAGED_ERR_ABI;
    int rc = check_device(a->device);
    if (rc != FA_PAGED_OK) return rc;
    if (a->dtype != FA_PAGED_FP16 && a->dtype != FA_PAGED_BF16) return FA_PAGED_ERR_DTYPE;
    if (a->batch < 0 || a->heads < 0 || a->heads_k < 0 || a->seqlen < 0 || a->position_batch_stride < 0)
        return FA_PAGED_ERR_SHAPE;
    if (a->head_dim != 64 && a->head_dim != 128) return FA_PAGED_ERR_HEAD_DIM;
    if (a->batch > FA_ROTARY_MAX_BATCH || static_cast<long long>(a->heads) + a->heads_k > (1 << 24)) return FA_PAGED_ERR_SHAPE;
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->q_out) || !aligned16(a->k_out) || !stride8(a->q_batch_stride) ||
        !stride8(a->q_head_stride) || !stride8(a->q_row_stride) || !stride8(a->k_batch_stride) || !stride8(a->k_head_stride) ||
        !stride8(a->k_row_stride))
        return FA_PAGED_ERR_ALIGN;
    rc = check_rotary(a->rotary, a->head_dim);
    const bool nothing = a->batch == 0 || a->seqlen == 0 || a->heads + a->heads_k == 0;
    if (rc != FA_PAGED_OK && !(nothing && rc == FA_PAGED_ERR_NULL)) return rc;
    if (nothing) return FA_PAGED_OK;
    if ((a->heads > 0 && (a->q == nullptr || a->q_out == nullptr)) ||
        (a->heads_k > 0 && (a->k == nullptr || a->k_out == nullptr)))
        return FA_PAGED_ERR_NULL;
    const int sms = sm_count(a->device);
    if (sms < 0) return sms;
    DeviceGuard guard(a->device);
    if (guard.err != cudaSuccess) return cuda_failed();
    RotaryParams p = {};
    fill_rotary(&p, a->rotary);
    const long long d = a->head_dim, plane = a->seqlen * d;
    p.rows[0] = Rows{static_cast<const uint16_t*>(a->q), static_cast<uint16_t*>(a->q_out), a->q_batch_stride,
                     a->q_head_stride, a->q_row_stride, a->heads * plane, plane, d, a->heads};
    p.rows[1] = Rows{static_cast<const uint16_t*>(a->k), static_cast<uint16_t*>(a->k_out), a->k_batch_stride,
                     a->k_head_stride, a->k_row_stride, a->heads_k * plane, plane, d, a->heads_k};
    p.position_outer = a->position_batch_stride;
    return launch_rotary(p, a->rotary.interleaved != 0, a->seqlen, a->batch, a->head_dim, a->dtype, sms, stream);
}

static int append(const FaPagedAppendArgs* a, cudaStream_t stream) {
    if (a == nullptr) return FA_PAGED_ERR_NULL;
    if (a->struct_size != sizeof(FaPagedAppendArgs)) return FA_PAGED_ERR_ABI;
    int rc = check_device(a->device);
    if (rc != FA_PAGED_OK) return rc;
    if (a->dtype != FA_PAGED_FP16 && a->dtype != FA_PAGED_BF16) return FA_PAGED_ERR_DTYPE;
    rc = check_cache(a->cache);
    if (rc != FA_PAGED_OK) return rc;
    if (a->num_tokens < 0 || a->num_tokens > INT_MAX || a->heads < 0 ||
        static_cast<long long>(a->heads) + 2LL * a->cache.heads_k > (1 << 24))
        return FA_PAGED_ERR_SHAPE;
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !stride8(a->q_token_stride) ||
        !stride8(a->q_head_stride) || !stride8(a->k_token_stride) || !stride8(a->k_head_stride) || !stride8(a->v_token_stride) ||
        !stride8(a->v_head_stride))
        return FA_PAGED_ERR_ALIGN;
    const bool turned = a->rotary.freqs != nullptr;
    if (turned) {
        rc = check_rotary(a->rotary, a->cache.head_dim);
        if (rc != FA_PAGED_OK && !(a->num_tokens == 0 && rc == FA_PAGED_ERR_NULL)) return rc;
    }
    if (a->num_tokens == 0) return FA_PAGED_OK;
    if (a->k == nullptr || a->v == nullptr || a->slots == nullptr || (a->heads > 0 && (a->q == nullptr || a->q_out == nullptr)))
        return FA_PAGED_ERR_NULL;
    const int sms = sm_count(a->device);
    if (sms < 0) return sms;
    DeviceGuard guard(a->device);
    if (guard.err != cudaSuccess) return cuda_failed();
    const FaPagedCache& c = a->cache;
    RotaryParams p = {};
    if (turned) fill_rotary(&p, a->rotary);
    const long long d = c.head_dim;
    p.rows[0] = Rows{static_cast<const uint16_t*>(a->q), static_cast<uint16_t*>(a->q_out), 0, a->q_head_stride,
                     a->q_token_stride, 0, d, a->heads * d, a->heads};
    p.rows[1] = Rows{static_cast<const uint16_t*>(a->k), static_cast<uint16_t*>(c.k), 0, a->k_head_stride,
                     a->k_token_stride, c.k_page_stride, c.k_head_stride, c.k_row_stride, c.heads_k};
    p.rows[2] = Rows{static_cast<const uint16_t*>(a->v), static_cast<uint16_t*>(c.v), 0, a->v_head_stride,
                     a->v_token_stride, c.v_page_stride, c.v_head_stride, c.v_row_stride, c.heads_k};
    p.slots = a->slots;
    p.slots_64 = a->slots_64 != 0;
    p.page_size = c.page_size;
    p.num_slots = static_cast<long long>(c.num_pages) * c.page_size;
    return launch_rotary(p, turned && a->rotary.interleaved != 0, a->num_tokens, 1, c.head_dim, a->dtype, sms, stream);
}

template <typename Args>
static int check_table(const Args* a) {
    if (a == nullptr) return FA_PAGED_ERR_NULL;
    if (a->struct_size != sizeof(Args)) return FA_PAGED_ERR_ABI;
    const int rc = check_device(a->device);
    if (rc != FA_PAGED_OK) return rc;
    if (a->batch < 0 || a->batch > FA_PAGED_MAX_REQUESTS || a->table_width < 0 || a->page_size <= 0 ||
        a->num_free_pages < 0 || a->table_stride < 0 ||
        static_cast<long long>(a->table_width) * a->page_size > INT_MAX)
        return FA_PAGED_ERR_SHAPE;
    if (a->free_head == nullptr || (a->batch > 0 && a->lens == nullptr) ||
        (a->batch > 0 && a->table_width > 0 && a->block_table == nullptr) ||
        (a->num_free_pages > 0 && a->free_pages == nullptr))
        return FA_PAGED_ERR_NULL;
    return FA_PAGED_OK;
}

static int extend(const FaPagedExtendArgs* a, cudaStream_t stream) {
    const int rc = check_table(a);
    if (rc != FA_PAGED_OK) return rc;
    if (a->num_tokens < 0 || a->num_tokens > INT_MAX) return FA_PAGED_ERR_SHAPE;
    if (a->cu == nullptr || a->head_out == nullptr || (a->batch > 0 && (a->new_lens == nullptr || a->lens_out == nullptr)) ||
        (a->num_tokens > 0 && (a->slots == nullptr || a->positions == nullptr)))
        return FA_PAGED_ERR_NULL;
    const int sms = sm_count(a->device);
    if (sms < 0) return sms;
    DeviceGuard guard(a->device);
    if (guard.err != cudaSuccess) return cuda_failed();
    static std::atomic<unsigned long long> done{0};
    const int most = (3 * FA_PAGED_MAX_REQUESTS + 1) * 4;
    const int ok = allow_smem(paged_extend_kernel, most, done, a->device);
    if (ok != FA_PAGED_OK) return ok;
    ExtendParams p = {};
    p.table = a->block_table, p.table_stride = a->table_stride, p.lens = a->lens, p.new_lens = a->new_lens;
    p.free_pages = a->free_pages, p.free_head = a->free_head, p.lens_out = a->lens_out, p.head_out = a->head_out;
    p.slots = reinterpret_cast<long long*>(a->slots), p.positions = a->positions, p.cu = a->cu;
    p.batch = a->batch, p.width = a->table_width, p.page = page_size_of(a->page_size), p.num_free = a->num_free_pages;
    p.num_tokens = a->num_tokens;
    const int ctas = a->num_tokens >= kTableTokens ? kTableCluster : 1;
    return launch_cluster(paged_extend_kernel, dim3(ctas), ctas > 1 ? kTableClusterThreads : kTableThreads, (3 * static_cast<size_t>(a->batch) + 1) * 4, ctas,
                          stream, p);
}

static int shrink(const FaPagedShrinkArgs* a, cudaStream_t stream) {
    const int rc = check_table(a);
    if (rc != FA_PAGED_OK) return rc;
    if (a->batch == 0) return FA_PAGED_OK;
    if (a->keep_lens == nullptr) return FA_PAGED_ERR_NULL;
    const int sms = sm_count(a->device);
    if (sms < 0) return sms;
    DeviceGuard guard(a->device);
    if (guard.err != cudaSuccess) return cuda_failed();
    static std::atomic<unsigned long long> done{0};
    const int ok = allow_smem(paged_shrink_kernel, 3 * FA_PAGED_MAX_REQUESTS * 4, done, a->device);
    if (ok != FA_PAGED_OK) return ok;
    ShrinkParams p = {};
    p.table = a->block_table, p.table_stride = a->table_stride, p.lens = a->lens, p.keep = a->keep_lens;
    p.free_pages = a->free_pages, p.free_head = a->free_head;
    p.batch = a->batch, p.width = a->table_width, p.page = page_size_of(a->page_size), p.num_free = a->num_free_pages;
    return launch_chained(paged_shrink_kernel, dim3(1), kTableThreads, 3 * static_cast<size_t>(a->batch) * 4, stream, p);
}

}  // namespace fa_paged

extern "C" {

int fa_paged_extend_sm100(const FaPagedExtendArgs* args, void* stream) {
    return fa_paged::extend(args, static_cast<cudaStream_t>(stream));
}

int fa_paged_shrink_sm100(const FaPagedShrinkArgs* args, void* stream) {
    return fa_paged::shrink(args, static_cast<cudaStream_t>(stream));
}

int fa_rotary_sm100(const FaRotaryArgs* args, void* stream) {
    return fa_paged::rotary(args, static_cast<cudaStream_t>(stream));
}

int fa_paged_append_sm100(const FaPagedAppendArgs* args, void* stream) {
    return fa_paged::append(args, static_cast<cudaStream_t>(stream));
}

int fa_paged_attention_sm100_workspace_bytes(const FaPagedAttentionArgs* args, size_t* bytes) {
    if (bytes == nullptr) return FA_PAGED_ERR_NULL;
    fa_paged::AttnPlan plan;
    const int rc = fa_paged::attn_plan(args, &plan);
    if (rc == FA_PAGED_OK) *bytes = plan.bytes;
    return rc;
}

int fa_paged_attention_sm100(const FaPagedAttentionArgs* args, void* workspace, size_t workspace_bytes, void* stream) {
    return fa_paged::attention(args, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int fa_paged_sm100_abi_version(void) { return FA_PAGED_ABI_VERSION; }

int fa_paged_sm100_launch_count(uint64_t* launches) {
    if (launches == nullptr) return FA_PAGED_ERR_NULL;
    *launches = fa_paged::g_launches.load();
    return FA_PAGED_OK;
}

const char* fa_paged_sm100_strerror(int code) {
    switch (code) {
        case FA_PAGED_OK: return "ok";
        case FA_PAGED_ERR_NULL: return "a required pointer is NULL";
        case FA_PAGED_ERR_DTYPE: return "q, k, v and the cache must be float16 or bfloat16, of one type";
        case FA_PAGED_ERR_SHAPE: return "bad shape: a size is negative or too large, or n_heads is not divisible by n_kv_heads";
        case FA_PAGED_ERR_HEAD_DIM: return "Only head_dim=64 or head_dim=128 is supported";
        case FA_PAGED_ERR_ALIGN: return "tensors must be 16-byte aligned, with strides that are multiples of 8 elements";
        case FA_PAGED_ERR_WORKSPACE: return "workspace missing, misaligned or too small";
        case FA_PAGED_ERR_ARCH: return "no kernel for this GPU: compute capability 10.x (sm_100a) required";
        case FA_PAGED_ERR_CUDA: return "a CUDA call failed";
        case FA_PAGED_ERR_ROTARY: return "rot_dim must be even, at least 2 and at most head_dim; mscale must be finite";
        case FA_PAGED_ERR_SCORE: return "scale, softcap and window must be finite and not negative";
        case FA_PAGED_ERR_ABI: return "struct_size does not match this library";
        default: return "unknown error";
    }
}

}  // extern "C"
