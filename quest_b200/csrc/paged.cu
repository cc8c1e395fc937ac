// Serving over a paged cache: page tables and slots from request lengths, pages given back, rotary embedding into the pages,
// and the check of drafted tokens.  The attention that reads the pages is in paged_attention.cu.
#include <cooperative_groups.h>

#include "common.cuh"

namespace qb {

namespace cg = cooperative_groups;

constexpr int kPageThreads = 512;
constexpr int kMaxRequests = 8192;  // of one step: two arrays of that length lie in shared memory (64 KB)
constexpr int kMaxEntries = 1 << 30;  // of what threads walk over in strides of a grid: an int index stays below 2^31

// Inclusive sum over the block; `carry` is the sum of all earlier rounds and is advanced.  scratch: one word per warp.
__device__ __forceinline__ long long block_inclusive_sum(long long v, long long& carry, long long* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPageThreads / 32; ++w) {
        const long long s = scratch[w];
        before += w < warp ? s : 0;
        all += s;
    }
    v += carry + before;
    carry += all;
    return v;
}

__device__ __forceinline__ int saturate_int(long long v) { return (int)(v > 0x7fffffffll ? 0x7fffffffll : v); }

// First index whose (non-decreasing) end lies behind i.
__device__ __forceinline__ int find_request(const int* ends, int n, int i) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > i) hi = mid; else lo = mid + 1;
    }
    return lo;
}

struct AssignParams {
    int* page_table;
    const int *free_pages, *free_count, *cached, *added;
    int *cu, *kv_lens, *lens, *free_left;
    long long* slots;
    int* positions;
    int batch, width, pool, rows, page;
};

// Page tables and slots of a step.  With c cached and n new tokens a request needs the pages ceil(c/P) .. ceil((c+n)/P) - 1;
// they are taken from the end of the free list in the order of the requests, so that a running sum of the needs says which
// request gets which entry and whether the list holds them.  Every block computes both running sums for itself (a few
// microseconds at most, no second launch and no block that waits for another) and then deals with its share of the rows; the
// first row of a page writes its entry into the table.  Latency: three dependent loads and two block sums (64 requests with a new
// token each 4.3 us, 512 with prompts of 30000 tokens in all 4.8 us, in a graph).
__global__ void __launch_bounds__(kPageThreads) page_assign_kernel(const AssignParams p) {
    extern __shared__ int sm[];
    int* ends = sm;              // rows up to and with the request
    int* first = sm + p.batch;   // its first place below the end of the free list, -1: refused
    __shared__ long long scratch[kPageThreads / 32];
    const int held = min(max(*p.free_count, 0), p.pool);
    long long row_carry = 0, page_carry = 0, used = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kPageThreads) {
        const int b = b0 + threadIdx.x;
        const bool there = b < p.batch;
        const long long c = there ? max(p.cached[b], 0) : 0, n = there ? max(p.added[b], 0) : 0;
        const long long end = block_inclusive_sum(n, row_carry, scratch);
        const long long have = (c + p.page - 1) / p.page, want = (c + n + p.page - 1) / p.page;
        const bool fits = end <= p.rows && want <= p.width;
        const long long need = there && fits ? want - have : 0;
        const long long taken = block_inclusive_sum(need, page_carry, scratch);
        const bool granted = fits && (need == 0 || taken <= held);
        if (there) {
            ends[b] = saturate_int(end);
            first[b] = granted ? (int)(taken - need) : -1;
            if (blockIdx.x == 0) {
                p.cu[b + 1] = (int)(end < p.rows ? end : p.rows);
                p.kv_lens[b] = granted ? (int)(c + n) : 0;
                p.lens[b] = (int)(granted ? c + n : c);
            }
        }
        if (granted && need > 0) used = taken;
    }
    if (blockIdx.x == 0) {
        __shared__ int most;
        if (threadIdx.x == 0) most = 0;
        __syncthreads();
        atomicMax(&most, (int)used);
        __syncthreads();
        if (threadIdx.x == 0) *p.free_left = held - most, p.cu[0] = 0;
    }
    __syncthreads();
    for (int i = blockIdx.x * kPageThreads + threadIdx.x; i < p.rows; i += gridDim.x * kPageThreads) {
        const int b = find_request(ends, p.batch, i);
        long long slot = -1;
        int pos = 0;
        if (b < p.batch && first[b] >= 0) {
            const int c = max(p.cached[b], 0), start = b == 0 ? 0 : ends[b - 1];
            pos = c + (i - start);
            const int at = pos / p.page, have = (int)(((long long)c + p.page - 1) / p.page);
            int* entry = p.page_table + (long long)b * p.width + at;
            int id;
            if (at >= have) {
                id = p.free_pages[held - 1 - (first[b] + at - have)];
                if (pos % p.page == 0) *entry = id;
            } else {
                id = *entry;
            }
            if (id >= 0) slot = (long long)id * p.page + pos % p.page;
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
    }
}

struct ReleaseParams {
    const int* page_table;
    int* free_pages;
    const int *free_count, *lens, *keep;
    int* free_left;
    int batch, width, pool, page;
};

// The pages behind the tokens that are kept go to the end of the free list, in the order of requests and pages: a running sum
// of the counts gives every page its place (1000 requests, 8000 pages back: 6.9 us).
__global__ void __launch_bounds__(kPageThreads) page_release_kernel(const ReleaseParams p) {
    extern __shared__ int sm[];
    int* ends = sm;              // pages given back up to and with the request
    int* stay = sm + p.batch;    // pages that it keeps
    __shared__ long long scratch[kPageThreads / 32];
    const int held = min(max(*p.free_count, 0), p.pool);
    long long carry = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kPageThreads) {
        const int b = b0 + threadIdx.x;
        const bool there = b < p.batch;
        const long long n = there ? max(p.lens[b], 0) : 0;
        const long long k = there ? min((long long)max(p.keep[b], 0), n) : 0;
        const long long have = min((n + p.page - 1) / p.page, (long long)p.width), left = min((k + p.page - 1) / p.page, (long long)p.width);
        const long long end = block_inclusive_sum(have - left, carry, scratch);
        if (there) ends[b] = saturate_int(end), stay[b] = (int)left;
    }
    __syncthreads();
    const int total = (int)min(carry, (long long)(p.pool - held));
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.free_left = held + total;
    for (int i = blockIdx.x * kPageThreads + threadIdx.x; i < total; i += gridDim.x * kPageThreads) {
        const int b = find_request(ends, p.batch, i);
        const int start = b == 0 ? 0 : ends[b - 1];
        p.free_pages[held + i] = p.page_table[(long long)b * p.width + stay[b] + (i - start)];
    }
}

struct AppendParams {
    const __nv_bfloat16* qkv;
    long long ld;
    const void* table;
    const int* positions;
    const long long* slots;
    __nv_bfloat16 *k, *v, *q_out;
    long long k_page, k_token, k_head, v_page, v_token, v_head;  // strides in elements
    long long capacity;                                          // slots of the cache
    int rows, hq, hkv, head_dim, table_len, page;
};

// One block per row: q and k are rotated (interleaved pairs, fp32 products and sums rounded one by one as torch rounds them,
// then to bf16 once), k and v go to the row's slot.  A row without a slot or a position outside the table leaves everything as
// it was.  Bound by HBM: every element is read and written once, in 16-byte pieces (16384 rows of 64 + 2 x 8 heads: 115 us,
// 5.8 TB/s of the 6.55 of a copy).
template <typename T>
__global__ void __launch_bounds__(256) rope_paged_append_kernel(const AppendParams p) {
    const int row = blockIdx.x;
    const long long slot = p.slots[row];
    const int pos = p.positions[row];
    if (slot < 0 || slot >= p.capacity || pos < 0 || pos >= p.table_len) return;
    const long long page = slot / p.page, token = slot - page * p.page;
    const int head_chunks = p.head_dim / 8, chunks = (p.hq + 2 * p.hkv) * head_chunks;
    const uint4* src = reinterpret_cast<const uint4*>(p.qkv + row * p.ld);
    for (int i = threadIdx.x; i < chunks; i += 256) {
        const uint4 x = ld_stream16(src + i);
        const int head = i / head_chunks, c = (i - head * head_chunks) * 8;
        __nv_bfloat16* dst;
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        if (head < p.hq + p.hkv) {
            const T* t = static_cast<const T*>(p.table) + (long long)pos * p.head_dim + c;
            float cs[8];
            if (sizeof(T) == 4) {
                const float4 a = __ldg(reinterpret_cast<const float4*>(t)), b = __ldg(reinterpret_cast<const float4*>(t) + 1);
                cs[0] = a.x; cs[1] = a.y; cs[2] = a.z; cs[3] = a.w; cs[4] = b.x; cs[5] = b.y; cs[6] = b.z; cs[7] = b.w;
            } else {
                const uint4 a = __ldg(reinterpret_cast<const uint4*>(t));
                const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) cs[2 * j] = bf16lo_to_f32(u[j]), cs[2 * j + 1] = bf16hi_to_f32(u[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x0 = bf16lo_to_f32(w[j]), x1 = bf16hi_to_f32(w[j]), c0 = cs[2 * j], s0 = cs[2 * j + 1];
                w[j] = pack_bf16x2(__fsub_rn(__fmul_rn(x0, c0), __fmul_rn(x1, s0)), __fadd_rn(__fmul_rn(x0, s0), __fmul_rn(x1, c0)));
            }
            dst = head < p.hq ? p.q_out + ((long long)row * p.hq + head) * p.head_dim
                              : p.k + page * p.k_page + token * p.k_token + (head - p.hq) * p.k_head;
        } else {
            dst = p.v + page * p.v_page + token * p.v_token + (head - p.hq - p.hkv) * p.v_head;
        }
        *reinterpret_cast<uint4*>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct VerifyParams {
    const void *target, *draft;
    const long long* tokens;
    const int* cu;
    const float* u;
    long long* out;
    int* accepted;
    int batch, n_tokens, vocab, most;
};

constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32, kSegment = 256, kMostCluster = 8;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// A draft's probability: what is negative counts as 0, a NaN stays one (no comparison holds for it, so its draft is refused and nothing
// is drawn in its place).
__device__ __forceinline__ float not_negative(float q) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(q), "f"(0.f));
    return r;
}

// Rows of probabilities, and the memory that they are part of.
template <typename T>
struct Rows {
    const T *row, *begin, *end;
};
// Eight neighbouring entries of a row as they are read, zeros behind its end.  A row that does not begin on 16 bytes (an odd
// vocabulary) is read in whole pieces all the same, one more of them, and shifted into place by values8; single entries are read where
// a piece would reach beyond the tensor or the row.  500 requests at a vocabulary of 50257 took 45 us when
// this was built, and 64 entry by entry (bf16; now 50, fp32 65).
template <typename T, bool VEC>
struct Raw8 {
    static constexpr int PIECES = (int)sizeof(T) / 2 + (VEC ? 0 : 1);
    uint4 w[PIECES];
    int shift;  // bytes
};
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T, VEC> read8(const Rows<T>& rows, int at, int vocab) {
    Raw8<T, VEC> r;
    const T* row = rows.row;
    if (VEC && at + 8 <= vocab) {
#pragma unroll
        for (int j = 0; j < r.PIECES; ++j) r.w[j] = ld_stream16(reinterpret_cast<const uint4*>(row + at) + j);
        return r;
    }
    if (!VEC && at + 8 <= vocab) {
        r.shift = (int)(reinterpret_cast<uintptr_t>(row + at) & 15u);
        const uint4* piece = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + at) - r.shift);
        if (piece >= reinterpret_cast<const uint4*>(rows.begin) && reinterpret_cast<const T*>(piece + r.PIECES) <= rows.end) {
#pragma unroll
            for (int j = 0; j < r.PIECES; ++j) r.w[j] = __ldg(piece + j);
            return r;
        }
    }
    r.shift = 0;
#pragma unroll
    for (int j = 0; j < r.PIECES; ++j) r.w[j] = make_uint4(0, 0, 0, 0);
    if (at >= vocab) return r;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = at + j < vocab ? as_float(row[at + j]) : 0;
    if (sizeof(T) == 4) {
        r.w[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        r.w[sizeof(T) / 2 - 1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
    } else {
        r.w[0] = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    }
    return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void values8(const Raw8<T, VEC>& r, float (&x)[8]) {
    constexpr int WORDS = 4 * Raw8<T, VEC>::PIECES, OWN = 2 * (int)sizeof(T);
    uint32_t w[WORDS];
#pragma unroll
    for (int j = 0; j < WORDS / 4; ++j) w[4 * j] = r.w[j].x, w[4 * j + 1] = r.w[j].y, w[4 * j + 2] = r.w[j].z, w[4 * j + 3] = r.w[j].w;
    if (!VEC) {
#pragma unroll
        for (int step = 2; step > 0; step >>= 1)  // by two words, by one
#pragma unroll
            for (int j = 0; j + step < WORDS; ++j) w[j] = r.shift & (4 * step) ? w[j + step] : w[j];
        if (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < OWN; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], r.shift & 2 ? 16 : 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = sizeof(T) == 4 ? __uint_as_float(w[j % OWN]) : j % 2 ? bf16hi_to_f32(w[j / 2]) : bf16lo_to_f32(w[j / 2]);
}

// The same of a draft's row: what is negative counts as 0, a NaN as more than any probability, so that nothing is left of the target's.
template <typename T, bool VEC>
__device__ __forceinline__ void draft8(Raw8<T, VEC> r, float (&q)[8]) {
    if (sizeof(T) == 2) {  // two at once
        uint32_t* const w = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
        for (int j = 0; j < 4 * r.PIECES; ++j) {
            asm("min.bf16x2 %0, %0, %1;" : "+r"(w[j]) : "r"(0x7f7f7f7fu));  // the largest finite value
            asm("max.bf16x2 %0, %0, %1;" : "+r"(w[j]) : "r"(0u));
        }
    }
    values8(r, q);
    if (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = fmaxf(fminf(q[j], 3e38f), 0.f);
    }
}

__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void of_pair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t sub_pair(uint64_t a, uint64_t b) {  // one rounding, as a subtraction
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(b), "l"(0xbf800000bf800000ull), "l"(a));
    return r;
}

// Sum of eight weights max(p - q, 0).  It decides between tokens, so it has to be as good as one in 64 bits, but 64-bit arithmetic
// per entry cost more than reading it: with m = max(p, q) the difference m - q is split into h, its nearest multiple of 2^-22, whose sums
// are exact in fp32 up to 4, and the rest (m - h) - q, below 2^-23, whose sums lose less than 2^-44; two conversions for eight entries.  (m - h
// is exact: both are multiples of m's last place, and h is no larger than m or, by less than that, the next multiple.  So what rounding the
// difference itself would lose, next to a much smaller q, is in the rest.)  What rests lose in all is far less than what u can
// tell apart; where the aim is as near to a border as that, the decision is made in 64 bits (near_border).
__device__ __forceinline__ double sum8(const float (&p)[8], const float (&q)[8]) {
    uint64_t high = 0, low = 0;
    const uint64_t magic = pair_of(3.f, 3.f);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const uint64_t m2 = pair_of(fmaxf(p[j], q[j]), fmaxf(p[j + 1], q[j + 1])), q2 = pair_of(q[j], q[j + 1]);  // a NaN of p counts as nothing
        const uint64_t h = sub_pair(add_pair(sub_pair(m2, q2), magic), magic);
        high = add_pair(high, h), low = add_pair(low, sub_pair(sub_pair(m2, h), q2));
    }
    float a, b, c, d;
    of_pair(high, a, b), of_pair(low, c, d);
    return (double)(a + b) + (double)(c + d);
}

// How far from a border the sums of sum8 may be off.  A group's rests add up to at most 2^-20, or to the row's total where that is less, and
// lose some 2^-25 of it in either direction: over the groups of a row about 2^-25 times the root of that times the total.  (Emulated on the
// host over 70000 rows of all kinds: at most 2^-26.9 times that root where the total is above 2^-14, 2^-23.6 below.)  Weights that are no
// probabilities may lose all that 24 bits can.  So 200 numbers at a vocabulary of 131072 come near a border in one call of 300, which then
// takes some 45 us more.
__device__ __forceinline__ double near_border(double total) {
    const float t = (float)total;
    return t > 2.f ? t * 0x1p-21f : t < 0x1p-14f ? t * 0x1p-22f : sqrtf(t) * 0x1p-34f;
}

// The difference of a target's row and a draft's (or nothing, or all on the token `hot`), as verify_drafts_kernel reads it.
template <typename T, bool VEC>
struct Weights {
    Rows<T> target, draft;
    bool minus_draft;
    long long hot;  // has no weight; -1: none
    int vocab;
    __device__ __forceinline__ void read(int at, Raw8<T, VEC>& a, Raw8<T, VEC>& c) const {
        a = read8<T, VEC>(target, at, vocab);
        if (minus_draft) c = read8<T, VEC>(draft, at, vocab);
    }
    __device__ __forceinline__ void unpack(const Raw8<T, VEC>& a, const Raw8<T, VEC>& c, int at, float (&x)[8], float (&q)[8]) const {
        values8(a, x);
        if (minus_draft) {
            draft8(c, q);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                q[j] = 0;
                if (at + j == hot) x[j] = 0;
            }
        }
    }
};
template <typename T, bool VEC>
__device__ __forceinline__ Weights<T, VEC> weights_of(const VerifyParams& p, int b, int c0, int kept, bool residual) {
    const T *targets = static_cast<const T*>(p.target), *drafted = static_cast<const T*>(p.draft);
    return Weights<T, VEC>{Rows<T>{targets + (long long)(c0 + b + kept) * p.vocab, targets, targets + (long long)(p.n_tokens + p.batch) * p.vocab},
                           Rows<T>{p.draft == nullptr ? nullptr : drafted + (long long)(c0 + kept) * p.vocab, drafted, drafted + (long long)p.n_tokens * p.vocab},
                           residual && p.draft != nullptr, residual && p.draft == nullptr ? p.tokens[c0 + kept] : -1, p.vocab};
}

struct VerifyShared {
    int refused, last, hit, fall, near;  // last: last entry of this block with a weight, -1: none
    double warp[kVerifyWarps], total;
};
// The entry of a warp's stretch whose running sum, from base on, passes the goal (hit; none: 0x7fffffff), the last one with a weight
// (fall), and whether the border in front of the entry or that behind it is as near to the goal as `near`.
template <bool LAST_WORD, typename T, bool VEC>
__device__ __forceinline__ void search_stretch(VerifyShared& sh, const Weights<T, VEC>& weights, int first, int end, double base, double goal, double near) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sh.hit = 0x7fffffff, sh.fall = -1, sh.near = 0;
    for (int s = first; s < end; s += kVerifyWarps) {
        float x[8], q[8];
        double v[8], sum = 0;
        const int at = (s + warp) * kSegment + lane * 8;
        Raw8<T, VEC> a, c;
        weights.read(s + warp < end ? at : weights.vocab, a, c);
        weights.unpack(a, c, at, x, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = (double)x[j] - (double)q[j];
            v[j] = v[j] > 0 ? v[j] : 0;
            sum += v[j];
        }
        double run = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(~0u, run, d);
            if (lane >= d) run += o;
        }
        __syncthreads();  // the round before has been read
        if (lane == 31) sh.warp[warp] = run;
        __syncthreads();
        double mine = base;
        for (int k = 0; k < kVerifyWarps; ++k) {
            if (k == warp) mine = base;
            base += sh.warp[k];
        }
        const double end_here = mine + run, before = __shfl_up_sync(~0u, end_here, 1), start_here = lane == 0 ? mine : before;
        int fall = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) fall = v[j] > 0 ? at + j : fall;
        // One lane's sums pass the goal, but for their rounding in 64 bits.  Then a border is near, and the search is not the last word;
        // where it is, the first of each warp's lanes that are behind the goal counts, and of those the first.
        bool passes = end_here > goal && fall >= 0;
        if (LAST_WORD) {
            const uint32_t all = __ballot_sync(~0u, passes);
            passes = passes && lane == __ffs(all) - 1;
        } else {
            passes = passes && start_here <= goal;
        }
        if (passes) {
            double r = start_here, from = r, to = end_here;
            int hit = fall;
            bool found = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double up = r + v[j];
                if (!found && up > goal) found = true, hit = at + j, from = r, to = up;
                r = up;
            }
            atomicMin(&sh.hit, hit);
            if ((from > 0 && fabs(goal - from) <= near) || to - goal <= near) sh.near = 1;
        }
        fall = __reduce_max_sync(~0u, fall);
        if (lane == 0 && fall >= 0) atomicMax(&sh.fall, fall);
    }
    __syncthreads();
}

// The token once more, with all sums in 64 bits, by one block: where a border is near.  Seldom called, and a function of its own that
// begins anew, so that it costs the kernel few registers and instructions (7 requests: 5.8 us without it, 6.2 like this, 7.1 with it inside; 200 at 131072: 27.9, 28.9 and 30.4).
template <typename T, bool VEC>
__device__ __noinline__ void draw_in_64_bits(const VerifyParams* params, VerifyShared* sh, int b, int c0, int kept, bool residual, float u, int stretches) {
    __shared__ double sums[kMostCluster * kVerifyWarps];
    const VerifyParams& p = *params;
    const Weights<T, VEC> weights = weights_of<T, VEC>(p, b, c0, kept, residual);
    const int lane = threadIdx.x & 31, segments = (p.vocab + kSegment - 1) / kSegment, share = (segments + stretches - 1) / stretches;
    constexpr int AHEAD = (VEC ? 8 : 4) / sizeof(T);
    for (int i = threadIdx.x >> 5; i < stretches; i += kVerifyWarps) {
        const int end = min((i + 1) * share, segments);
        double sum = 0;
        for (int s = i * share; s < end; s += AHEAD) {
            Raw8<T, VEC> a[AHEAD], c[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) weights.read(s + k < end ? (s + k) * kSegment + lane * 8 : p.vocab, a[k], c[k]);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                float x[8], q[8];
                weights.unpack(a[k], c[k], (s + k) * kSegment + lane * 8, x, q);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += fmax((double)x[j] - (double)q[j], 0.0);
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (lane == 0) sums[i] = sum;
    }
    __syncthreads();
    double total = 0, base = 0;
    for (int i = 0; i < stretches; ++i) total += sums[i];
    const double aim = fmax((double)u * total, 0.0);
    int i = 0;
    for (; i + 1 < stretches && !(base + sums[i] > aim); ++i) base += sums[i];
    search_stretch<true>(*sh, weights, i * share, min((i + 1) * share, segments), base, aim, -1);
    if (threadIdx.x == 0) p.out[(long long)b * (p.most + 1) + kept] = sh->hit != 0x7fffffff ? sh->hit : sh->fall;
}

// Rejection sampling against a draft, one cluster of blocks per request.  Draft i is kept while u_i q_i(x_i) < p_i(x_i);
// the next token is drawn from max(p - q, 0) of the first refused row, or from the row behind the last draft, by inverting the
// running sum at u times the total.  Every warp of the cluster sums a stretch of the vocabulary; the totals go round the cluster, and
// the block that holds the border reads the stretch of that warp again, a segment of 256 entries per warp.  So a row is read once;
// without clusters a request would have a single SM's bandwidth or a second launch.  The chain of reads (offsets, tokens, their
// probabilities, rows, the border) is what small calls wait for: seven requests at 32000 take 6.2 us; 200 at 131072, two rows of bf16
// for two thirds of them, 29.0 us, 3.1 TB/s, in fp32 37.9.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads, 3) verify_drafts_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ VerifyShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), b = blockIdx.x / blocks, rank = blockIdx.x % blocks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c0 = min(max(p.cu[b], 0), p.n_tokens), c1 = min(max(p.cu[b + 1], c0), p.n_tokens);
    const int drafts = min(c1 - c0, p.most);
    const T* target = static_cast<const T*>(p.target) + (long long)(c0 + b) * p.vocab;
    const T* draft = static_cast<const T*>(p.draft) + (p.draft == nullptr ? 0 : (long long)c0 * p.vocab);
    if (threadIdx.x == 0) sh.refused = drafts;
    __syncthreads();
    for (int i = threadIdx.x; i < drafts; i += kVerifyThreads) {
        const long long x = p.tokens[c0 + i];
        bool good = false;
        if (x >= 0 && x < p.vocab) {
            const double q = p.draft == nullptr ? 1.0 : (double)not_negative(as_float(draft[(long long)i * p.vocab + x]));
            good = (double)p.u[c0 + b + i] * q < (double)as_float(target[(long long)i * p.vocab + x]);
        }
        if (!good) atomicMin(&sh.refused, i);
    }
    __syncthreads();
    const int kept = sh.refused;
    const bool refused = kept < drafts;
    const int segments = (p.vocab + kSegment - 1) / kSegment;
    const int share = (segments + blocks * kVerifyWarps - 1) / (blocks * kVerifyWarps);  // of a warp
    const int seg0 = min((rank * kVerifyWarps + warp) * share, segments), seg1 = min(seg0 + share, segments);
    bool residual = refused;
    Weights<T, VEC> weights = weights_of<T, VEC>(p, b, c0, kept, refused);
    constexpr int AHEAD = (VEC ? 8 : 4) / sizeof(T);  // segments whose reads are under way at once
    double total = 0, before = 0;  // of all blocks, of those before this one
    int last = -1;
    while (true) {
        if (threadIdx.x == 0) sh.last = -1;
        __syncthreads();
        int mine = -1;
        double sum = 0;
        for (int s = seg0; s < seg1; s += AHEAD) {
            Raw8<T, VEC> a[AHEAD], c[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) weights.read(s + k < seg1 ? (s + k) * kSegment + lane * 8 : p.vocab, a[k], c[k]);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                float x[8], q[8];
                const int at = (s + k) * kSegment + lane * 8;
                weights.unpack(a[k], c[k], at, x, q);
                const double add = sum8(x, q);
                sum += add;
                if (add > 0) mine = at;
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        mine = __reduce_max_sync(~0u, mine);
        if (lane == 0) {
            sh.warp[warp] = sum;
            if (mine >= 0) atomicMax(&sh.last, mine);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0;
            for (int w = 0; w < kVerifyWarps; ++w) t += sh.warp[w];
            sh.total = t;
        }
        cluster.sync();
        total = before = 0;
        last = -1;
        for (int r = 0; r < blocks; ++r) {
            if (r == rank) before = total;
            total += *cluster.map_shared_rank(&sh.total, r);
            last = max(last, *cluster.map_shared_rank(&sh.last, r));
        }
        cluster.sync();  // nobody leaves or starts over while another block reads
        if (total > 0 || !residual) break;
        residual = weights.minus_draft = false, weights.hot = -1;  // a refused draft whose distribution covers the target's: the target's own row
    }

    const double aim = fmax((double)p.u[c1 + b] * total, 0.0);
    if (rank == 0) {
        for (int i = threadIdx.x; i <= p.most; i += kVerifyThreads)
            if (i != kept) p.out[(long long)b * (p.most + 1) + i] = i < kept ? p.tokens[c0 + i] : -1;
        if (threadIdx.x == 0) p.accepted[b] = kept;
    }
    long long* slot = p.out + (long long)b * (p.most + 1) + kept;
    // The block whose part holds the aim; where u rounds to one the one with the last weight, and without any weight the first.
    const bool beyond = !(aim < total);
    const int per_block = share * kVerifyWarps * kSegment;
    if (beyond ? rank != (last < 0 ? 0 : last / per_block) : !(before <= aim && aim < before + sh.total)) return;
    if (beyond && last < 0) {
        if (threadIdx.x == 0) *slot = 0;
        return;
    }
    // ---- the warp's stretch, then the segment, then the entry
    int stretch = last < 0 ? 0 : last / (share * kSegment);
    double base = 0, near = -1;
    if (!beyond) {
        stretch = rank * kVerifyWarps, base = before;
        for (int w = 0; w + 1 < kVerifyWarps && !(base + sh.warp[w] > aim); ++w) base += sh.warp[w], ++stretch;
        if (aim > 0) near = near_border(total);
    }
    search_stretch<false>(sh, weights, stretch * share, min((stretch + 1) * share, segments), base, aim, near);
    if (!beyond && (sh.near != 0 || sh.hit == 0x7fffffff)) {
        const float u = p.u[c1 + b];
        __syncthreads();  // all have read
        draw_in_64_bits<T, VEC>(&p, &sh, b, c0, kept, residual, u, blocks * kVerifyWarps);
        return;
    }
    // Where u rounds to one, behind the last weight: that weight.
    if (threadIdx.x == 0) *slot = !beyond ? sh.hit : sh.fall >= 0 ? sh.fall : last;
}

}  // namespace qb

using namespace qb;

// What a launch may have without asking, 48 KB, holds the kernel's static shared memory, too (150 bytes at most here), so large
// batches ask; always for the most that any batch needs, since host threads share the setting.
template <typename Kernel>
static int allow_smem(Kernel kernel, size_t bytes) {
    return bytes <= 32 * 1024 ? QB200_OK : cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kMaxRequests));
}

extern "C" int page_assign_cuda(int* page_table, const int* free_pages, const int* free_count, const int* cached_lens,
                                const int* new_lens, int* cu_new, int* kv_lens, int* lens, long long* slots, int* positions,
                                int* free_left, int batch, int width, int pool, int rows, int page_size, cudaStream_t stream) {
    if (batch < 0 || width < 0 || pool < 0 || rows < 0 || page_size <= 0) return QB200_ERR_INVALID_ARGUMENT;
    if (batch > kMaxRequests || (long long)width * page_size > 0x7fffffffll || rows > kMaxEntries) return QB200_ERR_UNSUPPORTED;
    if (!free_count || !cu_new || !free_left || (batch && (!cached_lens || !new_lens || !kv_lens || !lens)) || (rows && (!slots || !positions)) ||
        (batch && width && !page_table) || (pool && !free_pages))
        return QB200_ERR_INVALID_ARGUMENT;
    AssignParams p{page_table, free_pages, free_count, cached_lens, new_lens, cu_new, kv_lens, lens, free_left, slots, positions,
                   batch, width, pool, rows, page_size};
    const size_t smem = 8u * batch;
    const int st = allow_smem(page_assign_kernel, smem);
    if (st != QB200_OK) return st;
    const int blocks = (rows + kPageThreads - 1) / kPageThreads;
    page_assign_kernel<<<blocks < 1 ? 1 : blocks > 148 ? 148 : blocks, kPageThreads, smem, stream>>>(p);
    return launch_status();
}

extern "C" int page_release_cuda(const int* page_table, int* free_pages, const int* free_count, const int* lens,
                                 const int* keep_lens, int* free_left, int batch, int width, int pool, int page_size,
                                 cudaStream_t stream) {
    if (batch < 0 || width < 0 || pool < 0 || page_size <= 0) return QB200_ERR_INVALID_ARGUMENT;
    if (batch > kMaxRequests || pool > kMaxEntries) return QB200_ERR_UNSUPPORTED;
    if (!free_count || !free_left || (batch && (!lens || !keep_lens)) || (batch && width && !page_table) || (pool && !free_pages))
        return QB200_ERR_INVALID_ARGUMENT;
    ReleaseParams p{page_table, free_pages, free_count, lens, keep_lens, free_left, batch, width, pool, page_size};
    const size_t smem = 8u * batch;
    const int st = allow_smem(page_release_kernel, smem);
    if (st != QB200_OK) return st;
    const int blocks = pool / (8 * kPageThreads);  // a block has eight pages per thread where the whole pool comes back
    page_release_kernel<<<blocks < 1 ? 1 : blocks > 148 ? 148 : blocks, kPageThreads, smem, stream>>>(p);
    return launch_status();
}

extern "C" int rope_paged_append_cuda_bf16(const void* qkv, long long ld, const void* table, int table_is_bf16,
                                           const int* positions, const long long* slots, void* k_cache, const long long* k_strides,
                                           void* v_cache, const long long* v_strides, void* q_out, int rows, int n_head,
                                           int n_kv_head, int head_dim, int table_len, int num_pages, int page_size,
                                           cudaStream_t stream) {
    if (rows < 0 || n_head < 0 || n_kv_head < 0 || head_dim <= 0 || table_len < 0 || num_pages < 0 || page_size <= 0 ||
        ld < (long long)(n_head + 2ll * n_kv_head) * head_dim)
        return QB200_ERR_INVALID_ARGUMENT;
    if (rows == 0 || n_head + n_kv_head == 0 || num_pages == 0 || table_len == 0) return QB200_OK;
    if (!qkv || !table || !positions || !slots || (n_head && !q_out) || !k_strides || !v_strides || (n_kv_head && (!k_cache || !v_cache)))
        return QB200_ERR_INVALID_ARGUMENT;
    if (n_head + 2ll * n_kv_head > kMaxEntries / head_dim || head_dim % 8 != 0 || ld % 8 != 0 || !aligned16(qkv) || !aligned16(table) || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache))
        return QB200_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return QB200_ERR_UNSUPPORTED;
    AppendParams p{static_cast<const __nv_bfloat16*>(qkv), ld, table, positions, slots, static_cast<__nv_bfloat16*>(k_cache),
                   static_cast<__nv_bfloat16*>(v_cache), static_cast<__nv_bfloat16*>(q_out), k_strides[0], k_strides[1], k_strides[2],
                   v_strides[0], v_strides[1], v_strides[2], (long long)num_pages * page_size, rows, n_head, n_kv_head, head_dim,
                   table_len, page_size};
    if (table_is_bf16) rope_paged_append_kernel<__nv_bfloat16><<<rows, 256, 0, stream>>>(p);
    else rope_paged_append_kernel<float><<<rows, 256, 0, stream>>>(p);
    return launch_status();
}

template <typename T, bool VEC>
static int launch_verify(const VerifyParams& p, cudaStream_t stream) {
    // As many blocks per request as are at work at once (three per SM), eight at most: with more, the same chain of reads is waited
    // for in several rounds (64 requests at a vocabulary of 32000: 13.3 us with eight, 9.2 with four).
    int cluster = kMostCluster;
    while (cluster > 1 && (long long)p.batch * cluster > 3 * 148) cluster /= 2;
    const cudaError_t e = launch_kernel_cluster(false, cluster, verify_drafts_kernel<T, VEC>, (long long)p.batch * cluster, kVerifyThreads, 0, stream, p);
    const int st = launch_status();
    return e == cudaSuccess ? st : QB200_ERR_CUDA;
}

extern "C" int verify_drafts_cuda(const void* target_probs, const void* draft_probs, int probs_are_bf16, const long long* draft_tokens,
                                  const int* cu_drafts, const float* uniforms, long long* tokens, int* accepted, int batch,
                                  int n_drafts, int vocab, int max_drafts, cudaStream_t stream) {
    if (batch < 0 || n_drafts < 0 || vocab <= 0 || max_drafts < 0) return QB200_ERR_INVALID_ARGUMENT;
    if (batch == 0) return QB200_OK;
    if (!target_probs || !cu_drafts || !uniforms || !tokens || !accepted || (n_drafts && !draft_tokens)) return QB200_ERR_INVALID_ARGUMENT;
    if (vocab > (1 << 23) || batch > (1 << 27) || n_drafts > kMaxEntries || max_drafts > kMaxEntries) return QB200_ERR_UNSUPPORTED;
    VerifyParams p{target_probs, draft_probs, draft_tokens, cu_drafts, uniforms, tokens, accepted, batch, n_drafts, vocab, max_drafts};
    const bool vec = vocab % 8 == 0 && aligned16(target_probs) && aligned16(draft_probs);
    if (probs_are_bf16) return vec ? launch_verify<__nv_bfloat16, true>(p, stream) : launch_verify<__nv_bfloat16, false>(p, stream);
    return vec ? launch_verify<float, true>(p, stream) : launch_verify<float, false>(p, stream);
}
