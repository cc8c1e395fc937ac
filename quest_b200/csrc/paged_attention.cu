// Attention of new tokens over a paged cache: out = softmax(scale q k^T) v, causal, for any mixture of single tokens, drafted
// tokens and chunks of prompts in one launch (and a second, small one that joins what was split).
//
// The rows of a request and a key/value head are its new tokens times the query heads that share the head; a tile has 256 of
// them (two streams of 128), a step 128 keys:
//   S = Q K^T   tcgen05.mma kind::f16, M128 N128, Q and K in shared memory (128-byte swizzle), S in tensor memory
//   P = exp2(c S - c m), running maximum m and sum l per row in fp32: thread = row, four warps per stream
//   O += P V    tcgen05.mma with P (bf16, over its S) in tensor memory, V [keys][columns] in shared memory as it lies in the page
// While one stream's warps work on its scores the tensor core works for the other stream.  P is rounded to bf16 (2^-9 of itself,
// the weight of one key among many) because the second product takes 16-bit operands; O, m and l stay in fp32.  O is rescaled only
// when a row's maximum has grown by more than 2^8: until then P and l simply exceed one.
// Where a tile has at most 128 rows (decoding) both streams share its queries and take every second step; their sums meet in
// shared memory at the end.
//
// Work is cut by steps, not by rows: all steps of all (request, head, tile) items form one line, every block takes an equal
// piece of it, whatever the lengths are; each block computes the line from the lengths on the device.  An item that crosses
// from one block to the next leaves partial (O, m, l) in the workspace, and the second kernel joins the pieces in order, so
// results do not depend on timing.
#include <math_constants.h>

#include "tcgen05.cuh"

namespace qb {
namespace pa {

constexpr int BM = 128, BN = 128, TILE_ROWS = 2 * BM;
constexpr int kThreads = 384;
constexpr int kTmaWarp = 0, kMmaWarp = 1, kItemWarp = 2, kFirstSoftmax = 4;
constexpr int ITEMS = 4;            // descriptors in flight between the item warp and the other roles
constexpr int kItemReaders = 10;    // copy warp, MMA warp, eight softmax warps
constexpr int kControlRegs = 72, kSoftmaxRegs = 216;  // 128 x 72 + 256 x 216 = 384 x 168, what the block is launched with
static_assert(128 * kControlRegs + 256 * kSoftmaxRegs <= kThreads * 168, "register shares exceed the launch");

template <int D>
struct Cfg {
    static constexpr int Q_BYTES = BM * D * 2;
    static constexpr int STAGE_BYTES = BN * D * 2;
    static constexpr int STAGES = D == 128 ? 5 : 10;
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = BM * 128;
    static constexpr int NUM_BARS = 2 * STAGES + 8 + 2 * ITEMS + 9;
    static constexpr int SMEM = 1024 + 2 * Q_BYTES + STAGES * STAGE_BYTES + NUM_BARS * 8 + ITEMS * 64 + 2 * BM * 4 + 16;
    static_assert(SMEM + 256 <= 232448, "shared memory of an SM");
    // f32 accumulate, bf16 x bf16; S: both K-major, N = 128; O: the second operand lies with its columns together (MN-major)
    static constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BM >> 4) << 24);
    static constexpr uint32_t IDESC_S = IDESC | ((uint32_t)(BN >> 3) << 17);
    static constexpr uint32_t IDESC_O = IDESC | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    static constexpr uint32_t S_COL = 0, O_COL = 256;  // per stream: S (and P over it) 128 columns, O D columns
};

struct Params {
    __nv_bfloat16* out;
    const __nv_bfloat16* q;
    const int *page_table, *kv_lens, *cu;
    float* partial;   // per block two slots of slot_rows x (D + 2) floats
    int* headers;     // per block: the item that begins there and goes on in the next block
    long long o_token, o_head, q_token, q_head;
    float c;          // |scale| log2(e)
    uint32_t flip;    // sign bits of a negative scale, applied to q
    int rows, batch, width, hkv, group, num_pages, page, page_shift, slot_rows, min_steps;
};

// One item, or the piece of it that a block works on.
struct Item {
    int start, n, kv, b, hk;  // rows start .. start + n of the batch, kv keys
    int r0, rows;             // packed rows (token * group + head) r0 .. r0 + rows
    int t0, steps[2];         // first step, steps of each stream
    int single;               // one stream's worth of rows: both streams share them and alternate
    int slot;                 // -1: the whole item; else the slot of the partial result
    int last;                 // nothing behind this descriptor (it carries no work)
};
static_assert(sizeof(Item) <= 64, "descriptor");

constexpr int HEADER = 8;  // ints: pieces (0: none), start, hk, r0, rows

struct Request {
    int start, n, kv;
};
__device__ __forceinline__ Request request_of(const Params& p, int b) {
    const int lo = min(max(p.cu[b], 0), p.rows), hi = min(max(p.cu[b + 1], lo), p.rows);
    return {lo, hi - lo, min(max(p.kv_lens[b], 0), p.width * p.page)};
}
// Keys that packed row r of a request sees.
__device__ __forceinline__ int keys_of(const Request& q, int r, int group) { return min(max(q.kv - q.n + r / group + 1, 0), q.kv); }
// Steps of a row range that ends with row r; a range that sees nothing still takes one, which gives its zeros.
__device__ __forceinline__ int steps_of(int keys) { return max((keys + BN - 1) / BN, 1); }

// sum over i < n of floor((a i + b) / m), a, b >= 0 (the Euclidean descent on a and m)
__device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
    long long sum = 0;
    while (n > 0) {
        sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
        a %= m, b %= m;
        const long long y = a * n + b;
        n = y / m, b = y % m;
        const long long t = m;
        m = a, a = t;
        if (m == 0) break;
    }
    return sum;
}
// Steps of the first `tiles` tiles of a request and one head.  A full tile i ends with token floor((256 i + 255) / group), so
// it takes max(floor((256 i + 255 + (kv - n) group) / (128 group)), 0) + 1 steps; the last one ends with the last token.
__device__ __forceinline__ long long steps_before(const Request& q, int tiles, int group) {
    const int all = (int)(((long long)q.n * group + TILE_ROWS - 1) / TILE_ROWS);
    long long sum = 0;
    if (tiles == all && tiles > 0) sum += steps_of(q.kv), --tiles;
    if (tiles > 0) {
        const long long e = 255 + (long long)(q.kv - q.n) * group;
        const long long first = e >= 0 ? 0 : (-e + 255) / 256;
        sum += tiles;
        if (tiles > first) sum += floor_sum(tiles - first, 128ll * group, 256, e + 256 * first);
    }
    return sum;
}
__device__ __forceinline__ int tiles_of(const Request& q, int group) { return (int)(((long long)q.n * group + TILE_ROWS - 1) / TILE_ROWS); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// D[tmem] (+)= A[tmem] . B[smem], bf16 operands.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 128-byte swizzle, operand with its columns together: 64 columns by 8 rows per 1024 bytes, the next 64 columns `lead` bytes on.
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
          "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
          "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// mbar_wait of tcgen05.cuh without a call: behind one the compiler keeps to the registers of the launch.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, int where) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        const long long waited = clock64() - t0;
        if (waited > kWaitLimitFloor && waited > *reinterpret_cast<volatile long long*>(&g_wait_limit_cycles)) {
            atomicCAS(&g_device_status, 0, (where << 8) | QB200_ERR_DEVICE_TIMEOUT);
            return false;
        }
    }
}

// Weight of a partial result with maximum m (in log2 units) when the common maximum is `top`.
__device__ __forceinline__ float weight_to(float m, float top) { return m == -CUDART_INF_F ? 0.f : ex2(m - top); }

// What the softmax warps of a stream keep of an item: the reference maximum and the sum of the thread's row.
struct RowState {
    float m, l;  // m in units of the scores; -inf: nothing seen
};

// One step of a row: scores in tensor memory -> probabilities over them.  `seen` keys of this step are visible to the row.
template <int D>
__device__ __forceinline__ void softmax_step(RowState& st, const uint32_t s_addr, const uint32_t o_addr, const int seen, const bool first, const float c) {
    uint32_t s[4][32];
#pragma unroll
    for (int i = 0; i < 4; ++i) tmem_ld32(s_addr + 32 * i, s[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) tmem_ld_wait32(s[i]);
    if (__any_sync(~0u, seen < BN)) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
            if (i >= seen) s[i / 32][i % 32] = 0xff800000u;  // whatever stands there
    }
    float top = -CUDART_INF_F;
    {
        float t[4] = {top, top, top, top};
#pragma unroll
        for (int i = 0; i < 32; i += 2)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = fmaxf(fmaxf(t[j], __uint_as_float(s[j][i])), __uint_as_float(s[j][i + 1]));
        top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
    }
    top = fmaxf(top, st.m);
    // 2^8 of growth is harmless in fp32 sums and bf16 probabilities alike
    const bool grown = top * c > st.m * c + 8.f || (st.m == -CUDART_INF_F && top != -CUDART_INF_F);
    if (__any_sync(~0u, grown)) {
        const float a = st.m == -CUDART_INF_F ? 0.f : ex2((st.m - top) * c);
        st.m = top;
        st.l *= a;
        if (!first) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                uint32_t o[32];
                tmem_ld32(o_addr + 32 * i, o);
                tmem_ld_wait32(o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * a);
                tmem_st32(o_addr + 32 * i, o);
            }
        }
    }
    const float off = st.m == -CUDART_INF_F ? 0.f : -st.m * c;
    const uint64_t c2 = pack2(c, c), off2 = pack2(off, off);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int e = half * 64 + 2 * i;
            const uint64_t x = fma2(pack2(__uint_as_float(s[e / 32][e % 32]), __uint_as_float(s[e / 32][e % 32 + 1])), c2, off2);
            float x0, x1;
            unpack2(x, x0, x1);
            x0 = ex2(x0), x1 = ex2(x1);
            sum[i & 1] = add2(sum[i & 1], pack2(x0, x1));
            pk[i] = pack_bf16x2(x0, x1);
        }
        tmem_st32(s_addr + half * 32, pk);
    }
    float a, b;
    unpack2(add2(sum[0], sum[1]), a, b);
    st.l += a + b;
    tmem_st_wait();
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_kernel(const Params p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using C = Cfg<D>;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const gen = raw + (base - smem_u32(raw));
    const uint32_t q_smem = base, ring = base + 2 * C::Q_BYTES, bars = ring + C::STAGES * C::STAGE_BYTES;
    const uint32_t kv_full = bars, kv_empty = kv_full + 8 * C::STAGES, q_full = kv_empty + 8 * C::STAGES, s_full = q_full + 16, p_full = s_full + 16,
                   o_full = p_full + 16, item_full = o_full + 16, item_empty = item_full + 8 * ITEMS, merge_full = item_empty + 8 * ITEMS, merge_empty = merge_full + 32,
                   done = merge_empty + 32;
    Item* const items = reinterpret_cast<Item*>(gen + (bars + 8 * C::NUM_BARS - base));
    float* const merge_m = reinterpret_cast<float*>(items) + ITEMS * 16;
    float* const merge_l = merge_m + BM;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(merge_l + BM);
    __shared__ long long scan[kThreads / 32];
    __shared__ long long found_before;  // steps of all requests before the one in which this block's piece begins
    __shared__ int found;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    } else if (warp == kTmaWarp && lane == 0) {
        tma_prefetch_desc(&kmap), tma_prefetch_desc(&vmap);
        for (int i = 0; i < C::STAGES; ++i) mbar_init(kv_full + 8 * i, 1), mbar_init(kv_empty + 8 * i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(q_full + 8 * i, 4), mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, 4), mbar_init(o_full + 8 * i, 1);
        for (int i = 0; i < ITEMS; ++i) mbar_init(item_full + 8 * i, 1), mbar_init(item_empty + 8 * i, kItemReaders);
        for (int i = 0; i < 4; ++i) mbar_init(merge_full + 8 * i, 1), mbar_init(merge_empty + 8 * i, 1);
        mbar_init(done, 1);
        fence_barrier_init();
    }
    let_dependents_launch();  // the joining kernel, which waits for this one's end

    // ---- the line of steps: all requests' sums, and the request in which this block's piece begins
    long long total = 0, u0 = 0, u1 = 0, share = 0;
    if (threadIdx.x == 0) found = -1;
    for (int pass = 0; pass < 2; ++pass) {  // the total first, then the place
        long long carry = 0;
        for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
            const int b = b0 + threadIdx.x;
            long long mine = 0;
            if (b < p.batch) {
                const Request q = request_of(p, b);
                mine = steps_before(q, tiles_of(q, p.group), p.group) * p.hkv;
            }
            long long run = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const long long o = __shfl_up_sync(~0u, run, d);
                if (lane >= d) run += o;
            }
            __syncthreads();
            if (lane == 31) scan[warp] = run;
            __syncthreads();
            long long all = 0;
            for (int w = 0; w < kThreads / 32; ++w) {
                if (w < warp) run += scan[w];
                all += scan[w];
            }
            run += carry;
            carry += all;
            if (pass == 1 && u0 >= run - mine && u0 < run) found = b, found_before = run - mine;
        }
        if (pass == 0) {
            total = carry;
            share = (total + gridDim.x - 1) / gridDim.x;
            if (share < p.min_steps) share = p.min_steps;
            u0 = share * blockIdx.x, u1 = u0 + share < total ? u0 + share : total;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    int* const header = p.headers + blockIdx.x * HEADER;
    if (found < 0) {  // no step for this block (and none behind it)
        if (threadIdx.x == 0) header[0] = 0;
        __syncthreads();
        if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
        return;
    }

    bool ok = true;  // false: a wait has given up; every role leaves its loop, no role waits for another without a limit

    // The register limits stand at the head of the roles: where they cannot be told apart the compiler takes the lower one.
    if (warp >= kFirstSoftmax) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ------------------------------ softmax, results ------------------------------
        const int s = (warp - kFirstSoftmax) >> 2, quad = warp & 3, row = quad * 32 + lane;  // this thread's row of its stream
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + C::S_COL + 128 * s + lanes, o_addr = tmem + C::O_COL + D * s + lanes;
        uint32_t s_uses = 0, o_uses = 0, merges = 0;
        for (uint32_t it = 0;; ++it) {
            const uint32_t st = it % ITEMS;
            ok = __all_sync(~0u, ok && wait_bar(item_full + 8 * st, (it / ITEMS) & 1u, 78));
            const Item d = items[st];
            __syncwarp();
            if (lane == 0) mbar_arrive(item_empty + 8 * st);
            if (!ok || d.last) break;
            const int steps = d.steps[s];
            const int r = d.r0 + (d.single ? 0 : s * BM) + row;  // packed row of the request
            const bool live = r < d.r0 + d.rows;
            const int token = r / p.group, head = d.hk * p.group + (r - token * p.group);
            const int keys = live ? min(max(d.kv - d.n + token + 1, 0), d.kv) : d.kv;  // rows that are not there need no mask
            const bool warp_live = d.r0 + (d.single ? 0 : s * BM) + quad * 32 < d.r0 + d.rows;

            if (steps > 0 && !(d.single && s == 1)) {  // queries -> shared memory, two (four) rows per warp instruction
                const long long off = (long long)(d.start + token) * p.q_token + (long long)head * p.q_head;
                constexpr int LANES = D / 8, PER = 32 / LANES;
                if (warp_live) {
#pragma unroll 8
                    for (int i = 0; i < 32 / PER; ++i) {
                        const int from = i * PER + lane / LANES, piece = lane % LANES;
                        const long long o = __shfl_sync(~0u, off, from);
                        const bool there = __shfl_sync(~0u, live, from);
                        uint4 x = make_uint4(0, 0, 0, 0);
                        if (there) x = *reinterpret_cast<const uint4*>(p.q + o + piece * 8);
                        x.x ^= p.flip, x.y ^= p.flip, x.z ^= p.flip, x.w ^= p.flip;
                        const int rr = quad * 32 + from;
                        sts128(q_smem + s * C::Q_BYTES + (piece / 8) * C::HALF_BYTES + rr * 128 + (((piece % 8) ^ (rr & 7)) << 4), x);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full + 8 * s);
            }

            RowState rs{-CUDART_INF_F, 0.f};
            for (int i = 0; i < steps; ++i) {
                const int step = d.t0 + (d.single ? 2 * i + s : i);
                ok = __all_sync(~0u, ok && wait_bar(s_full + 8 * s, s_uses & 1u, 79));
                if (!ok) break;
                ++s_uses;
                tc_fence_after();
                if (warp_live) softmax_step<D>(rs, s_addr, o_addr, keys - step * BN, i == 0, p.c);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * s);
            }
            if (steps > 0) {
                ok = __all_sync(~0u, ok && wait_bar(o_full + 8 * s, o_uses & 1u, 80));
                ++o_uses;
                tc_fence_after();
            }
            if (!ok) break;
            float m = rs.m == -CUDART_INF_F ? -CUDART_INF_F : rs.m * p.c, l = rs.l;

            // Piece j of 16 bytes of this thread's row in the shared memory of a stream's queries (whose products are done): the
            // bytes of a row stay a row's, so a warp that goes on to the next item's queries disturbs no other.
            auto row_piece = [&](int tile, int rr, int j) {
                return q_smem + tile * C::Q_BYTES + (j / 8) * C::HALF_BYTES + rr * 128 + (((j % 8) ^ (rr & 7)) << 4);
            };
            if (d.single && d.steps[1] > 0 && warp_live) {
                // The streams' sums of the same rows: the second stream's come over half by half, through the second tile's place.
                if (s == 1) {
                    merge_m[row] = m, merge_l[row] = l;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
#pragma unroll 1
                        for (int c0 = 0; c0 < D / 2; c0 += 32) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + half * (D / 2) + c0, o);
                            tmem_ld_wait32(o);
#pragma unroll
                            for (int j = 0; j < 8; ++j) sts128(row_piece(1, row, c0 / 4 + j), make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]));
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(merge_full + 8 * quad);
                        ok = __all_sync(~0u, ok && wait_bar(merge_empty + 8 * quad, merges & 1u, 81));
                        ++merges;
                    }
                } else {
                    float wa = 0.f, wb = 0.f;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        ok = __all_sync(~0u, ok && wait_bar(merge_full + 8 * quad, merges & 1u, 82));
                        ++merges;
                        if (half == 0) {
                            const float m1 = merge_m[row], top = fmaxf(m, m1);
                            wa = weight_to(m, top), wb = weight_to(m1, top);
                            l = l * wa + merge_l[row] * wb;
                            m = top;
                        }
#pragma unroll 1
                        for (int c0 = 0; c0 < D / 2; c0 += 32) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + half * (D / 2) + c0, o);
                            tmem_ld_wait32(o);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint4 x = lds128(row_piece(1, row, c0 / 4 + j));
                                o[4 * j] = __float_as_uint(__uint_as_float(o[4 * j]) * wa + __uint_as_float(x.x) * wb);
                                o[4 * j + 1] = __float_as_uint(__uint_as_float(o[4 * j + 1]) * wa + __uint_as_float(x.y) * wb);
                                o[4 * j + 2] = __float_as_uint(__uint_as_float(o[4 * j + 2]) * wa + __uint_as_float(x.z) * wb);
                                o[4 * j + 3] = __float_as_uint(__uint_as_float(o[4 * j + 3]) * wa + __uint_as_float(x.w) * wb);
                            }
                            tmem_st32(o_addr + half * (D / 2) + c0, o);
                        }
                        tmem_st_wait();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(merge_empty + 8 * quad);
                    }
                }
                if (!ok) break;
            }
            if (d.single && s == 1) continue;

            const bool none = steps == 0;  // the upper stream's rows see nothing of this piece
            if (d.slot < 0) {
                // The row's columns, divided by the sum, go through the shared memory of the stream's queries so that whole lines are stored.
                if (warp_live) {
                    const float inv = 1.f / l;
                    const bool empty = l == 0.f;  // no key in sight: zeros
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c0, o);
                        tmem_ld_wait32(o);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                w[k] = pack_bf16x2(__uint_as_float(o[8 * j + 2 * k]) * inv, __uint_as_float(o[8 * j + 2 * k + 1]) * inv);
                            sts128(row_piece(s, row, c0 / 8 + j), empty ? make_uint4(0, 0, 0, 0) : make_uint4(w[0], w[1], w[2], w[3]));
                        }
                    }
                    __syncwarp();
                    const long long off = (long long)(d.start + token) * p.o_token + (long long)head * p.o_head;
                    constexpr int LANES = D / 8, PER = 32 / LANES;
#pragma unroll 4
                    for (int i = 0; i < 32 / PER; ++i) {
                        const int from = i * PER + lane / LANES, piece = lane % LANES;
                        const long long o = __shfl_sync(~0u, off, from);
                        const bool there = __shfl_sync(~0u, live, from);
                        const int rr = quad * 32 + from;
                        const uint4 x = lds128(row_piece(s, rr, piece));
                        if (there) *reinterpret_cast<uint4*>(p.out + o + piece * 8) = x;
                    }
                    __syncwarp();
                }
            } else if (warp_live) {
                float* const slot = p.partial + (long long)d.slot * p.slot_rows * (D + 2);
                const int at = (d.single ? 0 : s * BM) + row;
                if (at < p.slot_rows) {
                    slot[p.slot_rows * D + at] = none ? -CUDART_INF_F : m;
                    slot[p.slot_rows * (D + 1) + at] = none ? 0.f : l;
                }
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + c0, o);
                    tmem_ld_wait32(o);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float4 x = *reinterpret_cast<float4*>(&o[4 * j]);
                        if (none) x = make_float4(0, 0, 0, 0);
                        if (at < p.slot_rows) reinterpret_cast<float4*>(slot)[(c0 / 4 + j) * p.slot_rows + at] = x;
                    }
                }
            }
            tc_fence_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == kItemWarp) {
            // ------------------------------ items ------------------------------
            if (lane == 0) {
                int b = found;
                Request q = request_of(p, b);
                int tiles = tiles_of(q, p.group);
                const long long per_head = steps_before(q, tiles, p.group);
                long long rest = u0 - found_before;
                int hk = (int)(rest / per_head);
                rest -= hk * per_head;
                int lo = 0, hi = tiles - 1;  // the last tile that begins at or before the place
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (steps_before(q, mid, p.group) <= rest) lo = mid; else hi = mid - 1;
                }
                int tile = lo, t0 = (int)(rest - steps_before(q, tile, p.group));
                bool head_written = false;
                uint32_t it = 0;
                for (long long u = u0;; ++it) {
                    const uint32_t st = it % ITEMS;
                    ok = ok && wait_bar(item_empty + 8 * st, ((it / ITEMS) & 1u) ^ 1u, 70);
                    Item* d = items + st;
                    if (u >= u1) {
                        d->last = 1;
                        mbar_arrive(item_full + 8 * st);
                        break;
                    }
                    const int r0 = tile * TILE_ROWS, r_end = min(r0 + TILE_ROWS, q.n * p.group);
                    const int steps = steps_of(keys_of(q, r_end - 1, p.group));
                    const int t1 = (int)min((long long)steps, t0 + (u1 - u));
                    const bool ends = t1 == steps;
                    d->last = 0;
                    d->start = q.start, d->n = q.n, d->kv = q.kv, d->b = b, d->hk = hk, d->r0 = r0, d->rows = r_end - r0, d->t0 = t0;
                    d->single = r_end - r0 <= BM;
                    d->slot = t0 == 0 && ends ? -1 : 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0);
                    if (d->single) {
                        d->steps[0] = (t1 - t0 + 1) / 2, d->steps[1] = (t1 - t0) / 2;
                    } else {
                        const int first = steps_of(keys_of(q, r0 + BM - 1, p.group));  // the upper stream's rows see fewer keys
                        d->steps[0] = max(min(t1, first) - t0, 0), d->steps[1] = t1 - t0;
                    }
                    mbar_arrive(item_full + 8 * st);
                    if (t0 == 0 && !ends) {  // begins here and goes on: the pieces behind it lie one per block
                        const long long behind = u + steps - u1;
                        header[1] = q.start, header[2] = hk, header[3] = r0, header[4] = r_end - r0;
                        header[0] = 1 + (int)((behind + share - 1) / share);
                        head_written = true;
                    }
                    u += t1 - t0;
                    t0 = 0;
                    if (ends && ++tile == tiles) {
                        tile = 0;
                        if (++hk == p.hkv) {
                            hk = 0;
                            do {  // u < u1 says that one with rows follows
                                if (++b >= p.batch) break;
                                q = request_of(p, b);
                                tiles = tiles_of(q, p.group);
                            } while (tiles == 0);
                        }
                    }
                }
                if (!head_written) header[0] = 0;
            }
        } else if (warp == kTmaWarp) {
            // ------------------------------ pages -> ring ------------------------------
            uint32_t ring_it = 0;
            const int box_rows = min(p.page, BN), boxes = BN / box_rows;
            for (uint32_t it = 0;; ++it) {
                const uint32_t st = it % ITEMS;
                ok = __all_sync(~0u, ok && wait_bar(item_full + 8 * st, (it / ITEMS) & 1u, 71));
                const Item d = items[st];
                __syncwarp();
                if (lane == 0) mbar_arrive(item_empty + 8 * st);
                if (!ok || d.last) break;
                const int steps = d.single ? d.steps[0] + d.steps[1] : d.steps[1];
                const int* table = p.page_table + (long long)d.b * p.width;
                const int held = (d.kv + p.page - 1) >> p.page_shift;
                // Lane l copies box l / HALVES, columns 64 (l % HALVES).  Where a box holds no key of the request the page is one
                // behind the pool: zeros without a read.
                const int box = lane / C::HALVES, half = lane % C::HALVES;
                auto page_at = [&](int step) {
                    const int at = (step * BN + box * box_rows) >> p.page_shift;
                    int id = p.num_pages;
                    if (box < boxes && at < held) id = table[at];
                    return (unsigned)id < (unsigned)p.num_pages ? id : p.num_pages;
                };
                auto load = [&](const CUtensorMap* map, int step, int id) {
                    const uint32_t s = ring_it % C::STAGES, ph = (ring_it / C::STAGES) & 1u;
                    ok = __all_sync(~0u, ok && wait_bar(kv_empty + 8 * s, ph ^ 1u, 72));
                    if (!ok) return;
                    ++ring_it;
                    if (lane == 0) mbar_arrive_expect_tx(kv_full + 8 * s, C::STAGE_BYTES);
                    __syncwarp();
                    if (box < boxes)
                        tma_load_4d(ring + s * C::STAGE_BYTES + half * C::HALF_BYTES + box * box_rows * 128, map, half * 64,
                                    (step * BN + box * box_rows) & (p.page - 1), d.hk, id, kv_full + 8 * s);
                };
                // keys run one step ahead of the values, two where the streams alternate
                const int lead = d.single ? 2 : 1;
                int ids[3] = {page_at(d.t0), steps > 1 ? page_at(d.t0 + 1) : 0, 0};
                load(&kmap, d.t0, ids[0]);
                if (lead == 2 && steps > 1) load(&kmap, d.t0 + 1, ids[1]);
                for (int i = 0; i < steps; ++i) {
                    if (i + 2 < steps) ids[2] = page_at(d.t0 + i + 2);
                    if (lead == 1 && i + 1 < steps) load(&kmap, d.t0 + i + 1, ids[1]);
                    load(&vmap, d.t0 + i, ids[0]);
                    if (lead == 2 && i + 2 < steps) load(&kmap, d.t0 + i + 2, ids[2]);
                    ids[0] = ids[1], ids[1] = ids[2];
                }
            }
            const uint32_t pending = ring_it < (uint32_t)C::STAGES ? ring_it : (uint32_t)C::STAGES;
            if (!ok)
                for (uint32_t j = 0; j < pending; ++j) {  // copies under way still land
                    const uint32_t i2 = ring_it - 1 - j;
                    wait_bar(kv_full + 8 * (i2 % C::STAGES), (i2 / C::STAGES) & 1u, 73);
                }
        } else if (warp == kMmaWarp) {
            // ------------------------------ matrix products ------------------------------
            uint32_t ring_it = 0, q_uses[2] = {0, 0}, p_uses[2] = {0, 0};
            auto stage = [&](uint32_t i) { return ring + (i % C::STAGES) * C::STAGE_BYTES; };
            auto wait_stage = [&](uint32_t i) { ok = __all_sync(~0u, ok && wait_bar(kv_full + 8 * (i % C::STAGES), (i / C::STAGES) & 1u, 74)); };
            auto free_stage = [&](uint32_t i) {
                if (ok && elect_one()) umma_commit(kv_empty + 8 * (i % C::STAGES));
                __syncwarp();
            };
            auto wait_q = [&](int s) {
                ok = __all_sync(~0u, ok && wait_bar(q_full + 8 * s, q_uses[s] & 1u, 75));
                ++q_uses[s];
            };
            auto wait_p = [&](int s) {
                ok = __all_sync(~0u, ok && wait_bar(p_full + 8 * s, p_uses[s] & 1u, 76));
                ++p_uses[s];
                tc_fence_after();
            };
            auto scores = [&](int s, int q_tile, uint32_t k_it) {  // S_s = Q K^T
                if (ok && elect_one()) {
                    const uint64_t a = make_smem_desc(q_smem + q_tile * C::Q_BYTES), b = make_smem_desc(stage(k_it));
    #pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t o = (k / 4) * (C::HALF_BYTES >> 4) + (k % 4) * 2;
                        umma_bf16(tmem + C::S_COL + 128 * s, a + o, b + o, C::IDESC_S, k > 0);
                    }
                    umma_commit(s_full + 8 * s);
                }
                __syncwarp();
            };
            auto values = [&](int s, uint32_t v_it, bool accumulate, bool end) {  // O_s += P V
                if (ok && elect_one()) {
                    const uint64_t b = make_mn_desc(stage(v_it), C::HALF_BYTES);
    #pragma unroll
                    for (int k = 0; k < BN / 16; ++k)
                        umma_bf16_ts(tmem + C::O_COL + D * s, tmem + C::S_COL + 128 * s + 8 * k, b + k * (2048 >> 4), C::IDESC_O, accumulate || k > 0);
                    if (end) umma_commit(o_full + 8 * s);
                }
                __syncwarp();
            };
            for (uint32_t it = 0;; ++it) {
                const uint32_t st = it % ITEMS;
                ok = __all_sync(~0u, ok && wait_bar(item_full + 8 * st, (it / ITEMS) & 1u, 77));
                const Item d = items[st];
                __syncwarp();
                if (lane == 0) mbar_arrive(item_empty + 8 * st);
                if (!ok || d.last) break;
                // Rows of the last page behind the request's tokens hold anything; a zero weight does not make a NaN harmless.
                auto clean = [&](uint32_t v_it, int step) {
                    const int live = d.kv - step * BN;
                    if (live >= BN) return;
                    const int from = max(live, 0), to = min(((from + p.page - 1) >> p.page_shift) << p.page_shift, BN);
                    if (from == to) return;
                    for (int i = from * C::HALVES * 8 + lane; i < to * C::HALVES * 8; i += 32) {
                        const int row = i / (C::HALVES * 8), piece = i % (C::HALVES * 8);
                        sts128(stage(v_it) + (piece / 8) * C::HALF_BYTES + row * 128 + (piece % 8) * 16, make_uint4(0, 0, 0, 0));
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                };
                if (d.single) {
                    const int n = d.steps[0] + d.steps[1];
                    wait_q(0);
                    for (int i = 0; i < 2 && i < n; ++i) {
                        wait_stage(ring_it);
                        scores(i, 0, ring_it);
                        free_stage(ring_it++);
                    }
                    for (int i = 0; i < n; ++i) {
                        const int s = i & 1;
                        wait_stage(ring_it);
                        clean(ring_it, d.t0 + i);
                        wait_p(s);
                        values(s, ring_it, i > 1, i + 2 >= n);
                        free_stage(ring_it++);
                        if (i + 2 < n) {
                            wait_stage(ring_it);
                            scores(s, 0, ring_it);
                            free_stage(ring_it++);
                        }
                    }
                } else {
                    const int n0 = d.steps[0], n1 = d.steps[1];
                    wait_stage(ring_it);
                    if (n0 > 0) {
                        wait_q(0);
                        scores(0, 0, ring_it);
                    }
                    wait_q(1);
                    scores(1, 1, ring_it);
                    free_stage(ring_it++);
                    for (int i = 0; i < n1; ++i) {
                        // next keys at ring_it, these values behind them
                        const bool more = i + 1 < n1;
                        const uint32_t k_it = ring_it, v_it = ring_it + (more ? 1 : 0);
                        ring_it = v_it + 1;
                        if (more) wait_stage(k_it);
                        wait_stage(v_it);
                        clean(v_it, d.t0 + i);
                        if (i < n0) {
                            wait_p(0);
                            values(0, v_it, i > 0, i + 1 == n0);
                            if (i + 1 < n0) scores(0, 0, k_it);
                        }
                        wait_p(1);
                        values(1, v_it, i > 0, !more);
                        free_stage(v_it);
                        if (more) {
                            scores(1, 1, k_it);
                            free_stage(k_it);
                        }
                    }
                }
            }
            // Every product has ended and every arrival that it owes has been made before the block's memory goes.
            if (elect_one()) umma_commit(done);
            __syncwarp();
            wait_bar(done, 0, 83);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the pieces of the item that begins in block x of the first kernel, 32 rows of it per block.
template <int D>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const Params p) {
    wait_for_preceding_grid();
    const int* header = p.headers + blockIdx.x * HEADER;
    const int pieces = header[0], start = header[1], hk = header[2], r0 = header[3], rows = header[4];
    const int row = blockIdx.y * 32 + (threadIdx.x & 31);
    if (pieces == 0 || row >= rows) return;
    const long long slot_floats = (long long)p.slot_rows * (D + 2);
    auto slot_of = [&](int i) { return p.partial + (2ll * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * slot_floats; };
    float top = -CUDART_INF_F;
    for (int i = 0; i < pieces; ++i) top = fmaxf(top, slot_of(i)[p.slot_rows * D + row]);
    constexpr int PER = D / 4 / 8;  // 16-byte pieces of the row per thread
    float l = 0;
    float4 o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = make_float4(0, 0, 0, 0);
    for (int i = 0; i < pieces; ++i) {
        const float* slot = slot_of(i);
        const float w = weight_to(slot[p.slot_rows * D + row], top);
        l += w * slot[p.slot_rows * (D + 1) + row];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float4 x = reinterpret_cast<const float4*>(slot)[((threadIdx.x >> 5) * PER + j) * p.slot_rows + row];
            o[j].x += w * x.x, o[j].y += w * x.y, o[j].z += w * x.z, o[j].w += w * x.w;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int r = r0 + row, token = r / p.group, head = hk * p.group + (r - token * p.group);
    __nv_bfloat16* out = p.out + (start + token) * p.o_token + head * p.o_head + (threadIdx.x >> 5) * PER * 4;
#pragma unroll
    for (int j = 0; j < PER; ++j)
        *reinterpret_cast<uint2*>(out + 4 * j) = make_uint2(pack_bf16x2(o[j].x * inv, o[j].y * inv), pack_bf16x2(o[j].z * inv, o[j].w * inv));
}

constexpr int kMaxDevices = 64;
static int current_device() {
    int dev = -1;
    return cudaGetDevice(&dev) == cudaSuccess && dev < kMaxDevices ? dev : -1;
}

// The number of SMs of the current device, 0 on an error.
static int sm_count() {
    static int counts[kMaxDevices];
    const int dev = current_device();
    if (dev < 0) return 0;
    if (counts[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        counts[dev] = n;
    }
    return counts[dev];
}

// Rows of a partial result: a tile's, or what the whole call has of one head where that is less.
static int slot_rows_of(int rows, int group) {
    const long long all = ((long long)rows * group + 31) / 32 * 32;
    return (int)(all < TILE_ROWS ? all : TILE_ROWS);
}

static int encode_page_map(CUtensorMap* map, const void* base, const long long* strides, int num_pages, int page, int heads, int D) {
    EncodeTiledFn fn = get_encode_fn();
    if (fn == nullptr) return QB200_ERR_DRIVER;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)num_pages};
    // the stride of a dimension of one entry is never used, but has to be a valid one
    const cuuint64_t st[3] = {(cuuint64_t)strides[1] * 2, (cuuint64_t)(heads > 1 ? strides[2] : D) * 2, (cuuint64_t)(num_pages > 1 ? strides[0] : D) * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page < BN ? page : BN), 1, 1}, unit[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, st, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? QB200_OK : QB200_ERR_DRIVER;
}

template <int D>
static int launch(Params p, const CUtensorMap& kmap, const CUtensorMap& vmap, int blocks, cudaStream_t stream) {
    static bool prepared[kMaxDevices];  // of the device, once; a second thread that does it again does no harm
    const int dev = current_device();
    if (dev < 0) return QB200_ERR_CUDA;
    if (!prepared[dev]) {
        if (cudaFuncSetAttribute(paged_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM) != cudaSuccess) return QB200_ERR_CUDA;
        prepared[dev] = true;
    }
    paged_attention_kernel<D><<<blocks, kThreads, Cfg<D>::SMEM, stream>>>(p, kmap, vmap);
    const int st = launch_status();
    if (st != QB200_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, (p.slot_rows + 31) / 32);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<D>, p));
}

}  // namespace pa

int paged_attention_fetch_and_clear_device_status(int* out) { return fetch_and_clear_device_status(out); }

}  // namespace qb

using namespace qb;

extern "C" int paged_attention_workspace(int rows, int batch, int n_head, int n_kv_head, int head_dim) {
    if (rows <= 0 || batch <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || head_dim > 128) return 0;
    const long long sms = pa::sm_count();
    return (int)(sms * (2ll * pa::slot_rows_of(rows, n_head / n_kv_head) * (head_dim + 2) * 4 + pa::HEADER * 4));
}

extern "C" int paged_attention_cuda_bf16(void* out, const long long* out_strides, const void* q, const long long* q_strides,
                                         const void* k_cache, const long long* k_strides, const void* v_cache,
                                         const long long* v_strides, const int* page_table, const int* kv_lens, const int* cu_new,
                                         void* workspace, float scale, int rows, int batch, int width, int n_head, int n_kv_head,
                                         int head_dim, int num_pages, int page_size, cudaStream_t stream) {
    if (rows < 0 || batch < 0 || width < 0 || n_head <= 0 || n_kv_head <= 0 || num_pages < 0 || page_size <= 0) return QB200_ERR_INVALID_ARGUMENT;
    if (rows == 0 || batch == 0) return QB200_OK;
    if (!out || !out_strides || !q || !q_strides || !k_strides || !v_strides || !kv_lens || !cu_new || !workspace || (width && !page_table) ||
        !k_cache || !v_cache || num_pages == 0)
        return QB200_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || n_head % n_kv_head != 0 || (page_size & (page_size - 1)) != 0 || page_size < 16 || page_size > 1024 ||
        !aligned16(out) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
        return QB200_ERR_UNSUPPORTED;
    const int group = n_head / n_kv_head;
    if ((long long)rows * group > (1ll << 30) || (long long)width * page_size * group > 0x7fffffffll) return QB200_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (k_strides[i] % 8 || v_strides[i] % 8 || (i < 2 && (q_strides[i] % 8 || out_strides[i] % 8))) return QB200_ERR_UNSUPPORTED;
    const int sms = pa::sm_count();
    if (sms == 0) return QB200_ERR_CUDA;
    CUtensorMap kmap, vmap;
    int st = pa::encode_page_map(&kmap, k_cache, k_strides, num_pages, page_size, n_kv_head, head_dim);
    if (st == QB200_OK) st = pa::encode_page_map(&vmap, v_cache, v_strides, num_pages, page_size, n_kv_head, head_dim);
    if (st != QB200_OK) return st;
    pa::Params p{};
    p.out = static_cast<__nv_bfloat16*>(out);
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.page_table = page_table, p.kv_lens = kv_lens, p.cu = cu_new;
    p.slot_rows = pa::slot_rows_of(rows, group);
    p.partial = static_cast<float*>(workspace);
    p.headers = reinterpret_cast<int*>(p.partial + sms * 2ll * p.slot_rows * (head_dim + 2));
    p.o_token = out_strides[0], p.o_head = out_strides[1], p.q_token = q_strides[0], p.q_head = q_strides[1];
    p.flip = scale < 0 ? 0x80008000u : 0u;
    p.c = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.17549435e-38f);  // above zero: what is masked stays at minus infinity
    p.rows = rows, p.batch = batch, p.width = width, p.hkv = n_kv_head, p.group = group, p.num_pages = num_pages, p.page = page_size;
    for (p.page_shift = 0; (1 << p.page_shift) < page_size; ++p.page_shift) {}
    p.min_steps = 1;
    return head_dim == 64 ? pa::launch<64>(p, kmap, vmap, sms, stream) : pa::launch<128>(p, kmap, vmap, sms, stream);
}
