// Attention of new tokens over a paged cache: out = softmax(scale q k^T) v, causal, for any mixture of single tokens, drafted
// tokens and chunks of prompts in one launch (and a second, small one that joins what was split).
//
// The rows of a request and a key/value head are its new tokens times the query heads that share the head; a stream works on 128 of
// them, a step has 128 keys:
//   S = Q K^T   tcgen05.mma kind::f16, M128 N128, Q and K in shared memory (128-byte swizzle), S in tensor memory
//   P = exp2(c S - c m), running maximum m and sum l per row in fp32: thread = row, four warps per stream
//   O += P V    tcgen05.mma with P (bf16, over its S) in tensor memory, V [keys][columns] in shared memory as it lies in the page
// P is rounded to bf16 (at most 2^-8 of itself, and it is the weight of one key among many) because the second product takes 16-bit
// operands; O, m and l stay in fp32.  O is rescaled only when a row's weights have grown far beyond one; until then P and l simply
// exceed it.
// A tile has whole tokens: 128 / group of them per stream.  The two streams of a block work in one of two ways.  As a pair they share
// the keys and values of one tile of 256 rows, and while one stream's warps work on its scores the tensor core works for the
// other.  Alone (tiles of at most 128 rows: decoding, the ends of chunks) each stream has tiles of its own, with half of the
// shared memory, an issuing warp and a copying warp of its own: such work is bound by HBM, and what an item costs besides its
// steps (its queries, its result) disappears behind the other stream.
//
// Work is cut by steps, not by tiles: the steps of all pair items form one line, those of all single items another; every block
// takes an equal piece of the first (cut at an item's edge where one is near), then each of its streams an equal piece of the second,
// whatever the lengths are.  Each block computes its places in the lines from the lengths on the device.  An item that crosses from
// one piece to the next leaves partial (O, m, l) in the workspace, and a second kernel joins them in order, so results do not depend on
// timing.
//
// Measured in a graph (copy 6.55 TB/s, matrix product 1655 TFLOP/s, 1408 sustained; heads of 128; a range ends with what the power
// limit leaves when the calls go on for long):
//   64 requests of up to 16384 tokens (137000 in all), 64 / 8 heads, one new token   100 - 112 us, 5.0 - 5.6 TB/s; of that 9 us until
//                                                the first product, 85 - 90 at the rate of HBM, 6 for the join
//   one request of 1001 tokens, 16 / 16 heads, one new token    13 us, nearly all of it the chain of latencies
//   one request of 32768 tokens, 64 / 8 heads, one new token    38 us, 3.5 TB/s
//   the same with 8 / 1 heads                                  23 us, 0.7 TB/s: a chain of latencies, the join among them
//   128 requests of at most 1000 tokens, 32 / 32 heads          116 - 130 us, 3.9 - 4.3 TB/s
//   16 prompts of 1024, 16 / 16 heads                           107 - 120 us; tensor pipe and exponentials a third each
//   4 prompts of 4096, 32 / 8 heads                             471 - 535 us, 1167 - 1028 TFLOP/s; head_dim 64 410 us
//   a chunk of 4096 behind 28672 tokens, among 15 single tokens, 64 / 8 heads    3.10 - 3.88 ms, 1330 - 1060 TFLOP/s
// A step of 128 rows by 128 keys costs the tensor core 2 x 8 products of 64 cycles and its warps 128 exponentials per thread, 16 a
// cycle and SM: 1024 cycles each.  A stream's steps form a chain, 1900 cycles of softmax and 1330 of products and their hand-over; two
// streams keep the tensor core busy two thirds of that.
// Other splits that were built: an issuing warp per stream for pairs 4.2 ms for the chunk (3.45 then); keys as the rows of S for tiles of
// at most 32 rows 12.3 us for one request, but 118 for the 64 (110 then); the result through shared memory 146 us for the 16 prompts (134
// then), or with four lanes to a row of it 117 (108 then).
#include <math_constants.h>

#include "tcgen05.cuh"

namespace qb {
namespace pa {

constexpr int BM = 128, BN = 128, HN = BN / 2;  // rows of a stream, keys of a step, keys of a slot
constexpr int kThreads = 384;
constexpr int kCopyWarp0 = 0, kMmaWarp0 = 1, kMmaWarp1 = 2, kCopyWarp1 = 3, kFirstSoftmax = 4;
constexpr int ITEMS = 4;                            // descriptors in flight on each list
constexpr int kControlRegs = 96, kSoftmaxRegs = 200;  // 128 x 96 + 256 x 200 is what the block is launched with, 384 x 168, or less
static_assert(128 * kControlRegs + 256 * kSoftmaxRegs <= kThreads * 168, "register shares exceed the launch");
// Steps that an item's queries and result are worth in the lines, and how near to an item's edge a pair's line is cut there and not in
// the item (4 prompts of 4096: 500 us with one step for a pair, 471 with two, 481 with three; 16 of at most 200: 29 us with two
// and every cut where it falls, 23 like this.  Single items: 128 requests of 1000 tokens 115 us with one step, 129 with two; cuts
// moved by up to two places leave 5 drafts for 32 requests at 38 us in place of 34.5).
constexpr int kPairCost = 2, kPairNear = 1, kSingleCost = 1;
// Steps of an item from which a stream's piece of the line has three places at least (two from a quarter of that), and a pair's eight,
// however few requests there are: pieces have to be joined, too (single items of 256 steps: 28.4 us with one, 23.8 with two, 23.0 with
// three, 23.6 with four; 70: 23.1, 19.6, 20.3; 32: 17.2, 16.6, 20.0; 16: 15.1 with one, 16.5 with two.  64 tokens behind 32704, 8 / 1
// heads, two pairs of 256 steps: 57 us at four, 44 at eight, 37 with the join's reads of four pieces at once).
constexpr int kLongItem = 128;

template <int D>
struct Cfg {
    static constexpr int Q_BYTES = BM * D * 2;
    static constexpr int SLOT_BYTES = HN * D * 2;         // the ring of a single stream has slots of 64 keys
    static constexpr int STAGE_BYTES = 2 * SLOT_BYTES;    // that of a pair stages of 128
    static constexpr int STAGES = D == 128 ? 5 : 10;      // stages of the pair's ring = slots of each stream's
    static constexpr int HALVES = D / 64;
    // barriers: pair ring, slots; queries, scores, probabilities, outputs (of the pair's streams, of single ones); three lists; ends
    static constexpr int PAIR_FULL = 0, PAIR_EMPTY = PAIR_FULL + STAGES, SLOT_FULL = PAIR_EMPTY + STAGES, SLOT_EMPTY = SLOT_FULL + 2 * STAGES,
                         Q_FULL = SLOT_EMPTY + 2 * STAGES, Q_EMPTY = Q_FULL + 4, S_FULL = Q_EMPTY + 4, P_FULL = S_FULL + 4, O_FULL = P_FULL + 4,
                         LIST_FULL = O_FULL + 4, LIST_EMPTY = LIST_FULL + 3 * ITEMS, PAIRS_DONE = LIST_EMPTY + 3 * ITEMS, DONE = PAIRS_DONE + 1,
                         NUM_BARS = DONE + 2;
    static constexpr int SMEM = 1024 + 2 * Q_BYTES + STAGES * STAGE_BYTES + NUM_BARS * 8 + 16 + 3 * ITEMS * 64;
    static_assert(SMEM + 512 <= 232448, "shared memory of an SM");
    // f32 accumulate, bf16 x bf16; S: both K-major; O: the second operand lies with its columns together (MN-major)
    static constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BM >> 4) << 24);
    static constexpr uint32_t IDESC_S = IDESC | ((uint32_t)(BN >> 3) << 17), IDESC_S_SLOT = IDESC | ((uint32_t)(HN >> 3) << 17);
    static constexpr uint32_t IDESC_O = IDESC | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    static constexpr uint32_t S_COL = 0, O_COL = 256;  // per stream: S (and P over it) 128 columns, O D columns
};

struct Params {
    __nv_bfloat16* out;
    const __nv_bfloat16 *q, *k, *v;  // read here only by visible_row
    long long q_token, q_head, k_page, k_token, k_head, v_page, v_token, v_head;
    const int *page_table, *kv_lens, *cu;
    float* partial;   // 8 slots per block of slot_rows x (D + 2) floats: for each worker a piece that began before it, one that goes on
    int* headers;     // 4 per block: for each worker the item that begins there and goes on
    long long o_token, o_head;
    float c;          // scale log2(e)
    int rows, batch, width, hkv, group, tokens /* of a stream's tile */, half_tokens /* of half a tile */, num_pages, page, page_shift, slot_rows, wide_stores;
};

// One item, or the piece of it that a worker (the pair, or a single stream) has.
struct Item {
    int start, n, kv, b, hk;  // rows start .. start + n of the batch, kv keys
    int tok0;                 // first token (the second stream of a pair: p.tokens further)
    int t0, steps0, steps1;   // first step, steps of each stream
    int slot;                 // -1: the whole item; else the place of the partial result (second stream: 2 gridDim.x further)
    int last;                 // nothing behind this descriptor (it carries no work)
};
// (Two members and no array: indexed by the stream, an array of a local Item would lie in memory.)
static_assert(sizeof(Item) <= 64, "descriptor");

constexpr int HEADER = 8;  // ints: pieces (0: none), start, hk, tok0, rows

struct Request {
    int start, n, kv;
};
__device__ __forceinline__ Request request_of(const Params& p, int b) {
    const int lo = min(max(p.cu[b], 0), p.rows), hi = min(max(p.cu[b + 1], lo), p.rows);
    return {lo, hi - lo, min(max(p.kv_lens[b], 0), p.width * p.page)};
}
// Keys that a token of a request sees, and the steps of a tile that ends with it; a tile that sees nothing still takes one
// step, which gives its zeros.
__device__ __forceinline__ int keys_of(const Request& q, int token) { return min(max(q.kv - q.n + token + 1, 0), q.kv); }
__device__ __forceinline__ int steps_of(int keys) { return max((keys + BN - 1) / BN, 1); }
__device__ __forceinline__ int pair_tiles(const Request& q, int tokens) { return (q.n + tokens - 1) / (2 * tokens); }
__device__ __forceinline__ bool has_single(const Request& q, int tokens) { return q.n > 0 && (q.n - 1) % (2 * tokens) < tokens; }

// sum over i < n of floor((a i + b) / 128), a, b >= 0, a n + b < 2^31: whole multiples of the divisor out of a and b, then the same
// sum the other way round (over the values of the quotient), until the slope is zero.
__device__ __forceinline__ long long sum_of_quotients(uint32_t n, uint32_t a, uint32_t b) {
    long long sum = 0;
    uint32_t m = BN;
    while (true) {
        const uint32_t qa = a / m, qb = b / m;
        sum += (long long)n * (n - 1) / 2 * qa + (long long)n * qb;
        a -= qa * m, b -= qb * m;
        const uint32_t y = a * n + b;
        if (y < m) return sum;
        n = y / m, b = y - n * m;
        const uint32_t t = m;
        m = a, a = t;
    }
}
// Places that the first `tiles` pair tiles of a request and one head take in the line: their steps and kPairCost each.  A full
// tile i of w = 2 tokens ends with token (i + 1) w - 1, so it takes max(floor(((i + 1) w - 1 + kv - n) / 128), 0) + 1 steps;
// one that is not full ends with the last token.
__device__ __forceinline__ long long pairs_before(const Request& q, int tiles, int tokens) {
    long long sum = (long long)tiles * kPairCost;
    if ((long long)tiles * 2 * tokens > q.n) sum += steps_of(q.kv), --tiles;
    if (tiles > 0) {
        const int w = 2 * tokens, e = w - 1 + q.kv - q.n;
        const int first = e >= 0 ? 0 : (-e + w - 1) / w;
        sum += tiles;
        if (tiles > first) sum += sum_of_quotients(tiles - first, w, e + w * first);
    }
    return sum;
}
__device__ __forceinline__ long long single_places(const Params& p, const Request& q) {
    return has_single(q, p.tokens) ? (long long)(steps_of(q.kv) + kSingleCost) * p.hkv : 0;
}

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
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
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
// Units of 2^32 cycles (some two seconds) that a wait lasts at most.  A warp that sums rows again (visible_row), which over a long context
// may take that long, adds what this may take before it begins.
__device__ __forceinline__ int& wait_units() {
    __shared__ int units;
    return units;
}
constexpr int kWaitUnits = 2;  // the first begins anywhere in a unit: two to four seconds
constexpr long long kAgainCycles = 1000;  // of visible_row per key, at the very most (about 150 measured)
__device__ __forceinline__ uint32_t clock_units() {
    uint32_t t;
    asm volatile("mov.u32 %0, %%clock_hi;" : "=r"(t));
    return t;
}
// A bounded wait, without a call - behind one the compiler cannot give the roles registers of their own - and
// short: it stands at some fifty places, and the kernel's time on small calls is the time that its instructions take to arrive (128
// requests of 1000 tokens: 113.4 us with a limit of 4 10^9 cycles and no more, 115.6 like this, 119 - 122 where every wait looked whether a
// warp sums again and began anew).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint32_t t0 = clock_units();
#pragma unroll 1
    do {
        if (mbar_try_wait(bar, parity)) return true;
    } while (clock_units() - t0 < (uint32_t)*(volatile int*)&wait_units());
    return false;
}

// Weight of a partial result with maximum m (in log2 units) when the common maximum is `top`.
__device__ __forceinline__ float weight_to(float m, float top) { return m == -CUDART_INF_F ? 0.f : ex2(m - top); }

// 32 columns of a row, in 32-byte stores where its alignment allows: a thread has a row of its own, so a store instruction
// touches 32 lines either way.
__device__ __forceinline__ void store_row32(__nv_bfloat16* dst, const uint32_t (&w)[16], int wide) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 2 * i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                         "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(dst + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
}

// What the softmax warps of a stream keep of an item: the reference maximum and the sum of the thread's row.
struct RowState {
    float m, l;  // m in units of the scores; -inf: nothing seen
};
constexpr float kMostSum = 1024.f;  // of a step's weights before the reference maximum is looked at again

// exp2 of a pair on the arithmetic pipes: the nearest integer n by adding 1.5 2^23, 2^n by shifting it into place, and a polynomial
// of degree 3 for the rest in [-1/2, 1/2] (best in relative error: 7.5e-5, a fiftieth of what rounding to bf16 may add).
// From 2^-126.5 down the result is zero, as what is masked has to be.
__device__ __forceinline__ void ex2_pair(uint64_t x2, float& r0, float& r1) {
    float a, b;
    unpack2(x2, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(127.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(127.f));
    x2 = pack2(a, b);
    const uint64_t t = add2(x2, pack2(12582912.f, 12582912.f)), n = add2(t, pack2(-12582912.f, -12582912.f)), f = fma2(n, pack2(-1.f, -1.f), x2);
    uint64_t p = fma2(pack2(0.0551716685f, 0.0551716685f), f, pack2(0.2426111251f, 0.2426111251f));
    p = fma2(p, f, pack2(0.6932609677f, 0.6932609677f));
    p = fma2(p, f, pack2(0.9999280572f, 0.9999280572f));
    unpack2(t, a, b);
    const float e0 = __int_as_float((__float_as_int(a) << 23) + 0x3f800000), e1 = __int_as_float((__float_as_int(b) << 23) + 0x3f800000);
    unpack2(fma2(p, pack2(e0, e1), 0), r0, r1);
}
// exp2(c s + off) of 32 scores, packed to bf16, and their sum.  The special function unit gives 16 a cycle; some pairs go the other
// way: at D 128, where the products cost as much as the exponentials, two of sixteen (4 prompts of 4096: 530 us with none, 495 with
// two, 502 with three, 549 with four), at D 64, where they cost half, five (485 with none, 442 with two, 430 with three or six, 426 with
// five, 438 with eight).
template <int D>
__device__ __forceinline__ void weights32(const uint32_t (&s)[32], uint64_t c2, uint64_t off2, uint32_t* pk, uint64_t (&sum)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x0, x1;
        const uint64_t x2 = fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, off2);
        if (D == 64 ? i % 3 == 2 : i % 8 == 7) {
            ex2_pair(x2, x0, x1);
        } else {
            unpack2(x2, x0, x1);
            x0 = ex2(x0), x1 = ex2(x1);
        }
        sum[i & 1] = add2(sum[i & 1], pack2(x0, x1));
        pk[i] = pack_bf16x2(x0, x1);
    }
}

// One step of a row: scores in tensor memory -> probabilities over them.  `seen` keys of this step are visible to the row.
// Mostly all of them are, and the reference maximum still serves: then nothing has to be known of the scores before their
// exponentials, and the sum tells afterwards (no weight beyond kMostSum can hide in it, nor a NaN).  Else a pass for the maximum comes
// first, which writes what is masked back as minus infinity.  A chunk of 4096 behind 28672 tokens: 3.35 ms with the maximum taken in
// every step, 3.10 like this.  The code is kept short for calls of many short items, between which the roles' instructions have to
// come in again: with 26 KB more of it 128 requests of 1000 tokens took 138 us in place of 115.
template <int D>
__device__ __forceinline__ void softmax_step(RowState& st, const uint32_t s_addr, const uint32_t o_addr, const int seen, const bool live, const bool first, const float c) {
    const bool partial = __any_sync(~0u, seen < BN);
    bool check = !partial && !__any_sync(~0u, live && st.m == -CUDART_INF_F);
    uint32_t pk[2][32];
    float l, slack = 8.f;
    while (true) {
        if (!check) {
            float top = st.m;
#pragma unroll 1
            for (int i0 = 0; i0 < BN; i0 += 32) {
                uint32_t s[32];
                tmem_ld32(s_addr + i0, s);
                tmem_ld_wait32(s);
                if (partial) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (i0 + i >= seen) s[i] = 0xff800000u;  // whatever stands there
                    tmem_st32(s_addr + i0, s);
                }
                float t[4] = {top, top, top, top};
#pragma unroll
                for (int i = 0; i < 32; i += 2) t[i / 2 % 4] = fmaxf(fmaxf(t[i / 2 % 4], __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
            }
            // 2^8 of growth is harmless in fp32 sums and bf16 probabilities alike; where the sum has shown more the maximum follows at once
            const bool grown = live && (top * c > st.m * c + slack || (st.m == -CUDART_INF_F && top != -CUDART_INF_F));
            if (__any_sync(~0u, grown)) {
                const float a = st.m == -CUDART_INF_F ? 0.f : ex2((st.m - top) * c);
                st.m = top;
                st.l *= a;
                if (!first) {
#pragma unroll 1
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
            tmem_st_wait();
        }
        const float off = st.m == -CUDART_INF_F ? 0.f : -st.m * c;
        const uint64_t c2 = pack2(c, c), off2 = pack2(off, off);
        uint64_t sum[2] = {0, 0};
        uint32_t s[2][32];
        tmem_ld32(s_addr, s[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tmem_ld_wait32(s[i & 1]);
            if (i < 3) tmem_ld32(s_addr + 32 * (i + 1), s[(i + 1) & 1]);
            weights32<D>(s[i & 1], c2, off2, pk[i / 2] + 16 * (i & 1), sum);
        }
        float a, b;
        unpack2(add2(sum[0], sum[1]), a, b);
        l = a + b;
        if (!check || !__any_sync(~0u, live && !(l <= kMostSum))) break;
        check = false, slack = 0.f;
    }
    st.l += l;
    tmem_st32(s_addr, pk[0]);
    tmem_st32(s_addr + 32, pk[1]);
    tmem_st_wait();
}

// D / 32 neighbouring columns of a row of keys or values.
template <int D>
__device__ __forceinline__ void lane_columns(const __nv_bfloat16* src, bool live, float (&x)[D / 32]) {
    uint2 w = make_uint2(0, 0);
    if (live) {
        if (D == 128) w = *reinterpret_cast<const uint2*>(src);
        else w.x = *reinterpret_cast<const uint32_t*>(src);
    }
    x[0] = bf16lo_to_f32(w.x), x[1] = bf16hi_to_f32(w.x);
    if (D == 128) x[D / 32 - 2] = bf16lo_to_f32(w.y), x[D / 32 - 1] = bf16hi_to_f32(w.y);
}

// The sum over keys from .. to - 1 of exp2(c q.k - off) v for one row, by a warp; a lane has D / 32 columns.  For rows whose tile holds
// keys that they do not see and whose values are not finite: there the product's zero weights give NaN.  Eight keys at a time (`from`
// is a multiple of eight, so they lie in one page), the next ones' page asked for ahead: about 150 cycles per key.
template <int D>
__device__ __forceinline__ void visible_row(const Params& p, const Item& d, int token, int head, int from, int to, float off, int lane, float (&o)[D / 32]) {
    constexpr int E = D / 32, KEYS = 8;
    float q[E];
    lane_columns<D>(p.q + (long long)(d.start + token) * p.q_token + (long long)head * p.q_head + lane * E, true, q);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0;
    const int* table = p.page_table + (long long)d.b * p.width;
    int next = table[from >> p.page_shift];
#pragma unroll 1
    for (int j = from; j < to; j += KEYS) {
        const int id = next, at = j & (p.page - 1);
        if (j + KEYS < to) next = table[(j + KEYS) >> p.page_shift];
        const bool there = (unsigned)id < (unsigned)p.num_pages;  // a page outside the pool reads as zeros
        const __nv_bfloat16* k = p.k + (there ? id : 0) * p.k_page + at * p.k_token + d.hk * p.k_head + lane * E;
        const __nv_bfloat16* v = p.v + (there ? id : 0) * p.v_page + at * p.v_token + d.hk * p.v_head + lane * E;
        float s[KEYS], x[KEYS][E];
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            float y[E];
            lane_columns<D>(k + i * p.k_token, there && j + i < to, y);
            lane_columns<D>(v + i * p.v_token, there && j + i < to, x[i]);
            s[i] = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) s[i] = fmaf(q[e], y[e], s[i]);
        }
#pragma unroll
        for (int n = 16; n > 0; n >>= 1)
#pragma unroll
            for (int i = 0; i < KEYS; ++i) s[i] += __shfl_xor_sync(~0u, s[i], n);
#pragma unroll
        for (int i = 0; i < KEYS; ++i) {
            const float w = j + i < to ? ex2(fmaf(s[i], p.c, -off)) : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[i][e], o[e]);
        }
    }
}

// Where a line is cut `off` places into an item of `cost`: at the item's edge if that is at most `near` places away.
__device__ __forceinline__ int cut_at(int off, int cost, int near) { return off <= near ? 0 : cost - off <= near ? cost : off; }
// Pieces of an item that begins in worker w's part and goes on: one per worker up to that of its last place, where the cut before
// that is not moved to the item's end.
__device__ __forceinline__ int pieces_of(long long item_end, long long share, int near, int w) {
    const int last = (int)((item_end - 1) / share);
    return last - w + (last == w || item_end - last * share > near);
}

// A worker's place in a line: from u to end, beginning in request b `rest` places behind the request's first.
struct Place {
    long long u, end, rest, share, per_head;  // per_head: places of the request's pairs and one head
    int b;
    Request q;  // request b
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_kernel(const Params p, const __grid_constant__ CUtensorMap qmap,
                                                                      const __grid_constant__ CUtensorMap hqmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using C = Cfg<D>;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const gen = raw + (base - smem_u32(raw));
    const uint32_t q_smem = base, ring = base + 2 * C::Q_BYTES, bars = ring + C::STAGES * C::STAGE_BYTES;
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
    Item* const items = reinterpret_cast<Item*>(gen + (bars - base) + 8 * C::NUM_BARS);  // three lists: pairs, stream 0, stream 1
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(items + 3 * ITEMS);
    __shared__ long long scan[2][kThreads / 32];
    __shared__ int scan_longest[kThreads / 32];
    __shared__ Place places[3];  // of this block's pair, of its streams

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = gridDim.x;
    if (warp == kMmaWarp0) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    } else if (warp == kCopyWarp0) {
        if (lane == 0) tma_prefetch_desc(&qmap), tma_prefetch_desc(&hqmap), tma_prefetch_desc(&kmap), tma_prefetch_desc(&vmap);
        for (int i = lane; i < C::NUM_BARS; i += 32) {
            int count = 1;
            if (i >= C::P_FULL && i < C::P_FULL + 4) count = 4;                   // four warps of a stream
            if (i >= C::LIST_EMPTY && i < C::LIST_EMPTY + ITEMS) count = 11;      // MMA warps, copier of the queries, eight softmax warps
            if (i >= C::LIST_EMPTY + ITEMS && i < C::LIST_EMPTY + 3 * ITEMS) count = 5;  // MMA warp, four softmax warps
            mbar_init(bar(i), count);
        }
        fence_barrier_init();
    }
    if (threadIdx.x < 3) places[threadIdx.x].b = -1;
    if (threadIdx.x == 0) wait_units() = kWaitUnits;
    if (threadIdx.x >= 32 && threadIdx.x < 36) p.headers[((threadIdx.x - 32) * blocks + blockIdx.x) * HEADER] = 0;
    let_dependents_launch();  // the joining kernel, which waits for this one's end

    // ---- the lines: all requests' sums, and the requests in which this block's pieces begin
    Request mine;
    int longest = 0;  // steps of the longest item, or a little more
    long long per_head, places_of[2], run[2], carry[2] = {0, 0};  // of this thread's request; up to and with it; of all rounds so far
    auto sum_round = [&](int b) {
        mine = Request{0, 0, 0};
        if (b < p.batch) mine = request_of(p, b);
        per_head = pairs_before(mine, pair_tiles(mine, p.tokens), p.tokens);
        places_of[0] = run[0] = per_head * p.hkv, places_of[1] = run[1] = single_places(p, mine);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const long long o = __shfl_up_sync(~0u, run[k], d);
                if (lane >= d) run[k] += o;
            }
        }
        const int most = __reduce_max_sync(~0u, mine.n > 0 ? steps_of(mine.kv) : 0);
        __syncthreads();
        if (lane == 31) scan[0][warp] = run[0], scan[1][warp] = run[1], scan_longest[warp] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) longest = max(longest, scan_longest[w]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            long long all = 0;
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w) {
                const long long x = scan[k][w];
                run[k] += w < warp ? x : 0;
                all += x;
            }
            run[k] += carry[k];
            carry[k] += all;
        }
    };
    long long total[2], share[2];
    auto find = [&](int b) {
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            const int k = w > 0;
            const long long u = share[k] * (w == 2 ? blocks + (int)blockIdx.x : (int)blockIdx.x), before = run[k] - places_of[k];
            if (u >= before && u < run[k]) places[w] = Place{u, min(u + share[k], total[k]), u - before, share[k], per_head, b, mine};
        }
    };
    for (int pass = 0; pass < 2; ++pass) {  // the totals, then the places
        for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
            sum_round(b0 + (int)threadIdx.x);
            if (pass == 1) find(b0 + (int)threadIdx.x);
        }
        if (pass == 0) {
            total[0] = carry[0], total[1] = carry[1], carry[0] = carry[1] = 0;
            share[0] = max((total[0] + blocks - 1) / blocks, longest >= kLongItem ? 8ll : 1ll);
            share[1] = max((total[1] + 2 * blocks - 1) / (2 * blocks), longest >= kLongItem ? 3ll : longest >= kLongItem / 4 ? 2ll : 1ll);
            if (p.batch <= kThreads) {  // this thread's sums are still at hand
                find((int)threadIdx.x);
                break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const bool has_pairs = places[0].b >= 0;
    const bool none = !has_pairs && places[1].b < 0 && places[2].b < 0;

    bool ok = true;  // false: a wait has given up; every role leaves its loop, no role waits for another without a limit

    // Takes the next descriptor of a list; false: the list has ended (or a wait has given up).
    auto take = [&](int list, uint32_t& it, Item& d) {
        const uint32_t at = it % ITEMS, ph = (it / ITEMS) & 1u;
        ++it;
        ok = __all_sync(~0u, ok && wait_bar(bar(C::LIST_FULL + list * ITEMS + at), ph));
        d = items[list * ITEMS + at];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::LIST_EMPTY + list * ITEMS + at));
        return ok && !d.last;
    };

    // The register limits stand at the head of the roles: where they cannot be told apart the compiler takes the lower one.
    if (none) {
    } else if (warp >= kFirstSoftmax) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ------------------------------ softmax, results ------------------------------
        const int s = (warp - kFirstSoftmax) >> 2, quad = warp & 3, lane_row = quad * 32 + lane;  // this thread's row of its stream
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + C::S_COL + 128 * s + lanes, o_addr = tmem + C::O_COL + D * s + lanes;
        const int tile_rows = p.tokens * p.group;
        for (int turn = has_pairs ? 0 : 1; turn < 2; ++turn) {  // the pairs, then the items of this stream alone
            const int list = turn == 0 ? 0 : 1 + s;
            if (!ok || places[list].b < 0) break;
            const uint32_t s_full = bar(C::S_FULL + 2 * turn + s), p_full = bar(C::P_FULL + 2 * turn + s), o_full = bar(C::O_FULL + 2 * turn + s);
            uint32_t s_ph = 0, o_ph = 0;
            Item d;
            for (uint32_t it = 0; take(list, it, d);) {
                const int steps = s == 0 ? d.steps0 : d.steps1, tok0 = d.tok0 + (list == 0 ? s * p.tokens : 0);
                // Where few rows are there the second stream's lie in the other two quadrants: its warps run on other parts of the SM.
                const int row = lane_row - (list > 0 && s == 1 && d.n - tok0 <= p.half_tokens ? BM / 2 : 0);
                const int row_token = row >= 0 ? row / p.group : 0, row_head = row - row_token * p.group, token = tok0 + row_token;
                const bool live = row >= 0 && row < tile_rows && token < d.n;
                const bool warp_live = __any_sync(~0u, live);
                const int keys = live ? min(max(d.kv - d.n + token + 1, 0), d.kv) : 0x7fffffff;  // a row that is not there needs no mask
                RowState rs{-CUDART_INF_F, 0.f};
                for (int i = 0; i < steps; ++i) {
                    ok = __all_sync(~0u, ok && wait_bar(s_full, s_ph));
                    if (!ok) break;
                    s_ph ^= 1u;
                    tc_fence_after();
                    if (warp_live) softmax_step<D>(rs, s_addr, o_addr, keys - (d.t0 + i) * BN, live, i == 0, p.c);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full);
                }
                if (steps > 0) {
                    ok = __all_sync(~0u, ok && wait_bar(o_full, o_ph));
                    o_ph ^= 1u;
                    tc_fence_after();
                }
                if (!ok) break;
                if (!warp_live) continue;
                const float l = rs.l;
                // Values that are not finite at keys which a row does not see (later tokens of its chunk) must not reach it.
                const int stop = min((d.t0 + steps) * BN, d.kv);
                const bool hidden = __any_sync(~0u, live && keys < stop);
                uint64_t check[2] = {0, 0};  // NaN where a column is not finite
                if (d.slot < 0) {
                    const float inv = 1.f / l;
                    const bool empty = l == 0.f;  // no key in sight: zeros
                    __nv_bfloat16* const dst = p.out + (long long)(d.start + token) * p.o_token + (long long)(d.hk * p.group + row_head) * p.o_head;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32], w[16];
                        tmem_ld32(o_addr + c0, o);
                        tmem_ld_wait32(o);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            w[j] = empty ? 0u : pack_bf16x2(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv);
                        if (hidden) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) check[j % 2] = fma2(pack2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1])), 0, check[j % 2]);
                        }
                        if (live) store_row32(dst + c0, w, p.wide_stores);
                    }
                } else {
                    const bool nothing = l == 0.f;  // the row sees nothing of this piece (which may have no step for its stream)
                    float* const slot = p.partial + (long long)(d.slot + (list == 0 ? 2 * blocks * s : 0)) * p.slot_rows * (D + 2);
                    const bool mine = row >= 0 && row < p.slot_rows;
                    if (mine) {
                        slot[p.slot_rows * D + row] = rs.m == -CUDART_INF_F ? rs.m : rs.m * p.c;
                        slot[p.slot_rows * (D + 1) + row] = l;
                    }
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c0, o);
                        tmem_ld_wait32(o);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint4 x = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                            if (nothing) x = make_uint4(0, 0, 0, 0);
                            check[0] = fma2(pack2(__uint_as_float(x.x), __uint_as_float(x.y)), 0, check[0]);
                            check[1] = fma2(pack2(__uint_as_float(x.z), __uint_as_float(x.w)), 0, check[1]);
                            if (mine) reinterpret_cast<uint4*>(slot)[(c0 / 4 + j) * p.slot_rows + row] = x;
                        }
                    }
                }
                float nan0, nan1;
                unpack2(add2(check[0], check[1]), nan0, nan1);
                uint32_t bad = __ballot_sync(~0u, hidden && live && !(nan0 + nan1 == 0.f) && l > 0.f && l < CUDART_INF_F && keys < stop);
                if (bad != 0) {
                    __syncwarp();  // the rows' stores are behind
                    if (lane == 0) atomicAdd(&wait_units(), (int)(__popc(bad) * (stop - d.t0 * BN) * kAgainCycles >> 32));
                }
                while (bad != 0) {
                    const int from = __ffs(bad) - 1, r = __shfl_sync(~0u, row, from), t = __shfl_sync(~0u, token, from);
                    const int h = d.hk * p.group + __shfl_sync(~0u, row_head, from);
                    const float sum = __shfl_sync(~0u, l, from);
                    bad &= bad - 1;
                    float o[D / 32];
                    visible_row<D>(p, d, t, h, d.t0 * BN, min(__shfl_sync(~0u, keys, from), stop), __shfl_sync(~0u, rs.m, from) * p.c, lane, o);
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) {
                        const int col = lane * (D / 32) + e;
                        if (d.slot < 0)
                            p.out[(long long)(d.start + t) * p.o_token + (long long)h * p.o_head + col] = __float2bfloat16(o[e] / sum);
                        else
                            p.partial[(long long)(d.slot + (list == 0 ? 2 * blocks * s : 0)) * p.slot_rows * (D + 2) + ((col / 4) * p.slot_rows + r) * 4 + col % 4] = o[e];
                    }
                }
                tc_fence_before();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        if (warp == kCopyWarp0 || warp == kCopyWarp1) {
            // ------------------------------ items; pages and queries -> shared memory ------------------------------
            const int s = warp == kCopyWarp1;
            const int box_rows = min(p.page, HN), boxes = BN / box_rows;
            // Lane l copies box l / HALVES of a step, columns 64 (l % HALVES).
            const int box = lane / C::HALVES, half = lane % C::HALVES;
            auto publish = [&](int list, uint32_t& it, const Item& d) {
                const uint32_t at = it % ITEMS, ph = (it / ITEMS) & 1u;
                ++it;
                ok = __all_sync(~0u, ok && wait_bar(bar(C::LIST_EMPTY + list * ITEMS + at), ph ^ 1u));
                if (lane == 0) {
                    items[list * ITEMS + at] = d;
                    mbar_arrive(bar(C::LIST_FULL + list * ITEMS + at));
                }
                __syncwarp();
            };
            auto load_queries = [&](int tile, int set, uint32_t& ph, int token, int hk, bool upper) {
                const uint32_t full = bar(C::Q_FULL + 2 * set + tile);
                ok = __all_sync(~0u, ok && wait_bar(bar(C::Q_EMPTY + 2 * set + tile), ((ph >> tile) & 1u) ^ 1u));
                ph ^= 1u << tile;
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(full, (upper ? p.half_tokens : p.tokens) * p.group * D * 2);
                    for (int h = 0; h < C::HALVES; ++h)
                        tma_load_3d(q_smem + tile * C::Q_BYTES + h * (BM * 128) + (upper ? BM / 2 * 128 : 0), upper ? &hqmap : &qmap, 64 * h,
                                    hk * p.group, token, full);
                }
                __syncwarp();
            };
            // The page of this lane's box; where that holds no key of the request one behind the pool: zeros without a read.
            auto page_at = [&](const Item& d, int step) {
                const int at = (step * BN + box * box_rows) >> p.page_shift, held = (d.kv + p.page - 1) >> p.page_shift;
                int id = p.num_pages;
                if (box < boxes && at < held) id = p.page_table[(long long)d.b * p.width + at];
                return (unsigned)id < (unsigned)p.num_pages ? id : p.num_pages;
            };
            auto copy_box = [&](const CUtensorMap* map, uint32_t dst, int step, int hk, int id, uint32_t full) {
                tma_load_4d(dst, map, half * 64, (step * BN + box * box_rows) & (p.page - 1), hk, id, full);
            };
            if (has_pairs && s == 0) {
                uint32_t it = 0, stage = 0, ph = 0;
                auto load = [&](const CUtensorMap* map, const Item& d, int step, int id) {
                    ok = __all_sync(~0u, ok && wait_bar(bar(C::PAIR_EMPTY + stage), ph ^ 1u));
                    if (!ok) return;
                    const uint32_t full = bar(C::PAIR_FULL + stage);
                    if (lane == 0) mbar_arrive_expect_tx(full, C::STAGE_BYTES);
                    __syncwarp();
                    if (box < boxes) copy_box(map, ring + stage * C::STAGE_BYTES + half * (BN * 128) + box * box_rows * 128, step, d.hk, id, full);
                    if (++stage == C::STAGES) stage = 0, ph ^= 1u;
                };
                const Place w = places[0];
                int b = w.b;
                Request q = w.q;
                int tiles = pair_tiles(q, p.tokens);
                long long rest = w.rest;
                int hk = (int)(rest / w.per_head);
                rest -= hk * w.per_head;
                int tile = 0, hi = tiles - 1;  // the last tile that begins at or before the place
                long long begin = 0;
                while (tile < hi) {
                    const int mid = (tile + hi + 1) >> 1;
                    const long long at = pairs_before(q, mid, p.tokens);
                    if (at <= rest) tile = mid, begin = at; else hi = mid - 1;
                }
                int off = (int)(rest - begin);
                const int near = (int)min((long long)kPairNear, (w.share - 1) / 2);  // half a piece would reach the next cut
                long long u = w.u - off;
                off = cut_at(off, steps_of(keys_of(q, min((tile + 1) * 2 * p.tokens, q.n) - 1)) + kPairCost, near);
                Item d;
                for (u += off; ok && u < w.end;) {
                    d.start = q.start, d.n = q.n, d.kv = q.kv, d.b = b, d.hk = hk, d.tok0 = tile * 2 * p.tokens, d.last = 0;
                    const int steps = steps_of(keys_of(q, min(d.tok0 + 2 * p.tokens, q.n) - 1)), cost = steps + kPairCost;
                    int to = (int)min((long long)cost, off + (w.end - u));
                    if (to < cost) to = cut_at(to, cost, near);
                    if (to <= off && to < cost) break;
                    d.t0 = max(off - kPairCost, 0);
                    const int t1 = max(to - kPairCost, 0);
                    const bool begins = d.t0 == 0, ends = to == cost;
                    if (t1 > d.t0) {
                        d.slot = begins && ends ? -1 : 2 * (int)blockIdx.x + (begins ? 1 : 0);
                        d.steps0 = max(min(t1, steps_of(keys_of(q, d.tok0 + p.tokens - 1))) - d.t0, 0);  // its tokens see fewer keys
                        d.steps1 = t1 - d.t0;
                        publish(0, it, d);
                        if (begins && !ends && lane < 2) {  // the pieces behind this one: one per worker, up to that of the last place
                            int* h = p.headers + (lane * blocks + blockIdx.x) * HEADER;
                            const int tok0 = d.tok0 + lane * p.tokens;
                            h[1] = q.start, h[2] = hk, h[3] = tok0, h[4] = max(min(p.tokens, q.n - tok0), 0) * p.group;
                            h[0] = pieces_of(u + (cost - off), w.share, near, (int)blockIdx.x);
                        }
                        const int n = d.steps1;
                        int id = 0, next_id = page_at(d, d.t0);
#pragma unroll 1
                        for (int i = -1; ok && i < n; ++i) {  // keys run one step ahead of the values
                            const int far_id = i + 2 < n ? page_at(d, d.t0 + i + 2) : 0;  // asked for a step before it is needed
#pragma unroll 1
                            for (int k = 1; k >= 0; --k)
                                if (i + k >= 0 && i + k < n) load(k ? &kmap : &vmap, d, d.t0 + i + k, k ? next_id : id);
                            id = next_id, next_id = far_id;
                        }
                    }
                    u += to - off;
                    off = 0;
                    if (ends && ++tile == tiles) {
                        tile = 0;
                        if (++hk == p.hkv) {
                            hk = 0;
                            do {  // u < end says that one with pairs follows
                                if (++b >= p.batch) break;
                                q = request_of(p, b);
                                tiles = pair_tiles(q, p.tokens);
                            } while (tiles == 0);
                            if (b >= p.batch) break;
                        }
                    }
                }
                d.last = 1;
                publish(0, it, d);
            } else if (has_pairs) {
                uint32_t q_ph = 0;
                Item d;
                for (uint32_t it = 0; take(0, it, d);) {
#pragma unroll 1
                    for (int t = 0; t < 2; ++t)
                        if ((t == 0 ? d.steps0 : d.steps1) > 0) load_queries(t, 0, q_ph, d.start + d.tok0 + t * p.tokens, d.hk, false);
                }
            }
            const Place w = places[1 + s];
            if (w.b >= 0) {
                // The pairs' products have read the ring and the queries: now each stream has a half.
                if (has_pairs) ok = __all_sync(~0u, ok && wait_bar(bar(C::PAIRS_DONE), 0));
                const uint32_t own = ring + s * (C::STAGES * C::SLOT_BYTES), first = (uint32_t)(s * C::STAGES);
                const int id = s * blocks + (int)blockIdx.x;
                uint32_t it = 0, slot = 0, ph = 0, q_ph = 0;
                auto load = [&](const CUtensorMap* map, const Item& d, int step, int page_id) {
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        ok = __all_sync(~0u, ok && wait_bar(bar(C::SLOT_EMPTY + first + slot), ph ^ 1u));
                        if (!ok) return;
                        const uint32_t full = bar(C::SLOT_FULL + first + slot);
                        if (lane == 0) mbar_arrive_expect_tx(full, C::SLOT_BYTES);
                        __syncwarp();
                        const int at = box * box_rows - h * HN;  // the box's first row in this slot
                        if (at >= 0 && at < HN) copy_box(map, own + slot * C::SLOT_BYTES + half * (HN * 128) + at * 128, step, d.hk, page_id, full);
                        if (++slot == C::STAGES) slot = 0, ph ^= 1u;
                    }
                };
                int b = w.b;
                Request q = w.q;
                int cost = steps_of(q.kv) + kSingleCost;
                int hk = (int)(w.rest / cost), off = (int)(w.rest - (long long)hk * cost);
                Item d;
                for (long long u = w.u; ok && u < w.end;) {
                    const int to = (int)min((long long)cost, off + (w.end - u));
                    d.t0 = max(off - kSingleCost, 0);
                    const int t1 = max(to - kSingleCost, 0);
                    const bool begins = d.t0 == 0, ends = to == cost;
                    if (t1 > d.t0) {
                        d.start = q.start, d.n = q.n, d.kv = q.kv, d.b = b, d.hk = hk, d.last = 0;
                        d.tok0 = (q.n - 1) / (2 * p.tokens) * (2 * p.tokens);
                        d.steps0 = d.steps1 = t1 - d.t0;  // the list's stream looks at its own
                        d.slot = begins && ends ? -1 : 4 * blocks + 2 * id + (begins ? 1 : 0);
                        int ids[3] = {page_at(d, d.t0), d.t0 + 1 < t1 ? page_at(d, d.t0 + 1) : 0, 0};  // asked for a step before they are needed
                        publish(1 + s, it, d);
                        for (int step = d.t0; ok && step < t1; ++step) {
                            if (step + 2 < t1) ids[2] = page_at(d, step + 2);
#pragma unroll 1
                            for (int k = 1; k >= 0; --k) {
                                load(k ? &kmap : &vmap, d, step, ids[0]);
                                if (k && step == d.t0) load_queries(s, 1, q_ph, d.start + d.tok0, d.hk, s == 1 && d.n - d.tok0 <= p.half_tokens);
                            }
                            ids[0] = ids[1], ids[1] = ids[2];
                        }
                        if (begins && !ends && lane == 0) {
                            int* h = p.headers + (2 * blocks + id) * HEADER;
                            h[1] = q.start, h[2] = hk, h[3] = d.tok0, h[4] = (q.n - d.tok0) * p.group;
                            h[0] = pieces_of(u + (cost - off), w.share, 0, id);
                        }
                    }
                    u += to - off;
                    off = 0;
                    if (ends && ++hk == p.hkv) {
                        hk = 0;
                        do {  // u < end says that one with such an item follows
                            if (++b >= p.batch) break;
                            q = request_of(p, b);
                        } while (!has_single(q, p.tokens));
                        if (b >= p.batch) break;
                        cost = steps_of(q.kv) + kSingleCost;
                    }
                }
                d.last = 1;
                publish(1 + s, it, d);
            }
            if (!ok) {  // a wait has given up: copies under way (microseconds) get a millisecond to land
                const long long t0 = clock64();
                while (clock64() - t0 < 2000000) {
                }
            }
        } else {
            // ------------------------------ matrix products ------------------------------
            // All lanes walk the loops on values that the compiler knows to be the same in all of them (see elect_one).
            const int s = warp == kMmaWarp1;
            const uint64_t q_desc = make_smem_desc(q_smem);
            auto wait_in = [&](int barrier, uint32_t ph) { ok = __all_sync(~0u, ok && wait_bar(bar(barrier), ph)); };
            auto take_uniform = [&](int list, uint32_t& it, Item& d) {
                Item x;
                const bool more = take(list, it, x);
                d.n = __shfl_sync(~0u, x.n, 0), d.kv = __shfl_sync(~0u, x.kv, 0), d.t0 = __shfl_sync(~0u, x.t0, 0);
                d.steps0 = __shfl_sync(~0u, x.steps0, 0), d.steps1 = __shfl_sync(~0u, x.steps1, 0);
                return __all_sync(~0u, more) != 0;
            };
            // Rows of the last page behind the request's tokens hold anything; a zero weight does not make a NaN harmless.
            // `rows` rows at `at` in shared memory begin with key `key`; the halves of the columns lie rows * 128 bytes apart.
            auto clean = [&](uint32_t at, int key, int rows, int kv) {
                const int live = kv - key;
                if (live >= rows) return;
                const int from = max(live, 0), to = min((((max(live, 0) + key + p.page - 1) >> p.page_shift) << p.page_shift) - key, rows);
                if (from >= to) return;
                for (int i = from * C::HALVES * 8 + lane; i < to * C::HALVES * 8; i += 32) {
                    const int row = i / (C::HALVES * 8), piece = i % (C::HALVES * 8);
                    sts128(at + (piece / 8) * (rows * 128) + row * 128 + (piece % 8) * 16, make_uint4(0, 0, 0, 0));
                }
                fence_proxy_async_smem();
                __syncwarp();
            };
            if (has_pairs && s == 0) {
                struct Stage {
                    uint32_t at, ph;
                    __device__ __forceinline__ Stage next() const { return at + 1 == C::STAGES ? Stage{0, ph ^ 1u} : Stage{at + 1, ph}; }
                };
                const uint64_t k_desc = make_smem_desc(ring), v_desc = make_mn_desc(ring, BN * 128);
                Stage next{0, 0};  // the next stage of the ring in the order of the copies
                uint32_t q_ph[2] = {0, 0}, p_ph[2] = {0, 0};
                auto wait_q = [&](int t) { wait_in(C::Q_FULL + t, q_ph[t]), q_ph[t] ^= 1u; };
                auto wait_p = [&](int t) {
                    wait_in(C::P_FULL + t, p_ph[t]), p_ph[t] ^= 1u;
                    tc_fence_after();
                };
                // S = Q K^T of stream t; `frees`: the stage has been read, `last`: so have the item's queries
                auto scores = [&](int t, const Stage& g, bool frees, bool last) {
                    const uint64_t a = q_desc + (uint64_t)(t * (C::Q_BYTES >> 4)), b = k_desc + (uint64_t)(g.at * (C::STAGE_BYTES >> 4));
                    if (ok && elect_one()) {
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t o = (k / 4) * (BM * 128 >> 4) + (k % 4) * 2;
                            umma_bf16(tmem + C::S_COL + 128 * t, a + o, b + o, C::IDESC_S, k > 0);
                        }
                        umma_commit(bar(C::S_FULL + t));
                        if (frees) umma_commit(bar(C::PAIR_EMPTY + g.at));
                        if (last) umma_commit(bar(C::Q_EMPTY + t));
                    }
                    __syncwarp();
                };
                // O += P V of stream t; `ends`: the item has no more of them
                auto values = [&](int t, const Stage& g, bool accumulate, bool frees, bool ends) {
                    const uint64_t b = v_desc + (uint64_t)(g.at * (C::STAGE_BYTES >> 4));
                    wait_p(t);
                    if (ok && elect_one()) {
                        umma_bf16_ts(tmem + C::O_COL + D * t, tmem + C::S_COL + 128 * t, b, C::IDESC_O, accumulate);
#pragma unroll
                        for (int k = 1; k < BN / 16; ++k)
                            umma_bf16_ts(tmem + C::O_COL + D * t, tmem + C::S_COL + 128 * t + 8 * k, b + k * (2048 >> 4), C::IDESC_O, 1u);
                        if (frees) umma_commit(bar(C::PAIR_EMPTY + g.at));
                        if (ends) umma_commit(bar(C::O_FULL + t));
                    }
                    __syncwarp();
                };
                Item d;
                for (uint32_t it = 0; take_uniform(0, it, d);) {
                    const int n0 = d.steps0, n1 = d.steps1;
                    wait_in(C::PAIR_FULL + next.at, next.ph);
                    if (n0 > 0) {
                        wait_q(0);
                        scores(0, next, false, n0 == 1);
                    }
                    wait_q(1);
                    scores(1, next, true, n1 == 1);
                    next = next.next();
                    for (int i = 0; i < n1; ++i) {
                        // the next keys, and these values behind them
                        const bool more = i + 1 < n1;
                        const Stage keys = next, vals = more ? next.next() : next;
                        next = vals.next();
                        if (more) wait_in(C::PAIR_FULL + keys.at, keys.ph);
                        wait_in(C::PAIR_FULL + vals.at, vals.ph);
                        clean(ring + vals.at * C::STAGE_BYTES, (d.t0 + i) * BN, BN, d.kv);
                        if (i < n0) values(0, vals, i > 0, false, i + 1 == n0);
                        if (i + 1 < n0) scores(0, keys, false, i + 2 == n0);
                        values(1, vals, i > 0, true, !more);
                        if (more) scores(1, keys, true, i + 2 == n1);
                    }
                }
                if (elect_one()) umma_commit(bar(C::PAIRS_DONE));
                __syncwarp();
            } else if (has_pairs) {  // only follows, so that its wait for the pairs' end is a short one
                Item d;
                for (uint32_t it = 0; take(0, it, d);) {
                }
            }
            if (places[1 + s].b >= 0) {
                if (has_pairs) wait_in(C::PAIRS_DONE, 0);
                const uint32_t own = ring + s * (C::STAGES * C::SLOT_BYTES);
                const int first = s * C::STAGES;
                const uint64_t k_desc = make_smem_desc(own), v_desc = make_mn_desc(own, HN * 128), a = q_desc + (uint64_t)(s * (C::Q_BYTES >> 4));
                const uint32_t s_col = tmem + C::S_COL + 128 * s, o_col = tmem + C::O_COL + D * s;
                uint32_t slot = 0, ph = 0, q_parity = 0, p_parity = 0;
                auto advance = [&]() {
                    if (++slot == C::STAGES) slot = 0, ph ^= 1u;
                };
                Item d;
                for (uint32_t it = 0; take_uniform(1 + s, it, d);) {
                    const int n = d.steps0;
                    wait_in(C::Q_FULL + 2 + s, q_parity), q_parity ^= 1u;
                    for (int i = 0; ok && i < n; ++i) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait_in(C::SLOT_FULL + first + (int)slot, ph);
                            const uint64_t b = k_desc + (uint64_t)(slot * (C::SLOT_BYTES >> 4));
                            if (ok && elect_one()) {
#pragma unroll
                                for (int k = 0; k < D / 16; ++k)
                                    umma_bf16(s_col + HN * h, a + (k / 4) * (BM * 128 >> 4) + (k % 4) * 2, b + (k / 4) * (HN * 128 >> 4) + (k % 4) * 2,
                                              C::IDESC_S_SLOT, k > 0);
                                umma_commit(bar(C::SLOT_EMPTY + first + slot));
                                if (h == 1) umma_commit(bar(C::S_FULL + 2 + s));
                                if (h == 1 && i + 1 == n) umma_commit(bar(C::Q_EMPTY + 2 + s));
                            }
                            __syncwarp();
                            advance();
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            wait_in(C::SLOT_FULL + first + (int)slot, ph);
                            clean(own + slot * C::SLOT_BYTES, (d.t0 + i) * BN + h * HN, HN, d.kv);
                            if (h == 0) {
                                wait_in(C::P_FULL + 2 + s, p_parity), p_parity ^= 1u;
                                tc_fence_after();
                            }
                            const uint64_t b = v_desc + (uint64_t)(slot * (C::SLOT_BYTES >> 4));
                            const uint32_t accumulate = i > 0 || h > 0;
                            if (ok && elect_one()) {
                                umma_bf16_ts(o_col, s_col + 32 * h, b, C::IDESC_O, accumulate);
#pragma unroll
                                for (int k = 1; k < HN / 16; ++k) umma_bf16_ts(o_col, s_col + 32 * h + 8 * k, b + k * (2048 >> 4), C::IDESC_O, 1u);
                                umma_commit(bar(C::SLOT_EMPTY + first + slot));
                                if (h == 1 && i + 1 == n) umma_commit(bar(C::O_FULL + 2 + s));
                            }
                            __syncwarp();
                            advance();
                        }
                    }
                }
            }
            // Every product has ended and every arrival that it owes has been made before the block's memory goes.
            if (elect_one()) umma_commit(bar(C::DONE + s));
            __syncwarp();
            ok = __all_sync(~0u, wait_bar(bar(C::DONE + s), 0)) && ok;
        }
    }
    if (!ok && lane == 0) atomicCAS(&g_device_status, 0, ((70 + warp) << 8) | QB200_ERR_DEVICE_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the pieces of the item that begins at worker x of the first kernel and goes on behind it.  A thread reads the results of several
// workers at a time, so that an item cut over many blocks costs a few latencies and not one per block.  SPREAD, for calls of so few
// requests and heads that an item is cut over hundreds of blocks: a row has a block, a thread an eighth of its pieces (one request of
// 32768 tokens, 8 / 1 heads: 46.7 -> 28.4 us at one step a piece; two of 16384, 12 / 2 heads of 64, four tokens: 64 -> 23; where items have less pieces the
// blocks that it takes cost more than that: one request of 1001 tokens, 16 / 16 heads 13.2 us, 15.4 with SPREAD).
template <int WIDE>
struct Joined {
    float top, l;
    float4 o[WIDE];
};
// Pieces first .. last - 1, AT_ONCE of them read at a time.
template <int D, int WIDE, int AT_ONCE>
__device__ __forceinline__ Joined<WIDE> join_pieces(const Params& p, const float* tail, int first, int last, int row, const int (&at)[WIDE]) {
    const long long slot_floats = (long long)p.slot_rows * (D + 2);
    Joined<WIDE> r;
    r.top = -CUDART_INF_F, r.l = 0;
#pragma unroll
    for (int k = 0; k < WIDE; ++k) r.o[k] = make_float4(0, 0, 0, 0);
    for (int i0 = first; i0 < last; i0 += AT_ONCE) {
        float m[AT_ONCE], s[AT_ONCE];
        float4 x[AT_ONCE][WIDE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j;
            const float* slot = tail + (2ll * i - (i == 0 ? 0 : 1)) * slot_floats;  // the first piece is a tail, the others are heads
            const bool there = i < last;
            m[j] = there ? slot[p.slot_rows * D + row] : -CUDART_INF_F;
            s[j] = there ? slot[p.slot_rows * (D + 1) + row] : 0.f;
#pragma unroll
            for (int k = 0; k < WIDE; ++k) x[j][k] = there ? reinterpret_cast<const float4*>(slot)[at[k]] : make_float4(0, 0, 0, 0);
        }
        float up = r.top;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) up = fmaxf(up, m[j]);
        const float w0 = weight_to(r.top, up);
        r.top = up;
        r.l *= w0;
#pragma unroll
        for (int k = 0; k < WIDE; ++k) r.o[k].x *= w0, r.o[k].y *= w0, r.o[k].z *= w0, r.o[k].w *= w0;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const float w = weight_to(m[j], up);
            r.l += w * s[j];
#pragma unroll
            for (int k = 0; k < WIDE; ++k) r.o[k].x += w * x[j][k].x, r.o[k].y += w * x[j][k].y, r.o[k].z += w * x[j][k].z, r.o[k].w += w * x[j][k].w;
        }
    }
    return r;
}
template <int WIDE>
__device__ __forceinline__ void store_joined(const Joined<WIDE>& r, __nv_bfloat16* dst) {
    const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
#pragma unroll
    for (int k = 0; k < WIDE; ++k)
        *reinterpret_cast<uint2*>(dst + 4 * k) = make_uint2(pack_bf16x2(r.o[k].x * inv, r.o[k].y * inv), pack_bf16x2(r.o[k].z * inv, r.o[k].w * inv));
}

constexpr int kSpreadItems = 4, kSpreadBlocks = 8;  // at most so many rows of the page table times heads; blocks for their rows
template <int D, bool SPREAD>
__global__ void __launch_bounds__(2 * D) paged_attention_join_kernel(const Params p) {
    constexpr int PARTS = 8, MEMBERS = 2 * D / PARTS;  // of the pieces; a row's pieces of four columns
    __shared__ float4 s_o[SPREAD ? PARTS : 1][MEMBERS];
    __shared__ float2 s_ml[SPREAD ? PARTS : 1][MEMBERS];
    wait_for_preceding_grid();
    const int* header = p.headers + blockIdx.x * HEADER;
    const int4 h = *reinterpret_cast<const int4*>(header);
    const int pieces = h.x, start = h.y, hk = h.z, tok0 = h.w, rows = header[4];
    if (pieces == 0) return;
    const float* const tail = p.partial + (2ll * blockIdx.x + 1) * p.slot_rows * (D + 2);
    auto out_of = [&](int row) {
        const int token = row / p.group, head = hk * p.group + (row - token * p.group);
        return p.out + (long long)(start + tok0 + token) * p.o_token + (long long)head * p.o_head;
    };
    if (rows > 32) {  // 32 rows and four pieces of four columns each per warp
        const int chunk = threadIdx.x / 32 * 4;
        for (int row = blockIdx.y * 32 + threadIdx.x % 32; row < rows; row += gridDim.y * 32) {
            const int at[4] = {chunk * p.slot_rows + row, (chunk + 1) * p.slot_rows + row, (chunk + 2) * p.slot_rows + row, (chunk + 3) * p.slot_rows + row};
            store_joined(join_pieces<D, 4, SPREAD ? 4 : 2>(p, tail, 0, pieces, row, at), out_of(row) + 4 * chunk);
        }
    } else if (!SPREAD) {  // eight rows at once
        const int chunk = threadIdx.x / 8;
        for (int row = blockIdx.y * 8 + threadIdx.x % 8; row < rows; row += gridDim.y * 8) {
            const int at[1] = {chunk * p.slot_rows + row};
            store_joined(join_pieces<D, 1, 8>(p, tail, 0, pieces, row, at), out_of(row) + 4 * chunk);
        }
    } else {  // the parts' results in order, too
        const int part = threadIdx.x / MEMBERS, chunk = threadIdx.x % MEMBERS;
        const int share = (pieces + PARTS - 1) / PARTS, first = min(part * share, pieces), last = min(first + share, pieces);
        for (int row = blockIdx.y; row < rows; row += gridDim.y) {
            const int at[1] = {chunk * p.slot_rows + row};
            Joined<1> r = join_pieces<D, 1, 8>(p, tail, first, last, row, at);
            s_o[part][chunk] = r.o[0], s_ml[part][chunk] = make_float2(r.top, r.l);
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int i = 1; i < PARTS; ++i) {
                    const float2 ml = s_ml[i][chunk];
                    const float4 o = s_o[i][chunk];
                    const float up = fmaxf(r.top, ml.x), a = weight_to(r.top, up), b = weight_to(ml.x, up);
                    r.top = up, r.l = r.l * a + ml.y * b;
                    r.o[0].x = r.o[0].x * a + b * o.x, r.o[0].y = r.o[0].y * a + b * o.y, r.o[0].z = r.o[0].z * a + b * o.z, r.o[0].w = r.o[0].w * a + b * o.w;
                }
                store_joined(r, out_of(row) + 4 * chunk);
            }
            __syncthreads();
        }
    }
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

// Rows of a partial result: a stream's, or what the whole call has of one head where that is less.
static int slot_rows_of(int rows, int group) {
    const long long all = ((long long)rows * group + 31) / 32 * 32;
    return (int)(all < BM ? all : BM);
}

static int encode_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                      CUtensorMapL2promotion promotion) {
    EncodeTiledFn fn = get_encode_fn();
    if (fn == nullptr) return QB200_ERR_DRIVER;
    const cuuint32_t unit[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? QB200_OK : QB200_ERR_DRIVER;
}
// The stride of a dimension of one entry is never used, but has to be a valid one.
static cuuint64_t stride_bytes(long long stride, long long entries, int D) { return (cuuint64_t)(entries > 1 ? stride : D) * 2; }

static int encode_page_map(CUtensorMap* map, const void* base, const long long* strides, int num_pages, int page, int heads, int D) {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)num_pages};
    const cuuint64_t st[3] = {stride_bytes(strides[1], page, D), stride_bytes(strides[2], heads, D), stride_bytes(strides[0], num_pages, D)};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page < HN ? page : HN), 1, 1};
    return encode_map(map, base, 4, dims, st, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
static int encode_query_map(CUtensorMap* map, const void* base, const long long* strides, int rows, int heads, int group, int tokens, int D) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t st[2] = {stride_bytes(strides[1], heads, D), stride_bytes(strides[0], rows, D)};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tokens};
    return encode_map(map, base, 3, dims, st, box, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

template <int D>
static int launch(const Params& p, const CUtensorMap& qmap, const CUtensorMap& hqmap, const CUtensorMap& kmap, const CUtensorMap& vmap, int blocks, cudaStream_t stream) {
    static bool prepared[kMaxDevices];  // of the device, once; a second thread that does it again does no harm
    const int dev = current_device();
    if (dev < 0) return QB200_ERR_CUDA;
    if (!prepared[dev]) {
        if (cudaFuncSetAttribute(paged_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM) != cudaSuccess) return QB200_ERR_CUDA;
        prepared[dev] = true;
    }
    paged_attention_kernel<D><<<blocks, kThreads, Cfg<D>::SMEM, stream>>>(p, qmap, hqmap, kmap, vmap);
    const int st = launch_status();
    if (st != QB200_OK) return st;
    cudaLaunchConfig_t cfg = {};
    const bool spread = (long long)p.batch * p.hkv <= kSpreadItems;
    cfg.gridDim = dim3(4 * blocks, spread ? kSpreadBlocks : (p.slot_rows + 63) / 64);  // one wave of blocks where there are more items
    cfg.blockDim = dim3(2 * D);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(spread ? cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<D, true>, p) : cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<D, false>, p));
}

}  // namespace pa

int paged_attention_fetch_and_clear_device_status(int* out) { return fetch_and_clear_device_status(out); }

}  // namespace qb

using namespace qb;

extern "C" int paged_attention_workspace(int rows, int batch, int n_head, int n_kv_head, int head_dim) {
    if (rows <= 0 || batch <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || head_dim <= 0 || head_dim > 128) return 0;
    const long long sms = pa::sm_count();
    return (int)(sms * (8ll * pa::slot_rows_of(rows, n_head / n_kv_head) * (head_dim + 2) * 4 + 4 * pa::HEADER * 4));
}

extern "C" int paged_attention_cuda_bf16(void* out, const long long* out_strides, const void* q, const long long* q_strides,
                                         const void* k_cache, const long long* k_strides, const void* v_cache,
                                         const long long* v_strides, const int* page_table, const int* kv_lens, const int* cu_new,
                                         void* workspace, float scale, int rows, int batch, int width, int n_head, int n_kv_head,
                                         int head_dim, int num_pages, int page_size, cudaStream_t stream) {
    if (rows < 0 || batch < 0 || width < 0 || n_head <= 0 || n_kv_head <= 0 || num_pages < 0 || page_size <= 0 || !(scale >= 0.f)) return QB200_ERR_INVALID_ARGUMENT;
    if (rows == 0 || batch == 0) return QB200_OK;
    if (!out || !out_strides || !q || !q_strides || !k_strides || !v_strides || !kv_lens || !cu_new || !workspace || (width && !page_table) ||
        !k_cache || !v_cache || num_pages == 0)
        return QB200_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || n_head % n_kv_head != 0 || n_head / n_kv_head > pa::BM || (page_size & (page_size - 1)) != 0 ||
        page_size < 16 || page_size > 1024 || (long long)width * page_size > (1ll << 25) || rows > (1 << 29) || batch > (1 << 20) || !aligned16(out) || !aligned16(q) ||
        !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(workspace))
        return QB200_ERR_UNSUPPORTED;
    for (int i = 0; i < 3; ++i)
        if (k_strides[i] % 8 || v_strides[i] % 8 || (i < 2 && (q_strides[i] % 8 || out_strides[i] % 8))) return QB200_ERR_UNSUPPORTED;
    const int group = n_head / n_kv_head, sms = pa::sm_count();
    if (sms == 0) return QB200_ERR_CUDA;
    CUtensorMap qmap, hqmap, kmap, vmap;
    const int tokens = pa::BM / group, half_tokens = pa::BM / 2 / group;  // 0: no tile has so few rows
    int st = pa::encode_query_map(&qmap, q, q_strides, rows, n_head, group, tokens, head_dim);
    if (st == QB200_OK) st = pa::encode_query_map(&hqmap, q, q_strides, rows, n_head, group, half_tokens > 0 ? half_tokens : tokens, head_dim);
    if (st == QB200_OK) st = pa::encode_page_map(&kmap, k_cache, k_strides, num_pages, page_size, n_kv_head, head_dim);
    if (st == QB200_OK) st = pa::encode_page_map(&vmap, v_cache, v_strides, num_pages, page_size, n_kv_head, head_dim);
    if (st != QB200_OK) return st;
    pa::Params p{};
    p.out = static_cast<__nv_bfloat16*>(out);
    p.q = static_cast<const __nv_bfloat16*>(q), p.k = static_cast<const __nv_bfloat16*>(k_cache), p.v = static_cast<const __nv_bfloat16*>(v_cache);
    p.q_token = q_strides[0], p.q_head = q_strides[1], p.k_page = k_strides[0], p.k_token = k_strides[1], p.k_head = k_strides[2];
    p.v_page = v_strides[0], p.v_token = v_strides[1], p.v_head = v_strides[2];
    p.page_table = page_table, p.kv_lens = kv_lens, p.cu = cu_new;
    p.slot_rows = pa::slot_rows_of(rows, group);
    p.partial = static_cast<float*>(workspace);
    p.headers = reinterpret_cast<int*>(p.partial + sms * 8ll * p.slot_rows * (head_dim + 2));
    p.o_token = out_strides[0], p.o_head = out_strides[1];
    p.wide_stores = reinterpret_cast<uintptr_t>(out) % 32 == 0 && p.o_token % 16 == 0 && p.o_head % 16 == 0;
    p.c = fmaxf(scale * 1.4426950408889634f, 1.17549435e-38f);  // above zero: what is masked stays at minus infinity
    p.rows = rows, p.batch = batch, p.width = width, p.hkv = n_kv_head, p.group = group, p.tokens = tokens, p.half_tokens = half_tokens;
    p.num_pages = num_pages, p.page = page_size;
    for (p.page_shift = 0; (1 << p.page_shift) < page_size; ++p.page_shift) {}
    return head_dim == 64 ? pa::launch<64>(p, qmap, hqmap, kmap, vmap, sms, stream) : pa::launch<128>(p, qmap, hqmap, kmap, vmap, sms, stream);
}
