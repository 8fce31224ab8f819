// Attention over packed prompts, causal or not, with grouped heads, on the tcgen05 tensor cores:
//
//     out[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(s q[i, h] . k_j - m_i),   j <= i + (keys - rows) of i's sequence,
//
// in one pass over the keys with a running reference m and sum per row. A CTA takes two tiles of 128 rows, which share the keys and
// values that stream through shared memory, one pair of 128 keys at a time. The rows of a tile are (token, head of a group), all
// query heads of one key head where that fills a tile well, so that short prompts fill tiles and a causal tile spans few tokens.
//
//   warps 0-3, 4-7   softmax of the first, of the second tile: a row per thread. S from TMEM, p back over it (16 bits), the sum in a
//                    register; at the end O from TMEM, divided and stored.
//   warp 8           issues the MMAs: S = Q K^T from shared memory, O += P V with P in TMEM. While one tile's rows are in the softmax
//                    the tensor core works for the other: O += P V of a key tile and S of the next one are issued together, the first reads
//                    the P that the second overwrites, and the tensor core takes them in order.
//   warp 9           TMA: both Q tiles, then keys and values in turn through a ring of stages.
//   warp 10          takes the CTA's next two row tiles from the work that is left, while the present ones are computed.
//   warp 11          takes infinities and NaN out of the values of keys that some rows must not see, in units that are done once more for them.
//
// The reference m only follows the maximum where a weight would pass 2^8 (fp16: 2^14); then the row's O is scaled in TMEM. That is rare, so no
// warps are kept for it. The S barrier of a key tile stands for the completion of all MMAs before it, so O is at rest when its S arrives.
//
// p is rounded to the operands' type for the second product (the tensor core wants one type for both); the sum is taken before
// that, all sums and O are fp32. All waits are bounded; one that runs out sets the status, and the CTA drains and leaves.
//
// A masked key counts 0 * v in a tile product, which is not 0 where v is infinite or NaN. Only the last one to three key tiles of a unit of work hold keys
// that not all of its rows see. Where a row of such a unit comes out infinite or NaN, the unit is done once more, clean: warp 11 makes what is infinite or
// NaN among the values of those keys 0 in shared memory before the product, and gives it back to the rows that see it behind it. What all rows see is left
// to the product. So such a unit takes twice its time, and the others 1 to 2 % for being ready for it (cleaning all of them: 3 to 9 %).
#include <cuda.h>

#include <type_traits>

#include "mf_attention.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using namespace mf::sm100;

constexpr int kTile = 128;  // rows of a tile, keys of a tile
constexpr int kThreads = 384;
constexpr uint32_t kHalf = kTile * 128;  // bytes of 64 columns of a tile
constexpr int kEarly = 64;  // keys whose P is handed over while the others are still computed
// Registers of a softmax thread, which holds a row of S, and of the others: 256 * 216 + 128 * 72 = the 384 * 168 of the launch. 16384 tokens, long loops:
// 200 and 96 1935 us, 216 and 72 1897, 232 and 40 1937.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;

// What the scheduler warp says about a CTA's next two row tiles.
struct Work {
    int q0, rows, t0;   // first query row of the sequence, their number, first token of the tiles
    int k0, keys, n;    // first key, their number, key tiles to go through; n < 0: no more work
    int sure, clean;    // keys that all rows see; whether the values of the others are to be cleaned
    int kvh, h0;
};

template <int D>
struct Shared {
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr uint32_t kTileBytes = (D / 64) * kHalf;
    unsigned char q[2][kTileBytes];
    unsigned char kv[kStages][kTileBytes];
    uint64_t qFull, qEmpty, kvFull[kStages], kvEmpty[kStages], kvRaw[kStages], sFull[2], pFull[2], pRest[2], oFull[2], workFull[2], workEmpty[2];
    uint4 claim;  // the answer to Claim()
    uint64_t claimed, drained;
    Work work[2], late;  // late: done clean, to get back what was taken out
    int odd[2];  // a row of the work came out infinite or NaN
    uint32_t tmem;
    int abortFlag;
};

// The first key tile that has to be cleaned.
__device__ __forceinline__ int CutTile(const Work &w) { return w.clean ? w.sure / kTile : w.n; }

struct Params {
    mf_prefill_attention_args_t a;
    int pack;      // heads in a tile's rows
    int tokens;    // tokens of two tiles: 2 * (128 / pack)
    int wide;      // output rows begin at multiples of 32 bytes: whole sectors are stored
    int headTiles; // kvHeads * group / pack
    int tiles;     // numbers of row tiles, empty ones among them
};

// The largest; NaN if there is one among them.
__device__ __forceinline__ float MaxNan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float MaxNan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t Both(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 Apart(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t Fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t Add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t Mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x for x <= 16 on the FMA pipe, for a share of the weights: the special function unit gives 16 results a cycle and SM, which is as long for a tile
// as its MMAs take at D = 128. x = n + f with n the nearest whole number (W. J. Cody, W. Waite, "Software Manual for the Elementary
// Functions", 1980), 2^f by the polynomial of least relative error on [-1/2, 1/2] among those that are 1 at 0 (linear program; 1.01e-4 of degree 3, 2.9e-6
// of degree 4, below the rounding of p to bf16 and fp16), n added to its exponent. That 1 makes masked weights exactly 0: whatever lies below -127 is
// taken for -127, where the bits of 1 less 127 exponents are none. With a least weight above 0, v of a masked key reaches the row if it is large enough.
// Between -127 and -126 the result lies below 2^-126. NaN comes out as 0: the row's sum knows about it.
template <bool BF16>
__device__ __forceinline__ float2 Exp2Poly(uint64_t x2)
{
    const float2 x = Apart(x2);
    x2 = Both(fmaxf(x.x, -127.0f), fmaxf(x.y, -127.0f));
    const uint64_t r2 = Add2(x2, Both(12582912.0f, 12582912.0f));  // 1.5 * 2^23: n stands in the lowest bits
    const uint64_t f2 = Fma2(Add2(r2, Both(-12582912.0f, -12582912.0f)), Both(-1.0f, -1.0f), x2);
    uint64_t p2;
    if (BF16) {
        p2 = Fma2(Both(0.055008932f, 0.055008932f), f2, Both(0.242210959f, 0.242210959f));
        p2 = Fma2(p2, f2, Both(0.693282927f, 0.693282927f));
    } else {
        p2 = Fma2(Both(0.009582853f, 0.009582853f), f2, Both(0.055906425f, 0.055906425f));
        p2 = Fma2(p2, f2, Both(0.240240986f, 0.240240986f));
        p2 = Fma2(p2, f2, Both(0.693124193f, 0.693124193f));
    }
    p2 = Fma2(p2, f2, Both(1.0f, 1.0f));
    const float2 r = Apart(r2), p = Apart(p2);
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}

// One pair of weights in so many goes to the FMA pipe. A pair takes it as long there (14 cycles of a scheduler, and 8 of the ALU; 16 with degree 4) as on
// the special function unit (16), so the share that pays is small. 8192 tokens, bf16: none 494, an eighth 482, three eighths 537 us; with the
// present split of registers an eighth 513, a quarter 506 us (long loops). fp16, 12 prompts: none 72, an eighth 73, a quarter 76 us.
template <bool BF16>
struct Poly {
    static constexpr int kShare = BF16 ? 4 : 8;
};

template <int REGS>
__device__ __forceinline__ void MoreRegisters()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void FewerRegisters()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Asks for a CTA of this grid that has not been launched yet, in the place of which the caller will work; 16 bytes of answer come to `answer` and are counted on `bar`.
__device__ __forceinline__ void ClaimCta(uint4 *answer, uint64_t *bar)
{
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(SmemAddr(answer)), "r"(SmemAddr(bar))
                 : "memory");
}
// Its blockIdx.x, or -1 if all have been launched.
__device__ __forceinline__ int ClaimedCta(const uint4 *answer)
{
    int x;
    asm volatile(
        "{\n.reg .b128 h;\n.reg .pred p;\n"
        "ld.shared.b128 h, [%1];\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
        "mov.b32 %0, -1;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n}\n"
        : "=r"(x)
        : "r"(SmemAddr(answer))
        : "memory");
    return x;
}

// Some waits last as long as a unit of work, 14 ns a key: a minute is enough for any number of keys.
__device__ __forceinline__ bool Wait(uint64_t *bar, uint32_t parity, volatile int *abortFlag) { return MbarWaitWarp(bar, parity, abortFlag, 60000000000ull); }

// Sequence b's query rows and keys, as far as there are tokens; none where the offsets descend or begin outside.
__device__ __forceinline__ void Extent(const mf_prefill_attention_args_t &a, int b, Work &w)
{
    auto within = [](int first, int next, int all) { return first < 0 || first >= all ? 0 : min(max(next, first), all) - first; };
    w.q0 = a.cuQ[b];
    w.rows = within(w.q0, a.cuQ[b + 1], a.tokensQ);
    w.k0 = a.cuK[b];
    w.keys = within(w.k0, a.cuK[b + 1], a.tokensK);
}

// Row tiles of sequence b have numbers from cuQ[b] / tokens + b on: enough for its rows wherever they begin, some numbers stay empty. Taken from
// the end, as the last tiles of a causal prompt are the longest. Whole warp; false: an empty number.
__device__ __forceinline__ bool Numbered(const Params &p, int number, Work &w)
{
    const mf_prefill_attention_args_t &a = p.a;
    const int lane = threadIdx.x & 31, tile = p.tiles - 1 - number;
    int lo = 0, hi = a.B;  // the last sequence whose first number is not behind `tile`: 32 places at a time
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned low = __ballot_sync(~0u, at < hi && a.cuQ[at] / p.tokens + at <= tile) | 1u;
        const int last = 31 - __clz(low);
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
    }
    Extent(a, lo, w);
    w.t0 = (tile - (w.q0 / p.tokens + lo)) * p.tokens;
    return w.t0 >= 0 && w.t0 < w.rows;
}

// The same for a few sequences, with the row tiles in order of the key tiles that they take, the most first: what is left at the end is small. How many
// row tiles take m key tiles or more follows from a sequence's lengths; the m of a number is found by bisection. A lane has two sequences, the lengths of
// which stay in registers, and divides by multiplying: with lengths loaded and divided for each number a search took 7000 cycles instead of 2300, and short
// prompts, whose row tiles take 8000, waited for it (31 of up to 190 tokens 27.6 against 24.8 us).
constexpr int kRanked = 64;
struct Ranking {
    Work seq[2];
    int tiles[2], most, all;
    uint32_t inverse;  // 2^32 / tokens, rounded up

    __device__ __forceinline__ void Begin(const Params &p)
    {
        const int lane = threadIdx.x & 31;
        inverse = 0xffffffffu / (uint32_t)p.tokens + 1;
        most = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int b = lane * 2 + i;
            seq[i].rows = seq[i].keys = 0;
            if (b < p.a.B) {
                Extent(p.a, b, seq[i]);
            }
            tiles[i] = seq[i].rows > 0 ? Tiles(p, seq[i].rows - 1) + 1 : 0;
            most = max(most, seq[i].keys > 0 ? (seq[i].keys - 1) / kTile + 1 : 0);
        }
        most = __reduce_max_sync(~0u, most);
        all = Count(p, 0);
    }
    // n / tokens, 0 <= n: the product is too high by n / 2^32 < 1/2 at most before it is cut
    __device__ __forceinline__ int Tiles(const Params &p, int n) const
    {
        const uint32_t t = __umulhi((uint32_t)n, inverse);
        return (int)(t * (uint32_t)p.tokens > (uint32_t)n ? t - 1 : t);
    }
    // the first row tile of a sequence that takes m key tiles or more (its number of row tiles, if none does)
    __device__ __forceinline__ int First(const Params &p, int i, int m) const
    {
        if (m <= 0) {
            return 0;
        }
        const int before = (m - 1) * kTile, past = seq[i].keys - seq[i].rows;
        if (seq[i].keys <= before) {
            return tiles[i];
        }
        return p.a.causal ? max(0, min(tiles[i] - 1, Tiles(p, max(before - past, 0)))) : 0;
    }
    __device__ __forceinline__ int Count(const Params &p, int m) const
    {
        return __reduce_add_sync(~0u, max(0, tiles[0] - First(p, 0, m)) + max(0, tiles[1] - First(p, 1, m)));
    }
    // Whole warp; false: an empty number.
    __device__ __forceinline__ bool Find(const Params &p, int number, Work &w) const
    {
        const int lane = threadIdx.x & 31;
        if (number >= all) {
            return false;
        }
        int lo = 0, hi = most + 1;  // Count(lo) > number >= Count(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (Count(p, mid) > number) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        const int from[2] = {First(p, 0, lo), First(p, 1, lo)};
        const int to[2] = {First(p, 0, lo + 1), First(p, 1, lo + 1)};
        int at = number - __reduce_add_sync(~0u, max(0, tiles[0] - to[0]) + max(0, tiles[1] - to[1]));  // among those that take `lo`
        const int mine[2] = {max(0, to[0] - from[0]), max(0, to[1] - from[1])};
        int before = mine[0] + mine[1];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(~0u, before, d);
            before += lane >= d ? y : 0;
        }
        before -= mine[0] + mine[1];
        const int which = at < before + mine[0] ? 0 : 1;
        const unsigned owner = __ballot_sync(~0u, at >= before && at < before + mine[0] + mine[1]);
        const int l = __ffs(owner) - 1;
        at -= before + (which ? mine[0] : 0);
        w.q0 = __shfl_sync(~0u, which ? seq[1].q0 : seq[0].q0, l);
        w.rows = __shfl_sync(~0u, which ? seq[1].rows : seq[0].rows, l);
        w.k0 = __shfl_sync(~0u, which ? seq[1].k0 : seq[0].k0, l);
        w.keys = __shfl_sync(~0u, which ? seq[1].keys : seq[0].keys, l);
        w.t0 = __shfl_sync(~0u, ((which ? from[1] : from[0]) + at) * p.tokens, l);
        return owner != 0 && w.t0 < w.rows;
    }
};

// Whether the low 16 bits are a finite T.
template <typename T>
__device__ __forceinline__ bool Finite(uint32_t x)
{
    constexpr uint32_t kExponent = Bf16<T>::value ? 0x7f80u : 0x7c00u;
    return (x & kExponent) != kExponent;
}

// What is infinite or NaN among the values of the keys from r0 on of a tile in shared memory becomes 0. Whole warp.
template <typename T, int D>
__device__ __noinline__ void Clean(unsigned char *tile, int r0)
{
    for (int c = 0; c < D / 64; c++) {
        uint4 *at = (uint4 *)(tile + c * kHalf);
        for (int i = r0 * 8 + (threadIdx.x & 31); i < kTile * 8; i += 32) {  // 128 bytes to a key
            uint4 x = at[i];
            uint32_t *const word[4] = {&x.x, &x.y, &x.z, &x.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                *word[e] &= (Finite<T>(*word[e]) ? 0xffffu : 0) | (Finite<T>(*word[e] >> 16) ? 0xffff0000u : 0);
            }
            at[i] = x;
        }
    }
    FenceProxyAsyncShared();  // the tensor core reads what was written here
}

// Gives the rows of a unit of work back what Clean() has taken out of values that they see, those of the keys [sure, limit of the row). What is added to an
// element of O is infinite or NaN, so it may as well be added to the result. A lane has two columns at a time, and four rows' loads in flight: with eight the
// kernel has to spill registers, and takes 3 % longer.
template <typename T, int D>
__device__ __noinline__ void Restore(const Params &p, const Work &w)
{
    const mf_prefill_attention_args_t &a = p.a;
    const int lane = threadIdx.x & 31, rows = min(p.tokens, w.rows - w.t0) * p.pack, past = w.keys - w.rows + w.t0 + 1;
    const int see = a.causal ? min(p.tokens, w.rows - w.t0) + past - 1 : w.keys;
    for (int turn = 0; turn < 3 * (D / 64); turn++) {
        const int kind = turn % 3, c = turn / 3 * 64 + lane * 2;
        const float more = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
        int first[2] = {see, see};  // the first key where each column is that
        const T *v = (const T *)a.v + (size_t)w.k0 * a.vStride[0] + (size_t)w.kvh * a.vStride[1] + c;
#pragma unroll 4
        for (int j = see - 1; j >= w.sure; j--) {
            const float2 x = Unpack2<T>(*(const uint32_t *)(v + j * a.vStride[0]));
            first[0] = kind == 0 ? (x.x != x.x ? j : first[0]) : x.x == more ? j : first[0];
            first[1] = kind == 0 ? (x.y != x.y ? j : first[1]) : x.y == more ? j : first[1];
        }
        const int least = min(first[0], first[1]);
        if (__all_sync(~0u, least == see)) {
            continue;
        }
        T *out = (T *)a.out + ((size_t)w.q0 + w.t0) * a.outStride[0] + (size_t)w.h0 * a.outStride[1] + c;
        constexpr int kAhead = 4;
        for (int r0 = 0; r0 < rows; r0 += kAhead) {
            uint32_t was[kAhead];
#pragma unroll
            for (int store = 0; store < 2; store++) {
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const int t = (r0 + u) / p.pack, limit = r0 + u >= rows ? least : a.causal ? min(w.keys, t + past) : w.keys;
                    uint32_t *const at = (uint32_t *)(out + t * a.outStride[0] + (r0 + u) % p.pack * a.outStride[1]);
                    if (limit > least) {
                        if (store) {
                            const float2 y = Unpack2<T>(was[u]);
                            *at = Pack2<T>(limit > first[0] ? y.x + more : y.x, limit > first[1] ? y.y + more : y.y);
                        } else {
                            was[u] = *at;
                        }
                    }
                }
            }
        }
    }
}

// A warp's view of the work list: the next two row tiles, or false at its end.
template <int D>
struct Worker {
    int k{0};
    __device__ __forceinline__ bool Next(Shared<D> &s, volatile int *abortFlag, Work &w)
    {
        if (!Wait(&s.workFull[k & 1], (k >> 1) & 1, abortFlag)) {
            return false;
        }
        w = s.work[k & 1];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            MbarArrive(&s.workEmpty[k & 1]);
        }
        k++;
        return w.n >= 0;
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
mf_prefill_attention_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                            const __grid_constant__ Params p)
{
    using X = Shared<D>;
    constexpr bool kBf16 = Bf16<T>::value;
    extern __shared__ unsigned char smemRaw[];
    X &s = *reinterpret_cast<X *>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
    const mf_prefill_attention_args_t &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.tokens / 2;

    if (threadIdx.x == 0) {
        MbarInit(&s.qFull, 1);
        MbarInit(&s.qEmpty, 1);
        for (int i = 0; i < X::kStages; i++) {
            MbarInit(&s.kvFull[i], 1);
            MbarInit(&s.kvEmpty[i], 1);
            MbarInit(&s.kvRaw[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            MbarInit(&s.sFull[i], 1);
            MbarInit(&s.pFull[i], 4);
            MbarInit(&s.pRest[i], 4);
            MbarInit(&s.oFull[i], 1);
            MbarInit(&s.workFull[i], 1);
            MbarInit(&s.workEmpty[i], 11);
            s.odd[i] = 0;
        }
        MbarInit(&s.claimed, 1);
        MbarInit(&s.drained, 1);
        s.abortFlag = 0;
        MbarInitFence();
        TmaPrefetchDesc(&mapQ);
        TmaPrefetchDesc(&mapK);
        TmaPrefetchDesc(&mapV);
    }
    if (warp == 8) {
        TmemAlloc(&s.tmem, 512);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = s.tmem;
    volatile int *abortFlag = &s.abortFlag;
    constexpr uint32_t kO = 2 * kTile;  // TMEM columns: S (and P) of the two tiles, then O
    GridDependency();  // what stands above ran under the end of the kernel before

    if (warp >= 8) {
        FewerRegisters<kOtherRegs>();
        if (warp == 10) {
            // ------------------------------------------------------------------ scheduler
            // Each unit of work is a CTA of the grid; a CTA that runs takes the next one that has not been launched yet when it begins with the one before.
            Ranking ranking;
            if (a.B <= kRanked) {
                ranking.Begin(p);
            }
            const Work none = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            int k = 0, unit = (int)blockIdx.x;
            // Hands a work out and waits until all warps have taken it: so the other place is free, and they are done with the one before, of which it is known
            // now whether it came out finite.
            bool ok = true, odd = false;
            auto put = [&](const Work &w) {
                if (ok) {
                    if (lane == 0) {
                        s.work[k & 1] = w;
                        s.odd[k & 1] = 0;
                        MbarArrive(&s.workFull[k & 1]);
                    }
                    ok = Wait(&s.workEmpty[k & 1], (k >> 1) & 1, abortFlag);
                    k++;
                    odd = ok && __shfl_sync(~0u, s.odd[k & 1], 0) != 0;
                }
            };
            for (uint32_t claims = 0; ok; claims++) {
                const bool end = unit < 0;
                const int number = unit / p.headTiles, ht = unit - number * p.headTiles;
                Work w = none;
                const bool there = !end && (a.B <= kRanked ? ranking.Find(p, number, w) : Numbered(p, number, w));
                if (there) {
                    const int see = a.causal ? min(w.keys, min(w.rows, w.t0 + p.tokens) + w.keys - w.rows) : w.keys;
                    w.n = see > 0 ? (see - 1) / kTile + 1 : 0;
                    w.sure = a.causal ? max(0, min(w.keys, w.t0 + w.keys - w.rows + 1)) : w.keys;
                    w.clean = 0;
                    const int perKv = a.group / p.pack;
                    w.kvh = ht / perKv;
                    w.h0 = w.kvh * a.group + (ht % perKv) * p.pack;
                }
                if (there || end) {  // at the end one without rows: then it is known of the last one, too
                    put(w);
                    if (odd) {
                        Work again = s.work[k & 1], last = s.work[(k + 1) & 1];  // the one before w, and w
                        __syncwarp();
                        for (bool more = true; ok && more && !again.clean && again.sure / kTile < again.n; again = last, last = none) {
                            again.clean = 1;
                            put(again);
                            more = odd;  // of `last`
                            put(none);   // when the warps have taken what comes behind this one, they are done with the clean one
                        }
                    }
                }
                if (end) {
                    if (lane == 0 && ok) {
                        s.work[k & 1].n = -1;
                        MbarArrive(&s.workFull[k & 1]);
                    }
                    break;
                }
                if (!ok) {
                    break;
                }
                if (lane == 0) {
                    MbarExpectTx(&s.claimed, 16);
                    ClaimCta(&s.claim, &s.claimed);
                }
                int own = 0;  // the answer is waited for even if the CTA gives up: it is written to its shared memory
                if (!Wait(&s.claimed, claims & 1, &own)) {
                    *abortFlag = 1;
                    break;
                }
                unit = ClaimedCta(&s.claim);
                FenceProxyAsyncShared();
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------------ TMA producer
            const bool elected = ElectOne();
            Worker<D> worker;
            Work w;
            uint32_t st = 0, ph = 0, qPh = 0, raw = 0, rawPh = 0;
            long long issued = 0;
            bool ok = true, qOpen = false;
            while (ok && worker.Next(s, abortFlag, w)) {
                if (w.n == 0) {
                    continue;
                }
                const bool two = w.t0 + half < w.rows;
                ok = Wait(&s.qEmpty, qPh ^ 1, abortFlag);
                if (!ok) {
                    break;
                }
                if (elected) {
                    MbarExpectTx(&s.qFull, (two ? 2 : 1) * (D / 64) * 128 * p.pack * half);
                    for (int i = 0; i < (two ? 2 : 1); i++) {
                        for (int c = 0; c < D / 64; c++) {
                            TmaLoad3D(s.q[i] + c * kHalf, &mapQ, &s.qFull, c * 64, w.h0, w.q0 + w.t0 + i * half);
                        }
                    }
                }
                qOpen = true;
                qPh ^= 1;
                const int cut = CutTile(w);
                for (int i = 0; i < 2 * w.n; i++) {
                    ok = Wait(&s.kvEmpty[st], ph ^ 1, abortFlag);
                    if (!ok) {
                        break;
                    }
                    const bool dirty = (i & 1) != 0 && (i >> 1) >= cut;  // goes to warp 11 first
                    uint64_t *const full = dirty ? &s.kvRaw[st] : &s.kvFull[st];
                    if (elected) {
                        MbarExpectTx(full, X::kTileBytes);
                        for (int c = 0; c < D / 64; c++) {
                            TmaLoad3D(s.kv[st] + c * kHalf, i & 1 ? &mapV : &mapK, full, c * 64, w.kvh, w.k0 + (i >> 1) * kTile);
                        }
                    }
                    raw = (raw & ~(1u << st)) | (dirty ? 1u << st : 0);
                    rawPh ^= dirty ? 1u << st : 0;
                    issued++;
                    if (++st == X::kStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
            if (*abortFlag != 0) {  // nothing may land in the shared memory of a CTA that has left
                int own = 0;
                if (qOpen) {
                    MbarWaitBounded(&s.qFull, qPh ^ 1, &own);
                }
                for (long long i = issued > X::kStages ? issued - X::kStages : 0; i < issued; i++) {
                    const uint32_t at = (uint32_t)(i % X::kStages);
                    if (raw >> at & 1) {
                        MbarWaitBounded(&s.kvRaw[at], (rawPh >> at & 1) ^ 1, &own);
                    } else {
                        MbarWaitBounded(&s.kvFull[at], (uint32_t)(i / X::kStages) & 1, &own);
                    }
                }
            }
        } else if (warp == 11) {
            // ------------------------------------------------------------------ values that are not finite
            // Such a tile's arrival is counted on kvRaw, which has a phase for each time that its stage holds one; kvFull is completed here, when it is clean. So
            // the MMA warp knows nothing of this: with one more barrier in its loop, never waited for, prompts took 1 to 2 % longer.
            Worker<D> worker;
            Work taken;
            uint32_t st = 0, rawPh = 0;
            int lateAt = -2;
            auto move = [&](uint32_t by) { st = (st + by) % X::kStages; };
            bool ok = true;
            for (bool more = true; more;) {
                more = worker.Next(s, abortFlag, taken);
                if (*abortFlag != 0) {
                    break;
                }
                if (worker.k == lateAt + 2) {  // the other warps have taken the one behind it, so its rows are stored
                    Restore<T, D>(p, s.late);
                }
                if (!more) {
                    break;
                }
                const Work &w = s.work[(worker.k - 1) & 1];  // stays until this warp has taken the next one
                const int cut = CutTile(w);
                move(2 * cut);
                for (int j = cut; j < w.n; j++) {
                    move(1);
                    ok = Wait(&s.kvRaw[st], rawPh >> st & 1, abortFlag);
                    if (!ok) {
                        break;
                    }
                    rawPh ^= 1u << st;
                    Clean<T, D>(s.kv[st], max(0, w.sure - j * kTile));
                    __syncwarp();
                    if (lane == 0) {
                        MbarArrive(&s.kvFull[st]);
                    }
                    move(1);
                }
                if (w.clean) {
                    if (lane == 0) {
                        s.late = w;
                    }
                    __syncwarp();
                    lateAt = worker.k;
                }
            }
        } else if (warp == 8) {
            // ------------------------------------------------------------------ MMA issuer
            // Everything that the loops and operands go by comes out of a warp reduction: the compiler then knows that it is the same in all lanes and
            // keeps descriptors in uniform registers. One warp for both tiles, so that the S of one is complete before that of the other is begun: issued by
            // a warp for each, they took turns and were both late (chunks of prompts 154 -> 147 us, 16384 tokens 1963 -> 1935).
            const bool elected = ElectOne();
            const uint32_t base = __reduce_or_sync(~0u, tmem);
            const uint64_t qDesc = SmemDescSw128(SmemAddr(s.q[0])), kDesc = SmemDescSw128(SmemAddr(s.kv[0])),
                           vDesc = SmemDescSw128Transposed(SmemAddr(s.kv[0]), kHalf);
            constexpr uint32_t iS = InstrDescF16(kTile, kTile, kBf16, false), iO = InstrDescF16(kTile, D, kBf16, true);
            auto scores = [&](int i, uint32_t stage) {  // S of tile i
                const uint64_t k0 = kDesc + stage * (X::kTileBytes >> 4), q0 = qDesc + i * (X::kTileBytes >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t off = (k / 4) * (kHalf >> 4) + (k % 4) * 2;
                    MmaF16(base + i * kTile, q0 + off, k0 + off, iS, k > 0);
                }
            };
            auto values = [&](int i, uint32_t stage, bool more, int k0, int k1) {  // O of tile i, keys [k0, k1)
                const uint64_t v0 = vDesc + stage * (X::kTileBytes >> 4);
#pragma unroll
                for (int k = k0 / 16; k < k1 / 16; k++) {
                    MmaF16Tmem(base + kO + i * D, base + i * kTile + k * 8, v0 + k * 128, iO, more || k > 0);
                }
            };
            Worker<D> worker;
            Work w;
            uint32_t st = 0, ph = 0, qPh = 0, pPh[2] = {0, 0};
            auto step = [&]() {
                if (++st == X::kStages) {
                    st = 0;
                    ph ^= 1;
                }
            };
            bool ok = true;
            while (ok && __any_sync(~0u, worker.Next(s, abortFlag, w))) {
                const int n = __reduce_max_sync(~0u, w.n), both = __reduce_max_sync(~0u, w.t0 + half < w.rows ? 2 : 1);
                if (n == 0) {
                    continue;
                }
                ok = Wait(&s.qFull, qPh, abortFlag) && Wait(&s.kvFull[st], ph, abortFlag);
                qPh ^= 1;
                if (!ok) {
                    break;
                }
                TcFenceAfter();
                if (elected) {
                    scores(0, st);
                    MmaCommit(&s.sFull[0]);
                    if (both == 2) {
                        scores(1, st);
                        MmaCommit(&s.sFull[1]);
                    }
                    MmaCommit(&s.kvEmpty[st]);
                    if (n == 1) {
                        MmaCommit(&s.qEmpty);
                    }
                }
                step();
                for (int j = 0; ok && j < n; j++) {
                    const uint32_t v = st, vPh = ph;
                    step();
                    const uint32_t k = st, kPh = ph;
                    const bool next = j + 1 < n;
                    if (next) {
                        step();
                    }
                    ok = Wait(&s.kvFull[v], vPh, abortFlag) && (!next || Wait(&s.kvFull[k], kPh, abortFlag));
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (!ok || i >= both) {
                            break;
                        }
                        ok = Wait(&s.pFull[i], pPh[i], abortFlag);
                        if (!ok) {
                            break;
                        }
                        TcFenceAfter();
                        if (elected) {
                            values(i, v, j > 0, 0, kEarly);
                        }
                        ok = Wait(&s.pRest[i], pPh[i], abortFlag);
                        if (!ok) {
                            break;
                        }
                        pPh[i] ^= 1;
                        TcFenceAfter();
                        if (elected) {
                            values(i, v, true, kEarly, kTile);
                            if (next) {
                                scores(i, k);
                                MmaCommit(&s.sFull[i]);
                                if (i + 1 == both) {
                                    MmaCommit(&s.kvEmpty[k]);
                                    if (j + 2 == n) {
                                        MmaCommit(&s.qEmpty);
                                    }
                                }
                            } else {
                                MmaCommit(&s.oFull[i]);
                            }
                            if (i + 1 == both) {
                                MmaCommit(&s.kvEmpty[v]);
                            }
                        }
                    }
                }
            }
        }
    } else {
        // ---------------------------------------------------------------------- softmax
        MoreRegisters<kSoftmaxRegs>();
        const int i = warp >> 2;  // the tile
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, sAt = tmem + lanes + i * kTile, oAt = tmem + lanes + kO + i * D;
        const float factor = a.scale * kLog2e, lift = Weights<T>::kLift / factor;
        float top = -INFINITY, sum = 0;
        // One key tile. CUT: the row sees its first `left` columns only, no row of the warp sees any from `cols` on.
        auto tile = [&](auto cut, bool first, int left, int cols) {
            constexpr bool kCut = decltype(cut)::value;
            float x[kTile];
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                TmemLd32Issue(sAt + c, x + c);
            }
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                TmemLdWait32(x + c);
            }
            if (kCut) {
#pragma unroll
                for (int c = 0; c < kTile; c++) {
                    x[c] = c < left ? x[c] : -INFINITY;
                }
            }
            float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int c = 4; c < kTile - 4; c += 8) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    m[e] = MaxNan(m[e], x[c + e], x[c + 4 + e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                m[e] = MaxNan(m[e], x[kTile - 4 + e]);
            }
            const float best = MaxNan(MaxNan(m[0], m[1]), m[2], m[3]);
            sum = best < INFINITY ? sum : NAN;  // a logit that is NaN or infinite: so is the row, whatever its weights come out as
            const bool grown = (best - top) * factor > Weights<T>::kSlack;
            if (__any_sync(~0u, grown)) {
                const float shrink = grown ? Exp2((top - best + lift) * factor) : 1.0f;
                top = grown ? best - lift : top;
                sum *= shrink;
                if (!first) {
#pragma unroll
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        TmemLd16Issue(oAt + c, o);
                        TmemLdWait16(o);
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            o[e] *= shrink;
                        }
                        TmemSt16(oAt + c, (const uint32_t *)o);
                    }
                }
            }
            const float from = top == -INFINITY ? 0.0f : -top * factor;
            const uint64_t factor2 = Both(factor, factor), from2 = Both(from, from);
            uint64_t part[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                uint32_t w16[16];
                if (!kCut || c < cols) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint64_t y = Fma2(Both(x[c + 2 * e], x[c + 2 * e + 1]), factor2, from2);
                        float2 u;
                        if (e % Poly<kBf16>::kShare == 0) {
                            u = Exp2Poly<kBf16>(y);
                        } else {
                            u = Apart(y);
                            u = make_float2(Exp2(u.x), Exp2(u.y));
                        }
                        part[e & 1] = Add2(part[e & 1], Both(u.x, u.y));
                        w16[e] = Pack2<T>(u.x, u.y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        w16[e] = 0;
                    }
                }
                TmemSt16(sAt + c / 2, w16);
                if (c + 32 == kEarly || c + 32 == kTile) {
                    TmemStWait();
                    TcFenceBefore();
                    __syncwarp();
                    if (lane == 0) {
                        MbarArrive(c + 32 == kEarly ? &s.pFull[i] : &s.pRest[i]);
                    }
                }
            }
            const float2 both = Apart(Add2(part[0], part[1]));
            sum += both.x + both.y;
        };
        // rows that the packing leaves over hold anything, and nobody looks at them
        const int rowToken = i * half + row / p.pack, rowHead = row % p.pack;
        const bool filled = row < p.pack * half;
        Worker<D> worker;
        Work w;
        uint32_t sPh = 0, oPh = 0;
        bool ok = true;
        while (ok && worker.Next(s, abortFlag, w)) {
            if (w.t0 + i * half >= w.rows) {
                continue;
            }
            const int token = w.t0 + rowToken, past = w.keys - w.rows, head = w.h0 + rowHead;
            const bool valid = filled && token < w.rows;
            const int limit = a.causal && valid ? min(w.keys, token + past + 1) : w.keys;  // keys that the row sees
            const int sure = __reduce_min_sync(~0u, limit), most = __reduce_max_sync(~0u, valid ? limit : 0);
            top = -INFINITY;
            sum = 0;
            for (int j = 0; j < w.n; j++) {
                if (!Wait(&s.sFull[i], sPh, abortFlag)) {
                    ok = false;
                    break;
                }
                sPh ^= 1;
                TcFenceAfter();
                if ((j + 1) * kTile <= sure) {
                    tile(std::false_type{}, j == 0, kTile, kTile);
                } else {
                    tile(std::true_type{}, j == 0, limit - j * kTile, most - j * kTile);
                }
            }
            if (!ok || (w.n > 0 && !Wait(&s.oFull[i], oPh, abortFlag))) {
                break;
            }
            oPh ^= w.n > 0 ? 1 : 0;
            TcFenceAfter();
            // ---- O / sum; the sum of a row that saw no key is 0
            const float scale = sum != 0 ? 1.0f / sum : 0.0f;
            const uint64_t scale2 = Both(scale, scale);
            T *out = (T *)a.out + ((size_t)w.q0 + token) * a.outStride[0] + (size_t)head * a.outStride[1];
            uint64_t odd = 0;  // stays 0 as long as what is added is 0 times something finite
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = 0;
                }
                if (w.n > 0) {
                    TmemLd32Issue(oAt + c, o);
                    TmemLdWait32(o);
                }
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                    uint32_t pk[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint64_t y = Both(o[h + 2 * e], o[h + 2 * e + 1]);
                        odd = Fma2(y, 0, odd);
                        const float2 z = Apart(Mul2(y, scale2));
                        pk[e] = Pack2<T>(z.x, z.y);
                    }
                    if (valid) {
                        if (p.wide) {
                            StGlobal32B(out + c + h, pk);
                        } else {
                            *(uint4 *)(out + c + h) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                            *(uint4 *)(out + c + h + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
                        }
                    }
                }
            }
            const float2 any = Apart(odd);
            if (!(any.x + any.y == 0.0f) && valid) {
                s.odd[(worker.k - 1) & 1] = 1;
            }
            if (a.lse != nullptr && valid) {
                a.lse[((size_t)w.q0 + token) * a.kvHeads * a.group + head] = top * factor * kLn2 + logf(sum);
            }
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (s.abortFlag != 0 && threadIdx.x == 0 && a.status != nullptr) {
        atomicCAS(a.status, 0, MF_K_GEMM_PIPELINE_EXPIRED);
    }
    if (warp == 8) {
        TcFenceAfter();
        if (s.abortFlag != 0) {  // products that are still under way read and write what is given back here
            int own = 0;
            if (ElectOne()) {
                MmaCommit(&s.drained);
            }
            __syncwarp();
            Wait(&s.drained, 0, &own);
            TcFenceAfter();
        }
        TmemDealloc(tmem, 512);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn GetEncodeTiled()
{
    static EncodeTiledFn fn = []() -> EncodeTiledFn {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) != cudaSuccess || st != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// [tokens][heads][D] with strides in elements; boxes of 64 columns, `boxHeads` heads, `boxTokens` tokens. What lies outside reads as zeros.
bool MakeMap(CUtensorMap *m, const void *base, bool bf16, int D, uint64_t heads, uint64_t tokens, const long long *stride, uint32_t boxHeads, uint32_t boxTokens)
{
    EncodeTiledFn enc = GetEncodeTiled();
    if (enc == nullptr) {
        return false;
    }
    // a dimension of one entry has no stride of its own
    const uint64_t headStride = heads > 1 ? (uint64_t)stride[1] * 2 : (uint64_t)D * 2, tokenStride = tokens > 1 ? (uint64_t)stride[0] * 2 : heads * headStride;
    cuuint64_t dims[3] = {(cuuint64_t)D, heads, tokens}, strides[2] = {headStride, tokenStride};
    cuuint32_t box[3] = {64, boxHeads, boxTokens}, one[3] = {1, 1, 1};
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
int Launch(const mf_prefill_attention_args_t &a, cudaStream_t stream)
{
    Params p;
    p.a = a;
    // as many heads of a group as fill tiles of whole tokens to 15/16 at least, and divide the group
    for (p.pack = a.group < kTile ? a.group : kTile; a.group % p.pack != 0 || kTile / p.pack * p.pack < kTile - kTile / 16; p.pack--) {
    }
    p.tokens = 2 * (kTile / p.pack);
    p.wide = ((uintptr_t)a.out | (uint64_t)a.outStride[0] * sizeof(T) | (uint64_t)a.outStride[1] * sizeof(T)) % 32 == 0;
    p.headTiles = a.kvHeads * a.group / p.pack;
    p.tiles = a.tokensQ / p.tokens + a.B;
    const long long units = (long long)p.tiles * p.headTiles;
    if (units > 0x7fffffffll) {
        return MF_K_TOO_LARGE;
    }
    const unsigned ctas = (unsigned)units;
    CUtensorMap q, k, v;
    constexpr bool kBf16 = Bf16<T>::value;
    // without keys their maps are never used, but have to describe something
    const bool none = a.tokensK == 0;
    if (!MakeMap(&q, a.q, kBf16, D, (uint64_t)a.kvHeads * a.group, a.tokensQ, a.qStride, p.pack, kTile / p.pack) ||
        !MakeMap(&k, none ? a.q : a.k, kBf16, D, none ? 1 : a.kvHeads, none ? 1 : a.tokensK, a.kStride, 1, kTile) ||
        !MakeMap(&v, none ? a.q : a.v, kBf16, D, none ? 1 : a.kvHeads, none ? 1 : a.tokensK, a.vStride, 1, kTile)) {
        return MF_K_INVALID;
    }
    const size_t smem = sizeof(Shared<D>) + 1024;
    if (!mf::AllowSmem<mf_prefill_attention_kernel<T, D>>(smem) ||
        LaunchDependent(mf_prefill_attention_kernel<T, D>, ctas, kThreads, smem, stream, q, k, v, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    return MF_K_OK;
}

}  // namespace

extern "C" int mf_k_prefill_attention(const mf_prefill_attention_args_t *args, int D, int type, mf_stream_t stream)
{
    if (args == nullptr || args->B < 0 || args->kvHeads <= 0 || args->group <= 0 || args->tokensQ < 0 || args->tokensK < 0 || (D != 64 && D != 128) ||
        (type != MF_K_BF16 && type != MF_K_FP16) || !(args->scale > 0)) {
        return MF_K_INVALID;
    }
    if (args->B == 0 || args->tokensQ == 0) {
        return MF_K_OK;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == MF_K_BF16) {
        return D == 64 ? Launch<__nv_bfloat16, 64>(*args, s) : Launch<__nv_bfloat16, 128>(*args, s);
    }
    return D == 64 ? Launch<__half, 64>(*args, s) : Launch<__half, 128>(*args, s);
}
