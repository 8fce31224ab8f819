// Attention over packed prompts, causal or not, with grouped heads, on the tcgen05 tensor cores:
//
//     out[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(s q[i, h] . k_j - m_i),   j <= i + (keys - rows) of i's sequence,
//
// in one pass over the keys with a running reference m and sum per row. A CTA takes two tiles of 128 rows, which share the keys and
// values that stream through shared memory, one pair of 128 keys at a time. The rows of a tile are (token, head of a group): as many
// query heads of one key head as there are in the largest power of two that divides the group, so that short prompts fill tiles and a
// causal tile spans few tokens.
//
//   warps 0-3, 4-7   softmax of the first, of the second tile: a row per thread. S from TMEM, p back over it (16 bits), the sum in a
//                    register; at the end O from TMEM, divided and stored.
//   warp 8           issues the MMAs: S = Q K^T from shared memory, O += P V with P in TMEM. While one tile's rows are in the softmax
//                    the tensor core works for the other: O += P V of a key tile and S of the next one are issued together, the first reads
//                    the P that the second overwrites, and the tensor core takes them in order.
//   warp 9           TMA: both Q tiles, then keys and values in turn through a ring of stages.
//
// The reference m only follows the maximum where that has grown by more than 2^8 since (p stays below 256, sums far below
// overflow); then the row's O is scaled in TMEM. That is rare, so no warps are kept for it. The S barrier of a key tile stands for the
// completion of all MMAs before it, so O is at rest when its S arrives.
//
// p is rounded to the operands' type for the second product (the tensor core wants one type for both); the sum is taken before that, all
// sums and O are fp32. A masked key counts 0 * v in a tile product, which is not 0 where v is infinite or NaN: a row whose result is not finite
// is computed again key by key. All waits are bounded; one that runs out sets the status, and the CTA drains and leaves.
#include <cuda.h>

#include "mf_attention.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using namespace mf::sm100;

constexpr int kTile = 128;  // rows of a tile, keys of a tile
constexpr int kThreads = 320;
constexpr uint32_t kHalf = kTile * 128;  // bytes of 64 columns of a tile
constexpr float kSlack = 8.0f;           // powers of two by which the reference may lag behind the maximum

template <int D>
struct Shared {
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr uint32_t kTileBytes = (D / 64) * kHalf;
    unsigned char q[2][kTileBytes];
    unsigned char kv[kStages][kTileBytes];
    uint64_t qFull, kvFull[kStages], kvEmpty[kStages], sFull[2], pFull[2], oFull[2];
    uint32_t tmem;
    int abortFlag;
};

struct Params {
    mf_prefill_attention_args_t a;
    int pack;      // heads in a tile's rows
    int tokens;    // tokens of a CTA: 256 / pack
    int headTiles; // kvHeads * group / pack
    int tiles;     // numbers of row tiles, empty ones among them
};

__device__ __forceinline__ float Max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

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
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    GridDependency();

    // Row tiles of sequence b have numbers from cuQ[b] / tokens + b on: enough for its rows wherever they begin, some numbers stay empty. The
    // last tiles of a causal prompt are the longest, so numbers are handed out from the end.
    const int tile = p.tiles - 1 - blockIdx.x / p.headTiles, ht = blockIdx.x % p.headTiles;
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (a.cuQ[mid] / p.tokens + mid <= tile ? lo : hi) = mid;
    }
    const int q0 = a.cuQ[lo], rows = min(a.cuQ[lo + 1], a.tokensQ) - q0, t0 = (tile - (q0 / p.tokens + lo)) * p.tokens;
    if (q0 < 0 || t0 < 0 || t0 >= rows) {
        return;
    }
    const int k0 = a.cuK[lo], keys = k0 < 0 ? 0 : min(a.cuK[lo + 1], a.tokensK) - k0, past = keys - rows;
    const int perKv = a.group / p.pack, kvh = ht / perKv, h0 = kvh * a.group + (ht % perKv) * p.pack;
    const int last = min(rows, t0 + p.tokens);  // token behind the CTA's last one
    const int see = a.causal ? min(keys, last + past) : keys, n = see > 0 ? (see + kTile - 1) / kTile : 0;
    const int half = p.tokens / 2;
    const bool two = t0 + half < rows;

    if (threadIdx.x == 0) {
        MbarInit(&s.qFull, 1);
        for (int i = 0; i < X::kStages; i++) {
            MbarInit(&s.kvFull[i], 1);
            MbarInit(&s.kvEmpty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            MbarInit(&s.sFull[i], 1);
            MbarInit(&s.pFull[i], 4);
            MbarInit(&s.oFull[i], 1);
        }
        s.abortFlag = 0;
        MbarInitFence();
    }
    if (warp == 8) {
        TmemAlloc(&s.tmem, 512);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = s.tmem;
    volatile int *abortFlag = &s.abortFlag;
    // TMEM columns: S (and P) of the two tiles, then O
    constexpr uint32_t kO = 2 * kTile;

    if (warp == 9) {
        const bool elected = ElectOne();
        if (n > 0 && elected) {
            MbarExpectTx(&s.qFull, (two ? 2 : 1) * X::kTileBytes);
            for (int i = 0; i < (two ? 2 : 1); i++) {
                for (int c = 0; c < D / 64; c++) {
                    TmaLoad3D(s.q[i] + c * kHalf, &mapQ, &s.qFull, c * 64, h0, q0 + t0 + i * half);
                }
            }
        }
        uint32_t st = 0, ph = 0;
        int issued = 0;
        for (int i = 0; i < 2 * n; i++) {
            if (!MbarWaitWarp(&s.kvEmpty[st], ph ^ 1, abortFlag)) {
                break;
            }
            if (elected) {
                MbarExpectTx(&s.kvFull[st], X::kTileBytes);
                for (int c = 0; c < D / 64; c++) {
                    TmaLoad3D(s.kv[st] + c * kHalf, i & 1 ? &mapV : &mapK, &s.kvFull[st], c * 64, kvh, k0 + (i >> 1) * kTile);
                }
            }
            issued++;
            if (++st == X::kStages) {
                st = 0;
                ph ^= 1;
            }
        }
        if (*abortFlag != 0 && n > 0) {  // nothing may land in the shared memory of a CTA that has left
            int own = 0;
            MbarWaitBounded(&s.qFull, 0, &own);
            for (int i = max(0, issued - X::kStages); i < issued; i++) {
                MbarWaitBounded(&s.kvFull[i % X::kStages], (i / X::kStages) & 1, &own);
            }
        }
    } else if (warp == 8) {
        const bool elected = ElectOne();
        const uint32_t base = __reduce_or_sync(~0u, tmem);
        const uint64_t qDesc = SmemDescSw128(SmemAddr(s.q[0])), kDesc = SmemDescSw128(SmemAddr(s.kv[0])), vDesc = SmemDescSw128Transposed(SmemAddr(s.kv[0]), kHalf);
        constexpr uint32_t iS = InstrDescF16(kTile, kTile, kBf16, false), iO = InstrDescF16(kTile, D, kBf16, true);
        auto scores = [&](int i, uint32_t stage) {  // S of tile i
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                const uint32_t off = (k / 4) * (kHalf >> 4) + (k % 4) * 2;
                MmaF16(base + i * kTile, qDesc + i * (X::kTileBytes >> 4) + off, kDesc + stage * (X::kTileBytes >> 4) + off, iS, k > 0);
            }
        };
        auto values = [&](int i, uint32_t stage, bool more) {  // O of tile i
#pragma unroll
            for (int k = 0; k < kTile / 16; k++) {
                MmaF16Tmem(base + kO + i * D, base + i * kTile + k * 8, vDesc + stage * (X::kTileBytes >> 4) + k * 128, iO, more || k > 0);
            }
        };
        uint32_t st = 0, ph = 0;
        auto step = [&]() {
            if (++st == X::kStages) {
                st = 0;
                ph ^= 1;
            }
        };
        bool ok = n > 0 && MbarWaitWarp(&s.qFull, 0, abortFlag) && MbarWaitWarp(&s.kvFull[0], 0, abortFlag);
        if (ok) {
            TcFenceAfter();
            if (elected) {
                scores(0, 0);
                MmaCommit(&s.sFull[0]);
                if (two) {
                    scores(1, 0);
                    MmaCommit(&s.sFull[1]);
                }
                MmaCommit(&s.kvEmpty[0]);
            }
            step();
        }
        for (int j = 0; ok && j < n; j++) {
            const uint32_t v = st, vPh = ph;
            step();
            const uint32_t k = st, kPh = ph;
            const bool next = j + 1 < n;
            if (next) {
                step();
            }
            ok = MbarWaitWarp(&s.kvFull[v], vPh, abortFlag) && (!next || MbarWaitWarp(&s.kvFull[k], kPh, abortFlag));
            for (int i = 0; ok && i < (two ? 2 : 1); i++) {
                ok = MbarWaitWarp(&s.pFull[i], j & 1, abortFlag);
                if (!ok) {
                    break;
                }
                TcFenceAfter();
                if (elected) {
                    values(i, v, j > 0);
                    if (i == 1 || !two) {
                        MmaCommit(&s.kvEmpty[v]);
                    }
                    if (next) {
                        scores(i, k);
                        MmaCommit(&s.sFull[i]);
                        if (i == 1 || !two) {
                            MmaCommit(&s.kvEmpty[k]);
                        }
                    } else {
                        MmaCommit(&s.oFull[i]);
                    }
                }
            }
        }
    } else {
        const int i = warp >> 2;  // the tile
        const int row = (warp & 3) * 32 + lane, token = t0 + i * half + row / p.pack, head = h0 + row % p.pack;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, sAt = tmem + lanes + i * kTile, oAt = tmem + lanes + kO + i * D;
        if (i == 0 || two) {
            const int limit = a.causal ? min(keys, token + past + 1) : keys;  // keys that the row sees
            const int sure = __reduce_min_sync(~0u, limit);
            const float factor = a.scale * kLog2e;
            float top = -INFINITY, sum = 0;
            bool ok = true;
            for (int j = 0; j < n; j++) {
                if (!__all_sync(~0u, MbarWaitBounded(&s.sFull[i], j & 1, abortFlag))) {
                    ok = false;
                    break;
                }
                TcFenceAfter();
                float x[kTile];
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    TmemLd32Issue(sAt + c, x + c);
                }
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    TmemLdWait32(x + c);
                }
                if ((j + 1) * kTile > sure) {
                    const int left = limit - j * kTile;
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
                        m[e] = Max3(m[e], x[c + e], x[c + 4 + e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    m[e] = fmaxf(m[e], x[kTile - 4 + e]);
                }
                const float best = Max3(Max3(m[0], m[1], m[2]), m[3], m[3]);
                const bool grown = (best - top) * factor > kSlack;
                if (__any_sync(~0u, grown)) {
                    const float shrink = grown ? Exp2((top - best) * factor) : 1.0f;
                    top = grown ? best : top;
                    sum *= shrink;
                    if (j > 0) {
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
                float part[4] = {0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float u = Exp2(fmaf(x[c + e], factor, from)), v = Exp2(fmaf(x[c + e + 1], factor, from));
                        part[e & 2] += u;
                        part[(e & 2) + 1] += v;
                        w[e / 2] = Pack2<T>(u, v);
                    }
                    TmemSt16(sAt + c / 2, w);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                TmemStWait();
                TcFenceBefore();
                __syncwarp();
                if (lane == 0) {
                    MbarArrive(&s.pFull[i]);
                }
            }
            if (n > 0 && ok) {
                ok = __all_sync(~0u, MbarWaitBounded(&s.oFull[i], 0, abortFlag));
                TcFenceAfter();
            }
            if (ok) {
                const float scale = sum != 0 ? 1.0f / sum : 0.0f;
                const size_t at = (size_t)(q0 + token);
                T *out = (T *)a.out + at * a.outStride[0] + (size_t)head * a.outStride[1];
                float *lse = a.lse != nullptr ? a.lse + at * a.kvHeads * a.group + head : nullptr;
                bool odd = false;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    if (n > 0) {
                        TmemLd32Issue(oAt + c, o);
                        TmemLdWait32(o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            o[e] = 0;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        odd |= !(fabsf(o[e]) <= 3.4e38f);
                    }
                    if (token < rows) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            *(uint4 *)(out + c + e) = make_uint4(Pack2<T>(o[e] * scale, o[e + 1] * scale), Pack2<T>(o[e + 2] * scale, o[e + 3] * scale),
                                                                 Pack2<T>(o[e + 4] * scale, o[e + 5] * scale), Pack2<T>(o[e + 6] * scale, o[e + 7] * scale));
                        }
                    }
                }
                if (lse != nullptr && token < rows) {
                    *lse = top * factor * kLn2 + logf(sum);
                }
                unsigned again = __ballot_sync(~0u, odd && token < rows);
                while (again != 0) {
                    const int r = (warp & 3) * 32 + __ffs(again) - 1, t = t0 + i * half + r / p.pack, h = h0 + r % p.pack;
                    again &= again - 1;
                    const size_t q = (size_t)(q0 + t);
                    AttendRow<T, D>((const T *)a.q + q * a.qStride[0] + (size_t)h * a.qStride[1], (const T *)a.k + (size_t)k0 * a.kStride[0] + (size_t)kvh * a.kStride[1],
                                    a.kStride[0], (const T *)a.v + (size_t)k0 * a.vStride[0] + (size_t)kvh * a.vStride[1], a.vStride[0],
                                    a.causal ? min(keys, t + past + 1) : keys, factor, (T *)a.out + q * a.outStride[0] + (size_t)h * a.outStride[1],
                                    a.lse != nullptr ? a.lse + q * a.kvHeads * a.group + h : nullptr);
                }
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
    p.pack = a.group & -a.group;
    p.pack = p.pack > kTile ? kTile : p.pack;
    p.tokens = 2 * kTile / p.pack;
    p.headTiles = a.kvHeads * a.group / p.pack;
    p.tiles = a.tokensQ / p.tokens + a.B;
    const long long ctas = (long long)p.tiles * p.headTiles;
    if (ctas > 0x7fffffffll) {
        return MF_K_TOO_LARGE;
    }
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
        LaunchDependent(mf_prefill_attention_kernel<T, D>, (unsigned)ctas, kThreads, smem, stream, q, k, v, p) != cudaSuccess) {
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
