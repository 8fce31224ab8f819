// Attention over packed prompts, causal or not, with grouped heads:
//
//     out[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(s q[i, h] . k_j - max_j),   j <= i + (keys - rows) of i's sequence,
//
// in one pass over the keys with a running maximum and sum. A CTA takes 64 rows of one query head, four warps 16 rows each; keys and values
// come in tiles of 64 through two stages of shared memory. p is rounded to the operands' type for the second product; its sum
// is taken before that, all sums in fp32.
#include "mf_attention.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using mf::sm100::GridDependency;

constexpr int kThreads = 128;
constexpr int kTileRows = 64;
constexpr int kTileKeys = 64;

template <int D>
struct Cfg {
    static constexpr uint32_t kRow = D * 2, kChunks = D / 8, kTile = kTileKeys * kRow, kSmem = 4 * kTile;
    static __device__ __forceinline__ uint32_t Place(uint32_t row, uint32_t chunk) { return row * kRow + ((chunk ^ (row & 7)) << 4); }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) mf_prefill_attention_kernel(const __grid_constant__ mf_prefill_attention_args_t a)
{
    using X = Cfg<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    GridDependency();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, pos = lane & 3;
    // Tiles of sequence b have numbers from cuQ[b] / 64 + b on: enough for its rows wherever they begin, some numbers stay empty.
    const int tile = blockIdx.x, h = blockIdx.y, kvh = h / a.group;
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (a.cuQ[mid] / kTileRows + mid <= tile ? lo : hi) = mid;
    }
    const int q0 = a.cuQ[lo], rows = min(a.cuQ[lo + 1], a.tokensQ) - q0, row0 = (tile - (q0 / kTileRows + lo)) * kTileRows;
    if (q0 < 0 || row0 < 0 || row0 >= rows) {
        return;
    }
    const int k0 = a.cuK[lo], keys = k0 < 0 ? 0 : min(a.cuK[lo + 1], a.tokensK) - k0;
    const int past = keys - rows;
    const int see = a.causal ? min(keys, row0 + kTileRows + past) : keys, tiles = see > 0 ? (see + kTileKeys - 1) / kTileKeys : 0;

    const uint32_t base = SmemAddr32(smem);
    auto fetch = [&](int t) {
        if (t < tiles) {
            const uint32_t at = base + (t & 1) * 2 * X::kTile;
#pragma unroll
            for (int i = 0; i < (int)(kTileKeys * X::kChunks) / kThreads; i++) {
                const uint32_t row = (i * kThreads + tid) / X::kChunks, chunk = (i * kThreads + tid) % X::kChunks;
                const int key = t * kTileKeys + row;
                const uint32_t bytes = key < keys ? 16 : 0;
                const size_t n = key < keys ? (size_t)k0 + key : 0;
                CpAsync16(at + X::Place(row, chunk), (const T *)a.k + n * a.kStride[0] + (size_t)kvh * a.kStride[1] + chunk * 8, bytes);
                CpAsync16(at + X::kTile + X::Place(row, chunk), (const T *)a.v + n * a.vStride[0] + (size_t)kvh * a.vStride[1] + chunk * 8, bytes);
            }
        }
        CpCommit();
    };
    fetch(0);

    uint32_t q[D / 16][4];
    int row[2];
#pragma unroll
    for (int half = 0; half < 2; half++) {
        row[half] = row0 + warp * 16 + quad + half * 8;
        const T *src = (const T *)a.q + (size_t)(q0 + row[half]) * a.qStride[0] + (size_t)h * a.qStride[1];
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
            q[s][half] = row[half] < rows ? *(const uint32_t *)(src + s * 16 + pos * 2) : 0;
            q[s][half + 2] = row[half] < rows ? *(const uint32_t *)(src + s * 16 + pos * 2 + 8) : 0;
        }
    }
    float acc[D / 8][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0, 0};
#pragma unroll
    for (int n = 0; n < D / 8; n++) {
        acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
    }
    const float factor = a.scale * kLog2e;
    for (int t = 0; t < tiles; t++) {
        fetch(t + 1);
        CpWait<1>();
        __syncthreads();
        const uint32_t at = base + (t & 1) * 2 * X::kTile;
        float s[kTileKeys / 8][4];
#pragma unroll
        for (int n = 0; n < kTileKeys / 8; n++) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0;
        }
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
#pragma unroll
            for (int n = 0; n < kTileKeys / 16; n++) {
                uint32_t m[4];
                LdMatrix4(m, at + X::Place(n * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * d + ((lane >> 3) & 1)));
                Mma16x8x16<T>(s[2 * n], q[d], m[0], m[1]);
                Mma16x8x16<T>(s[2 * n + 1], q[d], m[2], m[3]);
            }
        }
        uint32_t p[kTileKeys / 16][4];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int last = a.causal ? min(keys, row[half] + past + 1) : keys;  // keys that the row sees
            float best = top[half];
#pragma unroll
            for (int n = 0; n < kTileKeys / 8; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float &x = s[n][2 * half + e];
                    x = t * kTileKeys + n * 8 + pos * 2 + e < last ? x * factor : -INFINITY;
                    best = fmaxf(best, x);
                }
            }
            best = fmaxf(best, __shfl_xor_sync(~0u, best, 1));
            best = fmaxf(best, __shfl_xor_sync(~0u, best, 2));
            const float from = best == -INFINITY ? 0.0f : best, shrink = Exp2(top[half] - from);
            top[half] = best;
            sum[half] *= shrink;
#pragma unroll
            for (int n = 0; n < kTileKeys / 8; n++) {
                const float x = Exp2(s[n][2 * half] - from), y = Exp2(s[n][2 * half + 1] - from);
                sum[half] += x + y;
                p[n / 2][(n & 1) * 2 + half] = Pack2<T>(x, y);
            }
#pragma unroll
            for (int n = 0; n < D / 8; n++) {
                acc[n][2 * half] *= shrink;
                acc[n][2 * half + 1] *= shrink;
            }
        }
#pragma unroll
        for (int n = 0; n < kTileKeys / 16; n++) {
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                uint32_t m[4];
                LdMatrix4T(m, at + X::kTile + X::Place(n * 16 + (lane & 15), 2 * d + (lane >> 4)));
                Mma16x8x16<T>(acc[2 * d], p[n], m[0], m[1]);
                Mma16x8x16<T>(acc[2 * d + 1], p[n], m[2], m[3]);
            }
        }
        __syncthreads();
    }
    CpWait<0>();
#pragma unroll
    for (int half = 0; half < 2; half++) {
        sum[half] += __shfl_xor_sync(~0u, sum[half], 1);
        sum[half] += __shfl_xor_sync(~0u, sum[half], 2);
        const float scale = sum[half] != 0 ? 1.0f / sum[half] : 0.0f;
        bool odd = false;
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
            odd |= !(fabsf(acc[n][2 * half]) <= 3.4e38f) || !(fabsf(acc[n][2 * half + 1]) <= 3.4e38f);
        }
        unsigned again = __ballot_sync(~0u, odd && row[half] < rows);
        while (again != 0) {
            const int r = row0 + warp * 16 + half * 8 + ((__ffs(again) - 1) >> 2);
            again &= ~(15u << ((__ffs(again) - 1) & ~3));
            const size_t token = (size_t)(q0 + r);
            AttendRow<T, D>((const T *)a.q + token * a.qStride[0] + (size_t)h * a.qStride[1], (const T *)a.k + (size_t)k0 * a.kStride[0] + (size_t)kvh * a.kStride[1],
                            a.kStride[0], (const T *)a.v + (size_t)k0 * a.vStride[0] + (size_t)kvh * a.vStride[1], a.vStride[0],
                            a.causal ? min(keys, r + past + 1) : keys, factor, (T *)a.out + token * a.outStride[0] + (size_t)h * a.outStride[1],
                            a.lse != nullptr ? a.lse + token * a.kvHeads * a.group + h : nullptr);
        }
        odd = __shfl_sync(~0u, (int)odd, lane & ~3) | __shfl_sync(~0u, (int)odd, (lane & ~3) + 1) | __shfl_sync(~0u, (int)odd, (lane & ~3) + 2) |
              __shfl_sync(~0u, (int)odd, (lane & ~3) + 3);
        if (row[half] >= rows || odd) {
            continue;
        }
        T *out = (T *)a.out + (size_t)(q0 + row[half]) * a.outStride[0] + (size_t)h * a.outStride[1];
#pragma unroll
        for (int n = 0; n < D / 8; n++) {
            *(uint32_t *)(out + n * 8 + pos * 2) = Pack2<T>(acc[n][2 * half] * scale, acc[n][2 * half + 1] * scale);
        }
        if (a.lse != nullptr && pos == 0) {
            a.lse[(size_t)(q0 + row[half]) * a.kvHeads * a.group + h] = top[half] * kLn2 + logf(sum[half]);
        }
    }
}

template <typename T, int D>
int Launch(const mf_prefill_attention_args_t &a, cudaStream_t stream)
{
    if (!mf::AllowSmem<mf_prefill_attention_kernel<T, D>>(Cfg<D>::kSmem)) {
        return MF_K_LAUNCH_FAILED;
    }
    mf_prefill_attention_kernel<T, D><<<dim3(a.tokensQ / kTileRows + a.B, a.kvHeads * a.group), kThreads, Cfg<D>::kSmem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? MF_K_OK : MF_K_LAUNCH_FAILED;
}

}  // namespace

extern "C" int mf_k_prefill_attention(const mf_prefill_attention_args_t *args, int D, int type, mf_stream_t stream)
{
    if (args == nullptr || args->B < 0 || args->kvHeads <= 0 || args->group <= 0 || args->tokensQ < 0 || args->tokensK < 0 || (D != 64 && D != 128) ||
        (type != MF_K_BF16 && type != MF_K_FP16) || (long long)args->kvHeads * args->group > 65535) {
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
