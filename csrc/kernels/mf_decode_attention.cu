// Attention of one new token per sequence over a paged key-value cache:
//
//     out[b, h] = sum_j p_j v_j,   p_j = exp(s q[b, h] . k_j) / sum_i exp(s q[b, h] . k_i),   j < length of sequence b,
//
// where k_j, v_j of cache head h / (heads per cache head) are found through the sequence's page table. Memory bound: every key and
// value is read once and takes part in 4 * group operations per element, so what counts is that all SMs stream, all the time, whatever
// the lengths are.
//
// Work split. The keys of every (sequence, cache head) are cut into tiles of 64; the tiles of all rows form one line, and each CTA takes an
// equal, contiguous piece of it, whichever rows that touches (lengths live on the device: the host sizes the grid only). A row that lies
// within one CTA is written at once; of a row that crosses CTAs each leaves maximum, sum and unnormalised output in the workspace,
// at most two per CTA, and a second kernel joins them in the order of the CTAs, so results do not depend on timing. Where no row has more
// than kWholeTiles tiles, CTAs take whole rows and nothing has to be joined.
//
// A CTA is four warps that share nothing but their position: each takes 16 keys of every tile, fetches them through its own ring of
// cp.async stages (rows past the end of the sequence are filled with zeros: stale pages may hold anything, NaN included), computes
// q k^T and p v with m16n8k16 products (the group's query heads are the 16 rows) and keeps its own running maximum and sum; they
// meet at the end of a row. 8-bit caches are widened to fp16, which holds every e4m3 value; the query is scaled by a power of two per
// head so that it fits fp16 without loss. p is rounded to the cache's type (fp16 for 8-bit caches) for the second product, as the
// tensor cores want equal types; the sum is taken before that rounding, all sums in fp32.
#include "mf/device/mf_shm_device.cuh"
#include "mf_attention.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using mf::sm100::GridDependency;

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kWarpKeys = 16;
constexpr int kTileKeys = kWarps * kWarpKeys;
constexpr int kWholeTiles = 4;
constexpr int kRows = 16;                  // query heads of a tile
constexpr uint32_t kWarpRing = 24 * 1024;  // bytes of a warp's stages
constexpr int kPartialFloats = 2;          // maximum and sum before a row's values

template <typename C, int D>
struct Cfg {
    static constexpr uint32_t kRow = D * sizeof(C);
    static constexpr uint32_t kChunks = kRow / 16;
    static constexpr uint32_t kStage = kWarpKeys * kRow * 2;
    static constexpr int kStages = kWarpRing / kStage > 8 ? 8 : kWarpRing / kStage;
    static constexpr uint32_t kRing = kStages * kStage;
    static constexpr uint32_t kSmem = kWarps * kRing + kRows * D * 4;
    static __device__ __forceinline__ uint32_t Place(uint32_t row, uint32_t chunk)
    {
        const uint32_t x = kRow >= 128 ? row & 7 : (row >> 1) & 3;  // eight rows of one chunk lie in eight different bank groups
        return row * kRow + ((chunk ^ x) << 4);
    }
};

// The row that a position of the line of tiles lies in.
struct Cursor {
    int b, hg, tile, tiles, length;
};

struct Line {
    const int *lengths;
    const int *rows;
    int B, HG, cap, tableRows;
    __device__ __forceinline__ int Seq(int b) const { return rows != nullptr ? rows[b] : b; }
    __device__ __forceinline__ int Length(int b) const
    {
        const int seq = Seq(b);
        const int n = seq >= 0 && seq < tableRows ? lengths[seq] : 0;
        return n < 0 ? 0 : n > cap ? cap : n;
    }
    __device__ __forceinline__ void Open(Cursor &c, int b) const
    {
        c.length = 0;
        for (; b < B; b++) {
            c.length = Length(b);
            if (c.length > 0) {
                break;
            }
        }
        c.b = b;
        c.tiles = (c.length + kTileKeys - 1) / kTileKeys;
    }
    __device__ __forceinline__ void Next(Cursor &c) const
    {
        if (++c.tile == c.tiles) {
            c.tile = 0;
            if (++c.hg == HG) {
                c.hg = 0;
                Open(c, c.b + 1);
            }
        }
    }
};

template <typename Q, typename C>
struct Operand {
    using type = C;
};
template <typename Q>
struct Operand<Q, __nv_fp8_e4m3> {
    using type = __half;
};

// One partial result: [row]{maximum, sum} of kRows rows, then [row][D] values. Two per CTA: of the row that it enters in the middle, and of
// the row that goes on behind it.
template <int D>
__device__ __forceinline__ float *Partial(float *ws, int cta, int which)
{
    return ws + ((size_t)cta * 2 + which) * (kRows * (D + kPartialFloats));
}

template <typename Q, typename C, int D>
__global__ void __launch_bounds__(kThreads, 2) mf_decode_attention_kernel(const __grid_constant__ mf_decode_attention_args_t a)
{
    using X = Cfg<C, D>;
    using T = typename Operand<Q, C>::type;
    constexpr bool kWide = sizeof(C) == 1;
    constexpr int kSteps = D / 16;  // products along D of q k^T; pairs of column tiles of p v
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float joinMax[kWarps][kRows], joinSum[kWarps][kRows];
    __shared__ long long scan[kWarps][2];
    __shared__ int scanMax[kWarps];
    __shared__ int startB;
    __shared__ long long startOff;
    GridDependency();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, pos = lane & 3;
    const int GT = (a.group + kRows - 1) / kRows, HG = a.kvHeads * GT;
    const Line line{a.lengths, a.rows, a.B, HG, a.tableWidth * a.pageSize, a.tableRows};

    // ---- where this CTA's piece of the line begins and how long it is
    const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    long long tiles = 0, rows = 0;
    int longest = 0;
    for (int b = b0; b < b1; b++) {
        const int n = (line.Length(b) + kTileKeys - 1) / kTileKeys;
        tiles += n;
        rows += n > 0;
        longest = max(longest, n);
    }
    long long tilesUpTo = tiles, rowsUpTo = rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long t = __shfl_up_sync(~0u, tilesUpTo, d), r = __shfl_up_sync(~0u, rowsUpTo, d);
        if (lane >= d) {
            tilesUpTo += t;
            rowsUpTo += r;
        }
        longest = max(longest, __shfl_xor_sync(~0u, longest, d));
    }
    if (lane == 31) {
        scan[warp][0] = tilesUpTo;
        scan[warp][1] = rowsUpTo;
        scanMax[warp] = longest;
    }
    if (tid == 0) {
        startB = a.B;
        startOff = 0;
    }
    __syncthreads();
    long long total[2] = {0, 0}, before[2] = {tilesUpTo - tiles, rowsUpTo - rows};
    longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        for (int i = 0; i < 2; i++) {
            before[i] += w < warp ? scan[w][i] : 0;
            total[i] += scan[w][i];
        }
        longest = max(longest, scanMax[w]);
    }
    const bool whole = longest <= kWholeTiles;
    const long long units = (whole ? total[1] : total[0]) * HG;
    // a piece is worth a CTA from kWholeTiles tiles on; the CTAs behind the last piece have none
    const long long wanted = whole ? units : (units + kWholeTiles - 1) / kWholeTiles, parts = wanted < gridDim.x ? wanted : gridDim.x;
    long long first = 0, left = 0;
    if (blockIdx.x < parts) {
        first = units * blockIdx.x / parts;
        left = units * (blockIdx.x + 1) / parts - first;
    }
    {
        long long at = (whole ? before[1] : before[0]) * HG, mine = (whole ? rows : tiles) * HG;
        if (left > 0 && first >= at && first < at + mine) {
            for (int b = b0; b < b1; b++) {
                const int n = (line.Length(b) + kTileKeys - 1) / kTileKeys;
                const long long here = (long long)(whole ? n > 0 : n) * HG;
                if (first < at + here) {
                    startB = b;
                    startOff = first - at;
                    break;
                }
                at += here;
            }
        }
    }
    // sequences without a key
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (line.Length(b) == 0) {
            if (a.status != nullptr && tid == 0 && (line.Seq(b) < 0 || line.Seq(b) >= a.tableRows)) {
                *a.status = MF_DEV_ERR_BOUNDS;
            }
            for (int i = tid; i < a.kvHeads * a.group * (D / 8); i += kThreads) {
                const int h = i / (D / 8);
                *(uint4 *)((Q *)a.out + (size_t)b * a.outStride[0] + (size_t)h * a.outStride[1] + (i % (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
                if (a.lse != nullptr && i % (D / 8) == 0) {
                    a.lse[(size_t)b * a.kvHeads * a.group + h] = -INFINITY;
                }
            }
        }
    }
    __syncthreads();
    if (tid < 2 && a.workspace != nullptr) {
        ((int2 *)a.marks)[blockIdx.x * 2 + tid] = make_int2(-1, -1);  // {sequence, head group} of the two partial results
    }
    if (left <= 0) {
        return;
    }
    Cursor cur;
    line.Open(cur, startB);
    if (whole) {
        cur.hg = (int)startOff;
        cur.tile = 0;
    } else {
        cur.hg = (int)(startOff / cur.tiles);
        cur.tile = (int)(startOff % cur.tiles);
    }

    // ---- the warp's ring of stages
    const uint32_t ring = SmemAddr32(smem) + warp * X::kRing;
    float *join = (float *)(smem + kWarps * X::kRing);
    Cursor ahead = cur;
    long long aheadLeft = left;
    uint32_t fill = 0;
    auto fetch = [&]() {
        if (aheadLeft > 0) {
            const int key0 = ahead.tile * kTileKeys + warp * kWarpKeys;
            if (key0 < ahead.length) {
                // each lane looks one of the 16 rows up
                const int key = key0 + (lane & 15);
                const uint32_t page = (uint32_t)key / (uint32_t)a.pageSize, slot = (uint32_t)key % (uint32_t)a.pageSize;
                long long off = -1;
                if (key < ahead.length) {
                    const int p = a.table[(size_t)line.Seq(ahead.b) * a.tableStride + page];
                    if (p >= 0 && p < a.pages) {
                        off = p * a.stride[0] + (ahead.hg / GT) * a.stride[1] + (long long)slot * a.stride[2];
                    } else if (a.status != nullptr) {
                        *a.status = MF_DEV_ERR_BOUNDS;
                    }
                }
                const uint32_t at = ring + fill * X::kStage;
                constexpr int kPer = 32 / X::kChunks;  // rows of one trip
#pragma unroll
                for (int i = 0; i < kWarpKeys / kPer; i++) {
                    const uint32_t row = i * kPer + lane / X::kChunks, chunk = lane % X::kChunks;
                    const long long o = __shfl_sync(~0u, off, row);
                    const uint32_t bytes = o >= 0 ? 16 : 0;
                    const size_t from = o >= 0 ? (size_t)o * sizeof(C) + chunk * 16 : 0;
                    CpAsync16(at + X::Place(row, chunk), (const unsigned char *)a.k + from, bytes);
                    CpAsync16(at + kWarpKeys * X::kRow + X::Place(row, chunk), (const unsigned char *)a.v + from, bytes);
                }
            }
            aheadLeft -= !whole || ahead.tile + 1 == ahead.tiles;
            line.Next(ahead);
        }
        CpCommit();
        fill = fill + 1 == X::kStages ? 0 : fill + 1;
    };
#pragma unroll 1
    for (int i = 0; i < X::kStages - 1; i++) {
        fetch();
    }

    uint32_t q[kSteps][4];
    float acc[D / 8][4];
    float top[2], sum[2], factor[2];
    uint32_t take = 0;
    int rowStart = 0;
    bool open = true;
    while (left > 0) {
        if (open) {  // a row begins: its query heads, lane by lane as the products want them
            open = false;
            rowStart = cur.tile;
            const int kvh = cur.hg / GT, g0 = (cur.hg % GT) * kRows;
            const float ks = kWide ? a.kScale[kvh] : 1.0f;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int g = g0 + quad + half * 8;
                const Q *src = (const Q *)a.q + (size_t)cur.b * a.qStride[0] + (size_t)(kvh * a.group + g) * a.qStride[1];
                float biggest = 0;
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    // 8-bit keys come as four neighbouring columns to a lane, 16-bit ones as two and two
                    const int d = s * 16 + (kWide ? pos * 4 : pos * 2);
                    uint32_t lo = 0, hi = 0;
                    if (g < a.group) {
                        lo = *(const uint32_t *)(src + d);
                        hi = *(const uint32_t *)(src + d + (kWide ? 2 : 8));
                    }
                    q[s][half] = lo;
                    q[s][half + 2] = hi;
                    if (kWide) {
                        const float2 x = Unpack2<Q>(lo), y = Unpack2<Q>(hi);
                        biggest = fmaxf(fmaxf(biggest, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
                    }
                }
                factor[half] = a.scale * kLog2e * ks;
                if (kWide) {
                    biggest = fmaxf(biggest, __shfl_xor_sync(~0u, biggest, 1));
                    biggest = fmaxf(biggest, __shfl_xor_sync(~0u, biggest, 2));
                    int e = (int)(__float_as_uint(biggest) >> 23) - 127;  // its exponent: scaled values lie below two
                    e = biggest == 0 || e > 126 ? 0 : e < -100 ? -100 : e;
                    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                    factor[half] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                    for (int s = 0; s < kSteps; s++) {
                        const float2 x = Unpack2<Q>(q[s][half]), y = Unpack2<Q>(q[s][half + 2]);
                        q[s][half] = Pack2<__half>(x.x * down, x.y * down);
                        q[s][half + 2] = Pack2<__half>(y.x * down, y.y * down);
                    }
                }
                top[half] = -INFINITY;
                sum[half] = 0;
            }
#pragma unroll
            for (int n = 0; n < D / 8; n++) {
                acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0;
            }
        }
        CpWait<X::kStages - 2>();
        __syncwarp();  // the stage is there for all lanes, and nobody reads the one before it any more: that one is filled again
        fetch();
        const int key0 = cur.tile * kTileKeys + warp * kWarpKeys;
        if (key0 < cur.length) {
            const uint32_t at = ring + take * X::kStage;
            float s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0};
            const uint32_t kRowOf = (lane & 7) + ((lane >> 4) << 3), kChunkOf = (lane >> 3) & 1;
            if (kWide) {
#pragma unroll
                for (int s = 0; s < kSteps; s += 2) {
                    uint32_t m[4];
                    LdMatrix4(m, at + X::Place(kRowOf, s + kChunkOf));
                    Mma16x8x16<T>(s0, q[s], E4m3ToHalf2(m[0]), E4m3ToHalf2(m[0] >> 16));
                    Mma16x8x16<T>(s1, q[s], E4m3ToHalf2(m[2]), E4m3ToHalf2(m[2] >> 16));
                    Mma16x8x16<T>(s0, q[s + 1], E4m3ToHalf2(m[1]), E4m3ToHalf2(m[1] >> 16));
                    Mma16x8x16<T>(s1, q[s + 1], E4m3ToHalf2(m[3]), E4m3ToHalf2(m[3] >> 16));
                }
            } else {
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    uint32_t m[4];
                    LdMatrix4(m, at + X::Place(kRowOf, 2 * s + kChunkOf));
                    Mma16x8x16<T>(s0, q[s], m[0], m[1]);
                    Mma16x8x16<T>(s1, q[s], m[2], m[3]);
                }
            }
            uint32_t p[4];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float x[4] = {s0[2 * half] * factor[half], s0[2 * half + 1] * factor[half], s1[2 * half] * factor[half], s1[2 * half + 1] * factor[half]};
                if (key0 + kWarpKeys > cur.length) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (key0 + (i >> 1) * 8 + pos * 2 + (i & 1) >= cur.length) {
                            x[i] = -INFINITY;
                        }
                    }
                }
                float best = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                best = fmaxf(best, __shfl_xor_sync(~0u, best, 1));
                best = fmaxf(best, __shfl_xor_sync(~0u, best, 2));
                best = fmaxf(best, top[half]);
                const float base = best == -INFINITY ? 0.0f : best, shrink = Exp2(top[half] - base);
                top[half] = best;
                float add = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = Exp2(x[i] - base);
                    add += x[i];
                }
                sum[half] = sum[half] * shrink + add;  // of this lane's columns; the four lanes of a row are added at its end
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    acc[n][2 * half] *= shrink;
                    acc[n][2 * half + 1] *= shrink;
                }
                p[half] = Pack2<T>(x[0], x[1]);
                p[half + 2] = Pack2<T>(x[2], x[3]);
            }
            const uint32_t vAt = at + kWarpKeys * X::kRow, vRowOf = lane & 15, vChunkOf = lane >> 4;
            if (kWide) {
#pragma unroll
                for (int s = 0; s < kSteps; s += 2) {
                    uint32_t m[4];
                    LdMatrix4T(m, vAt + X::Place(vRowOf, s + vChunkOf));
#pragma unroll
                    for (int c = 0; c < 2; c++) {  // a 16-bit unit holds an even and an odd column of one key: they go to two column tiles
                        Mma16x8x16<T>(acc[2 * (s + c)], p, E4m3ToHalf2(__byte_perm(m[2 * c], 0, 0x4420)), E4m3ToHalf2(__byte_perm(m[2 * c + 1], 0, 0x4420)));
                        Mma16x8x16<T>(acc[2 * (s + c) + 1], p, E4m3ToHalf2(__byte_perm(m[2 * c], 0, 0x4431)),
                                      E4m3ToHalf2(__byte_perm(m[2 * c + 1], 0, 0x4431)));
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    uint32_t m[4];
                    LdMatrix4T(m, vAt + X::Place(vRowOf, 2 * s + vChunkOf));
                    Mma16x8x16<T>(acc[2 * s], p, m[0], m[1]);
                    Mma16x8x16<T>(acc[2 * s + 1], p, m[2], m[3]);
                }
            }
        }
        take = take + 1 == X::kStages ? 0 : take + 1;
        left -= !whole || cur.tile + 1 == cur.tiles;
        const bool rowEnd = cur.tile + 1 == cur.tiles;
        if (rowEnd || left <= 0) {
            // ---- the four warps' results of this row become one
#pragma unroll
            for (int half = 0; half < 2; half++) {
                sum[half] += __shfl_xor_sync(~0u, sum[half], 1);
                sum[half] += __shfl_xor_sync(~0u, sum[half], 2);
                if (pos == 0) {
                    joinMax[warp][quad + half * 8] = top[half];
                    joinSum[warp][quad + half * 8] = sum[half];
                }
            }
            __syncthreads();
            float weight[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int r = quad + half * 8;
                const float best = fmaxf(fmaxf(joinMax[0][r], joinMax[1][r]), fmaxf(joinMax[2][r], joinMax[3][r]));
                weight[half] = best == -INFINITY ? 0.0f : Exp2(top[half] - best);
            }
            // a quarter of the columns at a time, each warp at another one: the order of the additions is fixed by the quarter
#pragma unroll
            for (int turn = 0; turn < kWarps; turn++) {
                const int part = (warp + turn) & 3;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    if (n / (D / 32) == part) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int col = kWide ? (n >> 1) * 16 + pos * 4 + (e & 1) * 2 + (n & 1) : n * 8 + pos * 2 + (e & 1);
                            float *at = join + (quad + (e >> 1) * 8) * D + col;
                            const float x = acc[n][e] * weight[e >> 1];
                            *at = turn == 0 ? x : *at + x;
                        }
                    }
                }
                __syncthreads();
            }
            const int kvh = cur.hg / GT, g0 = (cur.hg % GT) * kRows;
            const bool complete = rowEnd && rowStart == 0;
            const int which = rowStart != 0 ? 0 : 1;
            const float vs = kWide ? a.vScale[kvh] : 1.0f;
            for (int i = tid; i < kRows * (D / 8); i += kThreads) {
                const int r = i / (D / 8), d = (i % (D / 8)) * 8;
                const float best = fmaxf(fmaxf(joinMax[0][r], joinMax[1][r]), fmaxf(joinMax[2][r], joinMax[3][r]));
                float all = 0;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    all += best == -INFINITY ? 0.0f : joinSum[w][r] * Exp2(joinMax[w][r] - best);
                }
                const float4 x = *(const float4 *)(join + r * D + d), y = *(const float4 *)(join + r * D + d + 4);
                if (!complete) {
                    float *ws = Partial<D>((float *)a.workspace, blockIdx.x, which);
                    if (d == 0) {
                        *(float2 *)(ws + r * kPartialFloats) = make_float2(best, all);
                    }
                    ws += kRows * kPartialFloats + r * D + d;
                    *(float4 *)ws = x;
                    *(float4 *)(ws + 4) = y;
                } else if (g0 + r < a.group) {
                    const int h = kvh * a.group + g0 + r;
                    const float scale = (all != 0 ? 1.0f / all : 0.0f) * vs;
                    uint4 packed = make_uint4(Pack2<Q>(x.x * scale, x.y * scale), Pack2<Q>(x.z * scale, x.w * scale), Pack2<Q>(y.x * scale, y.y * scale),
                                              Pack2<Q>(y.z * scale, y.w * scale));
                    *(uint4 *)((Q *)a.out + (size_t)cur.b * a.outStride[0] + (size_t)h * a.outStride[1] + d) = packed;
                    if (a.lse != nullptr && d == 0) {
                        a.lse[(size_t)cur.b * a.kvHeads * a.group + h] = best * kLn2 + logf(all);
                    }
                }
            }
            if (!complete && tid == 0) {
                ((int2 *)a.marks)[blockIdx.x * 2 + which] = make_int2(cur.b, cur.hg);
            }
            __syncthreads();
            open = true;
        }
        line.Next(cur);
    }
    CpWait<0>();
}

// One CTA for each row that is continued behind CTA blockIdx.x of the first kernel: that one's second partial result and the first ones
// of the CTAs behind it, as long as they are of the same row. A thread owns eight columns of a query head.
template <typename Q, int D, bool WIDE>
__global__ void __launch_bounds__(kRows * 16) mf_decode_join_kernel(const __grid_constant__ mf_decode_attention_args_t a, int ctas)
{
    GridDependency();
    const int2 *marks = (const int2 *)a.marks;
    const int c = blockIdx.x;
    const int2 row = marks[2 * c + 1];
    if (row.x < 0) {
        return;
    }
    const int GT = (a.group + kRows - 1) / kRows, kvh = row.y / GT, g = (row.y % GT) * kRows;
    const int r = threadIdx.x / (D / 8), d = (threadIdx.x % (D / 8)) * 8;
    int n = 1;
    while (c + n < ctas) {
        const int2 m = marks[2 * (c + n)];
        if (m.x != row.x || m.y != row.y) {
            break;
        }
        n++;
    }
    float best = -INFINITY, all = 0, out[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = 0; i < n; i++) {
        const float *ws = Partial<D>((float *)a.workspace, c + i, i == 0 ? 1 : 0);
        const float2 ms = *(const float2 *)(ws + r * kPartialFloats);
        const float4 x = *(const float4 *)(ws + kRows * kPartialFloats + r * D + d), y = *(const float4 *)(ws + kRows * kPartialFloats + r * D + d + 4);
        const float next = fmaxf(best, ms.x), base = next == -INFINITY ? 0.0f : next;
        const float keep = Exp2(best - base), weight = Exp2(ms.x - base);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        best = next;
        all = all * keep + ms.y * weight;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[j] = out[j] * keep + v[j] * weight;
        }
    }
    if (g + r >= a.group) {
        return;
    }
    const int h = kvh * a.group + g + r;
    const float scale = (all != 0 ? 1.0f / all : 0.0f) * (WIDE ? a.vScale[kvh] : 1.0f);
    *(uint4 *)((Q *)a.out + (size_t)row.x * a.outStride[0] + (size_t)h * a.outStride[1] + d) =
        make_uint4(Pack2<Q>(out[0] * scale, out[1] * scale), Pack2<Q>(out[2] * scale, out[3] * scale), Pack2<Q>(out[4] * scale, out[5] * scale),
                   Pack2<Q>(out[6] * scale, out[7] * scale));
    if (a.lse != nullptr && d == 0) {
        a.lse[(size_t)row.x * a.kvHeads * a.group + h] = best * kLn2 + logf(all);
    }
}

template <typename Q, typename C, int D>
int Launch(const mf_decode_attention_args_t &a, int ctas, cudaStream_t stream)
{
    using X = Cfg<C, D>;
    if (!mf::AllowSmem<mf_decode_attention_kernel<Q, C, D>>(X::kSmem)) {
        return MF_K_LAUNCH_FAILED;
    }
    if (mf::sm100::LaunchDependent(mf_decode_attention_kernel<Q, C, D>, ctas, kThreads, X::kSmem, stream, a) != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    // rows of at most kWholeTiles tiles are never cut
    if ((long long)a.tableWidth * a.pageSize > kWholeTiles * kTileKeys &&
        mf::sm100::LaunchDependent(mf_decode_join_kernel<Q, D, sizeof(C) == 1>, ctas, kRows * (D / 8), 0, stream, a, ctas) != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    return MF_K_OK;
}

template <typename Q, typename C>
int LaunchDim(const mf_decode_attention_args_t &a, int D, int ctas, cudaStream_t stream)
{
    return D == 64 ? Launch<Q, C, 64>(a, ctas, stream) : Launch<Q, C, 128>(a, ctas, stream);
}

int Ctas(int B, int kvHeads, int group, long long capacity)
{
    const int sms = mf_k_sm_count();
    const long long rows = (long long)B * kvHeads * ((group + kRows - 1) / kRows), tiles = rows * ((capacity + kTileKeys - 1) / kTileKeys);
    const long long most = 2ll * (sms > 0 ? sms : 1);
    return (int)(tiles < most ? (tiles > 1 ? tiles : 1) : most);
}

}  // namespace

extern "C" size_t mf_k_decode_attention_workspace(int B, int kvHeads, int group, int D, long long capacity)
{
    if (B <= 0 || kvHeads <= 0 || group <= 0 || (D != 64 && D != 128) || capacity < 0) {
        return 0;
    }
    const size_t ctas = (size_t)Ctas(B, kvHeads, group, capacity);
    return ctas * 2 * (kRows * (D + kPartialFloats) * sizeof(float) + sizeof(int2));
}

extern "C" int mf_k_decode_attention(const mf_decode_attention_args_t *args, int D, int qType, int cacheType, mf_stream_t stream)
{
    if (args == nullptr || args->B < 0 || args->kvHeads <= 0 || args->group <= 0 || args->pageSize <= 0 || args->tableWidth < 0 || (D != 64 && D != 128) ||
        (long long)args->tableWidth * args->pageSize > 0x7fffff00ll || (cacheType == MF_K_E4M3 && (args->kScale == nullptr || args->vScale == nullptr))) {
        return MF_K_INVALID;
    }
    if (args->B == 0) {
        return MF_K_OK;
    }
    mf_decode_attention_args_t a = *args;
    const long long capacity = (long long)a.tableWidth * a.pageSize;
    const int ctas = Ctas(a.B, a.kvHeads, a.group, capacity);
    if (a.workspace == nullptr) {
        return MF_K_INVALID;
    }
    a.marks = (unsigned char *)a.workspace + (size_t)ctas * 2 * kRows * (D + kPartialFloats) * sizeof(float);
    if (qType == MF_K_BF16 && cacheType == MF_K_BF16) {
        return LaunchDim<__nv_bfloat16, __nv_bfloat16>(a, D, ctas, (cudaStream_t)stream);
    }
    if (qType == MF_K_FP16 && cacheType == MF_K_FP16) {
        return LaunchDim<__half, __half>(a, D, ctas, (cudaStream_t)stream);
    }
    if (qType == MF_K_BF16 && cacheType == MF_K_E4M3) {
        return LaunchDim<__nv_bfloat16, __nv_fp8_e4m3>(a, D, ctas, (cudaStream_t)stream);
    }
    if (qType == MF_K_FP16 && cacheType == MF_K_E4M3) {
        return LaunchDim<__half, __nv_fp8_e4m3>(a, D, ctas, (cudaStream_t)stream);
    }
    return MF_K_INVALID;
}
