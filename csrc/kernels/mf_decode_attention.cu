// Attention of one new token per sequence over a paged key-value cache:
//
//     out[b, h] = sum_j p_j v_j,   p_j = exp(s q[b, h] . k_j) / sum_i exp(s q[b, h] . k_i),   j < length of sequence b,
//
// where k_j, v_j of cache head h / (heads per cache head) are found through the sequence's page table. Memory bound: every key and
// value is read once and takes part in 4 * group operations per element, so what counts is that all SMs stream, all the time, whatever
// the lengths are.
//
// Work split. The keys of every (sequence, cache head) are cut into tiles of 64 to 256; the tiles of all rows form one line, and each CTA takes an
// equal, contiguous piece of it, whichever rows that touches (lengths live on the device: the host sizes the grid only). A row that lies
// within one CTA is written at once; of a row that crosses CTAs each leaves maximum, sum and unnormalised output in the workspace,
// at most two per CTA, and a second kernel joins them in the order of the CTAs, so results do not depend on timing. Where all rows are
// short (kWholeTiles), CTAs take whole rows and nothing has to be joined.
//
// A CTA is four warps that share nothing but their position: each takes a quarter of the keys of every tile, fetches them through its own ring
// of cp.async stages (rows past the end of the sequence are filled with zeros: stale pages may hold anything, NaN included) and keeps its
// own maximum and sum; they meet at the end of a row. Products are m16n8k16 with the keys (then the columns of v) as the 16 rows and eight
// query heads as the columns, so a group of up to eight heads costs one product per 16 x 16 values of the cache and all statistics of a
// head lie in the lanes that hold its results. The reference of the exponentials follows the maximum only where a weight
// would pass 2^8 (fp16: 2^14): most tiles need one vote for it, no shuffles and no scaling of the output.
//
// 8-bit caches are widened to fp16, which holds every e4m3 value. The query is scaled by a power of two per head, its largest element into
// [2^14, 2^15): bf16 elements down to 2^-31 of that keep all their bits, smaller ones err by 2^-39 of it at most (half of fp16's least step).
// p is rounded to the cache's type (fp16 for 8-bit caches) for the second product, as the tensor cores want equal types; the sum is taken
// before that rounding, all sums in fp32.
#include "mf/device/mf_shm_device.cuh"
#include "mf_attention.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using mf::sm100::GridDependency;

constexpr int kThreads = 128;
constexpr int kMostCtasPerSm = 3;
constexpr int kWarps = 4;
constexpr int kWholeKeys = 256;    // rows up to here are never cut: no workspace
constexpr int kPartialFloats = 2;  // maximum and sum before a row's values
constexpr int kLeastPiece = 2;
// Groups of threads that share the parts of a row in the second kernel. 61 sequences: two 77.9, four 77.1 us; with 16 query heads per key head 82.6 and 84.3.
template <int NT>
constexpr int kJoinGroups = 4 / NT;

template <typename C, int D, int NT>
struct Cfg {
    static constexpr uint32_t kRow = D * sizeof(C);
    static constexpr uint32_t kChunks = kRow / 16;
    // Blocks of 16 keys that a warp works on in one step: as many as make 8 KiB of keys and values (D = 64, e4m3, 200 sequences: two 109, four 102 us).
    static constexpr int kBlocks = 256 / kRow;
    static constexpr int kWarpKeys = 16 * kBlocks, kTileKeys = kWarps * kWarpKeys;
    // Where all rows are this short none is cut. Two tiles of 256 keys (e4m3 of 64 values): 8 sequences of 500 tokens 12.0 -> 10.3 us, 200 of 1024 the same;
    // four tiles everywhere: 200 of up to 512 tokens 33 -> 39.
    static constexpr int kWholeTiles = kWholeKeys / kTileKeys > 2 ? kWholeKeys / kTileKeys : 2;
    static_assert(kWholeTiles * kTileKeys >= kWholeKeys, "rows without a workspace are not cut");
    // Tiles that beginning and ending a row takes as long as; its queries and results grow with D. 0 / 1 / 2 / 3 tiles: D = 128, 61 ragged sequences 79.5,
    // 77.4, 76.9, 77.8 us, 200 of up to 1200 tokens 90.9, 76.5, 73.2, 73.4; D = 64, e4m3, 200 ragged ones 114, 102, 115, 133.
    static constexpr int kRowCost = D / 64;
    static constexpr uint32_t kStage = kWarpKeys * kRow * 2;  // keys and values of a warp's part of a tile
    // Where a block of keys takes many instructions for its bytes (8-bit ones), three CTAs per SM with two stages hide more than two with three: 116 ->
    // 113 us for 128 sequences of e4m3, of 64 values 121 -> 115; with 16-bit rows of 64 values 95 -> 116 us.
    static constexpr int kCtasPerSm = sizeof(C) == 1 && NT == 1 ? 3 : 2;
    static constexpr int kStages = (kCtasPerSm == 3 ? 16384 : 24576) / kStage;
    static constexpr uint32_t kRing = kStages * kStage;
    static constexpr int kRows = 8 * NT;
    static constexpr int kJoinRow = D + 4;  // floats from head to head: the lanes of a store fall into 32 banks
    static constexpr int kJoins = 2 / NT;   // buffers in which the warps add up a row
    static constexpr uint32_t kSmem = kWarps * kRing + kJoins * kRows * kJoinRow * 4;
    static __device__ __forceinline__ uint32_t Place(uint32_t row, uint32_t chunk)
    {
        // eight rows of one chunk lie in eight different bank groups: rows 0-7, 8-15, and of 8-bit ones also Key(0) to Key(7), Key(8) to Key(15)
        uint32_t x = kRow >= 128 ? row & 7 : (row >> 1) & 3;
        if (sizeof(C) == 1) {
            x ^= row >> 3 & 1 ? (kRow >= 128 ? 2 : 1) : 0;
        }
        return row * kRow + ((chunk ^ x) << 4);
    }
    // The key of a block that is row `row` of its products. The transposing load of 8-bit values gives a lane four neighbouring keys, which the second
    // product takes as two pairs, eight rows apart.
    static __device__ __forceinline__ int Key(int row) { return sizeof(C) == 1 ? (row & 6) * 2 + (row & 1) + (row >> 3) * 2 : row; }
};

// The row that a position of the line of tiles lies in.
struct Cursor {
    int b, hg, tile, tiles, length;
};

template <int TILE>
struct Line {
    const int *lengths;
    const int *rows;
    int B, HG, cap, tableRows;
    static __device__ __forceinline__ int Tiles(int length) { return (length + TILE - 1) / TILE; }
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
        c.tiles = Tiles(c.length);
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

// One partial result: [row]{reference, sum} of ROWS rows, then [row][D] values. Two per CTA: of the row that it enters in the middle, and of
// the row that goes on behind it.
template <int D, int ROWS>
__device__ __forceinline__ float *Partial(float *ws, int cta, int which)
{
    return ws + ((size_t)cta * 2 + which) * (ROWS * (D + kPartialFloats));
}

// NT: query heads of a row of the line, in eights.
template <typename Q, typename C, int D, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<C, D, NT>::kCtasPerSm) mf_decode_attention_kernel(const __grid_constant__ mf_decode_attention_args_t a)
{
    using X = Cfg<C, D, NT>;
    using T = typename Operand<Q, C>::type;
    constexpr bool kWide = sizeof(C) == 1;
    using L = Line<X::kTileKeys>;
    constexpr int kRows = X::kRows, kSteps = D / 16, kBlocks = X::kBlocks, kWarpKeys = X::kWarpKeys, kTileKeys = X::kTileKeys;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float joinTop[kWarps][kRows], joinSum[kWarps][kRows];
    __shared__ long long scan[kWarps][2];
    __shared__ int scanMax[kWarps];
    __shared__ int startB;
    __shared__ long long startOff;
    GridDependency();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, pos = lane & 3;
    const int GT = (a.group + kRows - 1) / kRows, HG = a.kvHeads * GT;
    const L line{a.lengths, a.rows, a.B, HG, a.tableWidth * a.pageSize, a.tableRows};

    // ---- where this CTA's piece of the line begins and how long it is
    const int per = (a.B + kThreads - 1) / kThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    long long tiles = 0, rows = 0;
    int longest = 0;
    for (int b = b0; b < b1; b++) {
        const int n = L::Tiles(line.Length(b));
        tiles += n > 0 ? n + X::kRowCost : 0;
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
    const bool whole = longest <= X::kWholeTiles;
    // The line in units: a row is X::kRowCost of them, then one for each tile; or one if rows are not cut. A piece is worth a CTA from
    // kLeastPiece units on; the CTAs behind the last piece have none.
    const int price = whole ? 1 : X::kRowCost;
    const long long units = (whole ? total[1] : total[0]) * HG, wanted = whole ? units : (units + kLeastPiece - 1) / kLeastPiece,
                    parts = wanted < gridDim.x ? wanted : gridDim.x;
    long long first = 0, last = 0;
    if (blockIdx.x < parts) {
        first = units * blockIdx.x / parts;
        last = units * (blockIdx.x + 1) / parts;
    }
    {
        long long at = (whole ? before[1] : before[0]) * HG;
        const long long mine = (whole ? rows : tiles) * HG;
        if (first < last && first >= at && first < at + mine) {
            for (int b = b0; b < b1; b++) {
                const int n = L::Tiles(line.Length(b));
                const long long here = (long long)(n == 0 ? 0 : whole ? 1 : n + price) * HG;
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
    if (first >= last) {
        return;
    }
    // A CTA that begins within a row's cost begins with its first tile; one that ends there leaves the row to the next CTA. `left`: units from
    // the current tile's to the piece's end, none if not above 0.
    Cursor cur;
    line.Open(cur, startB);
    const int all = whole ? 1 : price + cur.tiles, into = (int)(startOff % all);
    cur.hg = (int)(startOff / all);
    cur.tile = into > price ? into - price : 0;
    long long left = last - first - (whole || into > price ? 0 : price - into);
    auto next = [&](Cursor &c, long long &units) {
        const bool end = c.tile + 1 == c.tiles;
        units -= whole ? end : end ? 1 + price : 1;
        line.Next(c);
    };

    // ---- the warp's ring of stages
    const uint32_t ring = SmemAddr32(smem) + warp * X::kRing;
    float *join = (float *)(smem + kWarps * X::kRing);
    const bool together = a.pageSize % 16 == 0;  // 16 keys from a multiple of 16 on lie in one page
    constexpr int kPer = 32 / X::kChunks;        // rows that the warp copies in one trip
    const long long perKey = a.stride[2] * (long long)sizeof(C), perTrip = kPer * perKey, kToV = (const unsigned char *)a.v - (const unsigned char *)a.k,
                    lanePart = lane / X::kChunks * perKey + lane % X::kChunks * 16;
    Cursor ahead = cur;
    long long aheadLeft = left;
    uint32_t fill = 0;
    auto fetch = [&]() {
        if (aheadLeft > 0) {
            const int *entry = a.table + (size_t)line.Seq(ahead.b) * a.tableStride;
            const long long head = (ahead.hg / GT) * a.stride[1];
#pragma unroll
            for (int block = 0; block < kBlocks; block++) {
                const int key0 = ahead.tile * kTileKeys + warp * kWarpKeys + block * 16;
                if (key0 >= ahead.length) {
                    break;
                }
                // each lane looks the first or one of the 16 rows up: its offset in bytes, or -1
                const int key = key0 + (together ? 0 : lane & 15);
                long long own = -1;
                if (key < ahead.length) {
                    const uint32_t page = a.pageSize == 1 ? key : __umulhi((uint32_t)key, a.pageMagic) >> a.pageShift;
                    const int p = entry[page];
                    if (p >= 0 && p < a.pages) {
                        own = (p * a.stride[0] + head) * (long long)sizeof(C) + (long long)((uint32_t)key - page * (uint32_t)a.pageSize) * perKey;
                    } else if (a.status != nullptr) {
                        *a.status = MF_DEV_ERR_BOUNDS;
                    }
                }
                const uint32_t at = ring + fill * X::kStage;
                if (together && own >= 0 && key0 + 16 <= ahead.length) {  // all sixteen, a fixed number of bytes apart
                    const unsigned char *from = (const unsigned char *)a.k + own + lanePart;
#pragma unroll
                    for (int i = 0; i < 16 / kPer; i++) {
                        const uint32_t to = at + X::Place(block * 16 + i * kPer + lane / X::kChunks, lane % X::kChunks);
                        CpAsync16(to, from, 16);
                        CpAsync16(to + kWarpKeys * X::kRow, from + kToV, 16);
                        from += perTrip;
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 16 / kPer; i++) {
                    const uint32_t row = i * kPer + lane / X::kChunks, chunk = lane % X::kChunks;
                    const long long o = together ? own + row * perKey : __shfl_sync(~0u, own, row);
                    const bool there = together ? own >= 0 && key0 + (int)row < ahead.length : o >= 0;
                    const unsigned char *from = (const unsigned char *)a.k + (there ? o + chunk * 16 : 0);
                    const uint32_t to = at + X::Place(block * 16 + row, chunk);
                    CpAsync16(to, from, there ? 16 : 0);
                    CpAsync16(to + kWarpKeys * X::kRow, from + kToV, there ? 16 : 0);
                }
            }
            next(ahead, aheadLeft);
        }
        CpCommit();
        fill = fill + 1 == X::kStages ? 0 : fill + 1;
    };
#pragma unroll 1
    for (int i = 0; i < X::kStages - 1; i++) {
        fetch();
    }

    uint32_t q[NT][kSteps][2];
    float acc[NT][kSteps][4];  // 16 columns of v by 8 heads each
    // Of the two heads whose results the lane holds: the reference that logits are taken relative to, how far they may be above it, the sum. Before the first
    // key that counts the reference is 0 and nothing may be above, so that a relative logit is one FMA of its product, and nothing is asked for each (logits
    // first, a reference of -inf: e4m3 with 16 query heads per key head 74.8 against 73.4 us).
    float from[NT][2], limit[NT][2], sum[NT][2], factor[NT][2];
    auto top = [&](int t, int e) { return limit[t][e] == -INFINITY ? -INFINITY : from[t][e]; };
    float ks = 1.0f;
    // A row's query heads, lane by lane as the products want them. 8-bit keys come as four neighbouring columns to a lane, 16-bit ones as two and two.
    auto loadQueries = [&](const Cursor &c) {
        const int kvh = c.hg / GT, g0 = (c.hg % GT) * kRows;
        if (kWide) {
            ks = a.kScale[kvh];
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int g = g0 + t * 8 + quad;
            const Q *src = (const Q *)a.q + (size_t)c.b * a.qStride[0] + (size_t)(kvh * a.group + g) * a.qStride[1];
#pragma unroll
            for (int s = 0; s < kSteps; s++) {
                const int d = s * 16 + (kWide ? pos * 4 : pos * 2);
                q[t][s][0] = g < a.group ? *(const uint32_t *)(src + d) : 0;
                q[t][s][1] = g < a.group ? *(const uint32_t *)(src + d + (kWide ? 2 : 8)) : 0;
            }
        }
    };
    loadQueries(cur);
    uint32_t take = 0;
    int rowStart = 0;
    bool open = true;
    while (left > 0) {
        if (open) {  // a row begins
            open = false;
            rowStart = cur.tile;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float up = 1.0f;
                if (kWide) {
                    float biggest = 0;
#pragma unroll
                    for (int s = 0; s < kSteps; s++) {
                        const float2 x = Unpack2<Q>(q[t][s][0]), y = Unpack2<Q>(q[t][s][1]);
                        biggest = fmaxf(fmaxf(biggest, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
                    }
                    biggest = fmaxf(biggest, __shfl_xor_sync(~0u, biggest, 1));
                    biggest = fmaxf(biggest, __shfl_xor_sync(~0u, biggest, 2));
                    // its exponent: what is finite lies below 2^15 when scaled, also beside an infinity
                    const int e = max(-100, min(127, (int)(__float_as_uint(biggest) >> 23) - 127));
                    const float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
                    up = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
                    for (int s = 0; s < kSteps; s++) {
                        const float2 x = Unpack2<Q>(q[t][s][0]), y = Unpack2<Q>(q[t][s][1]);
                        q[t][s][0] = Pack2<__half>(x.x * down, x.y * down);
                        q[t][s][1] = Pack2<__half>(y.x * down, y.y * down);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    factor[t][e] = a.scale * kLog2e * ks * (kWide ? __shfl_sync(~0u, up, (2 * pos + e) * 4) : 1.0f);
                    limit[t][e] = -INFINITY;
                    from[t][e] = sum[t][e] = 0;
                }
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    acc[t][s][0] = acc[t][s][1] = acc[t][s][2] = acc[t][s][3] = 0;
                }
            }
        }
        CpWait<X::kStages - 2>();
        __syncwarp();  // the stage is there for all lanes, and nobody reads the one before it any more: that one is filled again
        fetch();
        const int key0 = cur.tile * kTileKeys + warp * kWarpKeys;
        const uint32_t at = ring + take * X::kStage;
        if (key0 < cur.length) {
            // A block behind the end of the sequence holds what was there before: its scores are masked, its values left alone.
            const int blocks = kBlocks == 1 ? 1 : min(kBlocks, (cur.length - key0 + 15) / 16);
            float x[kBlocks][NT][4];  // [row quad, quad + 8][head 2 pos, 2 pos + 1]
            bool grown = false;
#pragma unroll
            for (int block = 0; block < kBlocks; block++) {
                float y[2][NT][4];  // two chains of products
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        y[0][t][e] = y[1][t][e] = 0;
                    }
                }
                if (kWide) {
                    // matrices: rows 0-7 and 8-15 of one chunk, the same of the next; four neighbouring columns to a lane
#pragma unroll
                    for (int s = 0; s < kSteps; s += 2) {
                        uint32_t m[4];
                        LdMatrix4(m, at + X::Place(block * 16 + X::Key(lane & 15), s + (lane >> 4)));
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const uint32_t a0 = E4m3ToHalf2(m[2 * c]), a1 = E4m3ToHalf2(m[2 * c + 1]), a2 = E4m3ToHalf2(m[2 * c] >> 16),
                                           a3 = E4m3ToHalf2(m[2 * c + 1] >> 16);
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                Mma16x8x16<T>(y[c][t], a0, a1, a2, a3, q[t][s + c][0], q[t][s + c][1]);
                            }
                        }
                    }
                } else {
                    // matrices: keys 0-7 and 8-15 of the first eight columns, the same of the next eight
#pragma unroll
                    for (int s = 0; s < kSteps; s++) {
                        uint32_t m[4];
                        LdMatrix4(m, at + X::Place(block * 16 + (lane & 15), 2 * s + (lane >> 4)));
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            Mma16x8x16<T>(y[s & 1][t], m[0], m[1], m[2], m[3], q[t][s][0], q[t][s][1]);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool seen = key0 + block * 16 + X::Key(quad + (e >> 1) * 8) < cur.length;
                        x[block][t][e] = seen ? fmaf(y[0][t][e] + y[1][t][e], factor[t][e & 1], -from[t][e & 1]) : -INFINITY;
                        grown |= x[block][t][e] > limit[t][e & 1];
                    }
                }
            }
            if (__any_sync(~0u, grown)) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float old = from[t][e];
                        float best = top(t, e) + Weights<T>::kLift;
#pragma unroll
                        for (int block = 0; block < kBlocks; block++) {
                            best = fmaxf(best, fmaxf(x[block][t][e], x[block][t][e + 2]) + old);
                        }
                        best = fmaxf(best, __shfl_xor_sync(~0u, best, 4));
                        best = fmaxf(best, __shfl_xor_sync(~0u, best, 8));
                        best = fmaxf(best, __shfl_xor_sync(~0u, best, 16));
                        best -= Weights<T>::kLift;
                        const float now = best == -INFINITY ? 0.0f : best, shrink = Exp2(top(t, e) - now), move = now == old ? 0.0f : old - now;
                        from[t][e] = now;
                        limit[t][e] = best == -INFINITY ? -INFINITY : Weights<T>::kSlack;
#pragma unroll
                        for (int block = 0; block < kBlocks; block++) {
                            x[block][t][e] += move;
                            x[block][t][e + 2] += move;
                        }
                        sum[t][e] *= shrink;
#pragma unroll
                        for (int s = 0; s < kSteps; s++) {
                            acc[t][s][e] *= shrink;
                            acc[t][s][e + 2] *= shrink;
                        }
                    }
                }
            }
            const uint32_t vAt = at + kWarpKeys * X::kRow;
#pragma unroll
            for (int block = 0; block < kBlocks; block++) {
                if (block >= blocks) {
                    break;
                }
                uint32_t p[NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[block][t][e] = Exp2(x[block][t][e]);
                        sum[t][e & 1] += x[block][t][e];  // of this lane's keys; the lanes of a head are added at the end of the row
                    }
                    p[t][0] = Transposed8x8(Pack2<T>(x[block][t][0], x[block][t][1]));
                    p[t][1] = Transposed8x8(Pack2<T>(x[block][t][2], x[block][t][3]));
                }
                if (kWide) {
                    // matrices of 16 keys and 16 columns, transposed: two chunks, of each columns 0-7 and 8-15; four neighbouring keys to a lane
#pragma unroll
                    for (int s = 0; s < kSteps; s += 2) {
                        uint32_t m[4];
                        LdMatrix2T8(m, vAt + X::Place(block * 16 + (lane & 15), s + (lane >> 4)));
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const uint32_t a0 = E4m3ToHalf2(m[2 * c]), a1 = E4m3ToHalf2(m[2 * c + 1]), a2 = E4m3ToHalf2(m[2 * c] >> 16),
                                           a3 = E4m3ToHalf2(m[2 * c + 1] >> 16);
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                Mma16x8x16<T>(acc[t][s + c], a0, a1, a2, a3, p[t][0], p[t][1]);
                            }
                        }
                    }
                } else {
                    // matrices, transposed: columns 0-7 and 8-15 of keys 0-7, the same of keys 8-15
#pragma unroll
                    for (int s = 0; s < kSteps; s++) {
                        uint32_t m[4];
                        LdMatrix4T(m, vAt + X::Place(block * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1)));
#pragma unroll
                        for (int t = 0; t < NT; t++) {
                            Mma16x8x16<T>(acc[t][s], m[0], m[1], m[2], m[3], p[t][0], p[t][1]);
                        }
                    }
                }
            }
        }
        take = take + 1 == X::kStages ? 0 : take + 1;
        const Cursor done = cur;
        const bool rowEnd = cur.tile + 1 == cur.tiles;
        next(cur, left);
        if (rowEnd || left <= 0) {
            if (left > 0) {
                loadQueries(cur);  // on their way while the row is put together
            }
            // ---- the four warps' results of this row become one
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    sum[t][e] += __shfl_xor_sync(~0u, sum[t][e], 4);
                    sum[t][e] += __shfl_xor_sync(~0u, sum[t][e], 8);
                    sum[t][e] += __shfl_xor_sync(~0u, sum[t][e], 16);
                    if (quad == 0) {
                        joinTop[warp][t * 8 + 2 * pos + e] = top(t, e);
                        joinSum[warp][t * 8 + 2 * pos + e] = sum[t][e];
                    }
                }
            }
            __syncthreads();
            float weight[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = t * 8 + 2 * pos + e;
                    const float best = fmaxf(fmaxf(joinTop[0][r], joinTop[1][r]), fmaxf(joinTop[2][r], joinTop[3][r]));
                    weight[t][e] = best == -INFINITY ? 0.0f : Exp2(top(t, e) - best);
                }
            }
            // A part of the columns at a time, each warp that adds up in the same buffer at another one: the order of the additions is fixed.
            constexpr int kTurns = kWarps / X::kJoins;
            float *mine = join + warp / kTurns * (kRows * X::kJoinRow);
#pragma unroll
            for (int turn = 0; turn < kTurns; turn++) {
                const int part = (warp + turn) % kTurns;
#pragma unroll
                for (int s = 0; s < kSteps; s++) {
                    if (s / (kSteps / kTurns) == part) {
#pragma unroll
                        for (int t = 0; t < NT; t++) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int d = s * 16 + quad + (e >> 1) * 8;
                                float *place = mine + (t * 8 + 2 * pos + (e & 1)) * X::kJoinRow + d;
                                const float y = acc[t][s][e] * weight[t][e & 1];
                                *place = turn == 0 ? y : *place + y;
                            }
                        }
                    }
                }
                __syncthreads();
            }
            const int kvh = done.hg / GT, g0 = (done.hg % GT) * kRows;
            const bool complete = rowEnd && rowStart == 0;
            const int which = rowStart != 0 ? 0 : 1;
            const float vs = kWide ? a.vScale[kvh] : 1.0f;
            for (int i = tid; i < kRows * (D / 8); i += kThreads) {
                const int r = i / (D / 8), d = (i % (D / 8)) * 8;
                const float best = fmaxf(fmaxf(joinTop[0][r], joinTop[1][r]), fmaxf(joinTop[2][r], joinTop[3][r]));
                float all = 0;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    all += best == -INFINITY ? joinSum[w][r] : joinSum[w][r] * Exp2(joinTop[w][r] - best);
                }
                float4 y = *(const float4 *)(join + r * X::kJoinRow + d), z = *(const float4 *)(join + r * X::kJoinRow + d + 4);
                if (X::kJoins == 2) {
                    const float *other = join + kRows * X::kJoinRow + r * X::kJoinRow + d;
                    const float4 y1 = *(const float4 *)other, z1 = *(const float4 *)(other + 4);
                    y = make_float4(y.x + y1.x, y.y + y1.y, y.z + y1.z, y.w + y1.w);
                    z = make_float4(z.x + z1.x, z.y + z1.y, z.z + z1.z, z.w + z1.w);
                }
                if (!complete) {
                    float *ws = Partial<D, kRows>((float *)a.workspace, blockIdx.x, which);
                    if (d == 0) {
                        *(float2 *)(ws + r * kPartialFloats) = make_float2(best, all);
                    }
                    ws += kRows * kPartialFloats + r * D + d;
                    *(float4 *)ws = y;
                    *(float4 *)(ws + 4) = z;
                } else if (g0 + r < a.group) {
                    const int h = kvh * a.group + g0 + r;
                    const float scale = (all != 0 ? 1.0f / all : 0.0f) * vs;
                    uint4 packed = make_uint4(Pack2<Q>(y.x * scale, y.y * scale), Pack2<Q>(y.z * scale, y.w * scale), Pack2<Q>(z.x * scale, z.y * scale),
                                              Pack2<Q>(z.z * scale, z.w * scale));
                    *(uint4 *)((Q *)a.out + (size_t)done.b * a.outStride[0] + (size_t)h * a.outStride[1] + d) = packed;
                    if (a.lse != nullptr && d == 0) {
                        a.lse[(size_t)done.b * a.kvHeads * a.group + h] = best * kLn2 + logf(all);
                    }
                }
            }
            if (!complete && tid == 0) {
                ((int2 *)a.marks)[blockIdx.x * 2 + which] = make_int2(done.b, done.hg);
            }
            __syncthreads();
            open = true;
        }
    }
    CpWait<0>();
}

// One CTA for each row that is continued behind CTA blockIdx.x of the first kernel: that one's second partial result and the first ones
// of the CTAs behind it, as long as they are of the same row. A thread owns eight columns of a query head.
template <typename Q, int D, bool WIDE, int NT>
__global__ void __launch_bounds__(NT * D * kJoinGroups<NT>) mf_decode_join_kernel(const __grid_constant__ mf_decode_attention_args_t a, int ctas)
{
    constexpr int kRows = 8 * NT;
    GridDependency();
    const int2 *marks = (const int2 *)a.marks;
    const int c = blockIdx.x;
    const int group = threadIdx.x / (NT * D), r = threadIdx.x % (NT * D) / (D / 8), d = (threadIdx.x % (D / 8)) * 8;
    // The first mark of each thread and the first part of each group are fetched before it is known how many there are (500 tokens each of 8 sequences 11.8 ->
    // 10.8 us); whatever stands there otherwise is left alone.
    const int2 row = marks[2 * c + 1];
    const int near = c + 1 + (int)threadIdx.x;
    const int2 mark0 = near < ctas ? marks[2 * near] : make_int2(-1, -1);
    const float *ws0 = Partial<D, kRows>((float *)a.workspace, min(c + group, ctas - 1), group == 0 ? 1 : 0);
    const float2 ms0 = *(const float2 *)(ws0 + r * kPartialFloats);
    const float4 x0 = *(const float4 *)(ws0 + kRows * kPartialFloats + r * D + d), y0 = *(const float4 *)(ws0 + kRows * kPartialFloats + r * D + d + 4);
    if (row.x < 0) {
        return;
    }
    const int GT = (a.group + kRows - 1) / kRows, kvh = row.y / GT, g = (row.y % GT) * kRows;
    // the CTAs behind that hold a part of the row: all marks at once
    __shared__ int behind;
    if (threadIdx.x == 0) {
        behind = ctas;
    }
    __syncthreads();
    for (int i = near; i < ctas; i += blockDim.x) {
        const int2 m = i == near ? mark0 : marks[2 * i];
        if (m.x != row.x || m.y != row.y) {
            atomicMin(&behind, i);
        }
    }
    __syncthreads();
    const int n = behind - c;
    const bool any = group < n;
    float best = any ? ms0.x : -INFINITY, all = any ? ms0.y : 0;
    float out[8] = {x0.x, x0.y, x0.z, x0.w, y0.x, y0.y, y0.z, y0.w};
    if (!any) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[j] = 0;
        }
    }
    constexpr int kAhead = 4;  // parts whose loads are in flight together
    for (int i = group + kJoinGroups<NT>; i < n; i += kAhead * kJoinGroups<NT>) {
        float2 ms[kAhead];
        float4 x[kAhead], y[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const float *ws = Partial<D, kRows>((float *)a.workspace, c + min(i + u * kJoinGroups<NT>, n - 1), 0);
            ms[u] = *(const float2 *)(ws + r * kPartialFloats);
            x[u] = *(const float4 *)(ws + kRows * kPartialFloats + r * D + d);
            y[u] = *(const float4 *)(ws + kRows * kPartialFloats + r * D + d + 4);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (i + u * kJoinGroups<NT> < n) {
                const float next = fmaxf(best, ms[u].x), base = next == -INFINITY ? 0.0f : next;
                const float keep = Exp2(best - base), weight = Exp2(ms[u].x - base);
                const float v[8] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x, y[u].y, y[u].z, y[u].w};
                best = next;
                all = all * keep + ms[u].y * weight;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    out[j] = out[j] * keep + v[j] * weight;
                }
            }
        }
    }
    __shared__ float tops[kJoinGroups<NT>][kRows], sums[kJoinGroups<NT>][kRows];
    __shared__ __align__(16) float values[kJoinGroups<NT>][kRows * D];
    if (d == 0) {
        tops[group][r] = best;
        sums[group][r] = all;
    }
    *(float4 *)&values[group][r * D + d] = make_float4(out[0], out[1], out[2], out[3]);
    *(float4 *)&values[group][r * D + d + 4] = make_float4(out[4], out[5], out[6], out[7]);
    __syncthreads();
    if (group != 0 || g + r >= a.group) {
        return;
    }
#pragma unroll
    for (int i = 1; i < kJoinGroups<NT>; i++) {
        const float next = fmaxf(best, tops[i][r]), base = next == -INFINITY ? 0.0f : next;
        const float keep = Exp2(best - base), weight = Exp2(tops[i][r] - base);
        best = next;
        all = all * keep + sums[i][r] * weight;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[j] = out[j] * keep + values[i][r * D + d + j] * weight;
        }
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

// Eights of query heads that are worked on together: two where the group has more than eight, which read a key once for both.
int Eights(int group) { return group > 8 ? 2 : 1; }

int Ctas(int B, int kvHeads, int group, long long capacity)
{
    const int sms = mf_k_sm_count(), rows = 8 * Eights(group);
    const long long tiles = (long long)B * kvHeads * ((group + rows - 1) / rows) * ((capacity + 63) / 64),  // tiles have 64 keys or more
                    most = (long long)kMostCtasPerSm * (sms > 0 ? sms : 1);
    return (int)(tiles < most ? (tiles > 1 ? tiles : 1) : most);
}

size_t PartialBytes(int ctas, int group, int D) { return (size_t)ctas * 2 * 8 * Eights(group) * (D + kPartialFloats) * sizeof(float); }

template <typename Q, typename C, int D, int NT>
int Launch(const mf_decode_attention_args_t &a, int ctas, cudaStream_t stream)
{
    using X = Cfg<C, D, NT>;
    constexpr uint32_t kSmem = X::kSmem;
    static_assert(X::kCtasPerSm <= kMostCtasPerSm, "the workspace has room for the partial results of that many");
    const int room = X::kCtasPerSm * mf_k_sm_count();
    ctas = ctas < room ? ctas : room;
    if (!mf::AllowSmem<mf_decode_attention_kernel<Q, C, D, NT>>(kSmem)) {
        return MF_K_LAUNCH_FAILED;
    }
    if (mf::sm100::LaunchDependent(mf_decode_attention_kernel<Q, C, D, NT>, ctas, kThreads, kSmem, stream, a) != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    // rows of at most kWholeKeys keys are never cut
    if ((long long)a.tableWidth * a.pageSize > kWholeKeys &&
        mf::sm100::LaunchDependent(mf_decode_join_kernel<Q, D, sizeof(C) == 1, NT>, ctas, NT * D * kJoinGroups<NT>, 0, stream, a, ctas) != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    return MF_K_OK;
}

template <typename Q, typename C>
int LaunchDim(const mf_decode_attention_args_t &a, int D, int ctas, cudaStream_t stream)
{
    if (Eights(a.group) == 1) {
        return D == 64 ? Launch<Q, C, 64, 1>(a, ctas, stream) : Launch<Q, C, 128, 1>(a, ctas, stream);
    }
    return D == 64 ? Launch<Q, C, 64, 2>(a, ctas, stream) : Launch<Q, C, 128, 2>(a, ctas, stream);
}

}  // namespace

extern "C" size_t mf_k_decode_attention_workspace(int B, int kvHeads, int group, int D, long long capacity)
{
    if (B <= 0 || kvHeads <= 0 || group <= 0 || (D != 64 && D != 128) || capacity <= kWholeKeys) {
        return 0;  // no row is cut
    }
    const int ctas = Ctas(B, kvHeads, group, capacity);
    return PartialBytes(ctas, group, D) + (size_t)ctas * 2 * sizeof(int2);
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
    // key / pageSize = umulhi(key, pageMagic) >> pageShift for keys below 2^31: the magic number of T. Granlund, P. Montgomery, "Division by
    // invariant integers using multiplication", 1994, with l = ceil(log2(pageSize)) and one bit less, as the keys have 31. A
    // page size of 1 would need 33 bits.
    a.pageShift = 0;
    while ((1ll << (a.pageShift + 1)) < a.pageSize) {
        a.pageShift++;
    }
    a.pageMagic = a.pageSize == 1 ? 0 : (uint32_t)(((1ull << (32 + a.pageShift)) + a.pageSize - 1) / a.pageSize);
    const long long capacity = (long long)a.tableWidth * a.pageSize;
    const int ctas = Ctas(a.B, a.kvHeads, a.group, capacity);
    if (capacity <= kWholeKeys) {
        a.workspace = a.marks = nullptr;
    } else if (a.workspace == nullptr || a.workspaceBytes < mf_k_decode_attention_workspace(a.B, a.kvHeads, a.group, D, capacity)) {
        return MF_K_INVALID;
    } else {
        a.marks = (unsigned char *)a.workspace + PartialBytes(ctas, a.group, D);
    }
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
