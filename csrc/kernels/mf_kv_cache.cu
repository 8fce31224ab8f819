// Book-keeping and data movement of a paged key-value cache, on the device, so that a serving loop needs no host round trip and can be
// captured into a CUDA graph. A page holds `pageSize` tokens of every layer, [layer][page][key, value][head][slot][dim]; refs counts the
// sequences that hold a page. What is handed out is always the lowest-numbered free page, so results do not depend on timing.
//
//   write    new tokens' keys and values into their slots of one layer, as they are or quantised to e4m3 with a scale per head
//   reserve  pages and slots for new tokens; a shared, partly filled last page is copied first (its filled rows, all layers)
//   fork     a sequence that shares another one's pages
//   free     sequences dropped, pages without a holder free
//   compact  the n pages in use moved to the places [0, n): those behind go, in ascending order, into the free ones before
//
// The planning steps run in one CTA (they are scans over a few ten thousand words, which cost less than a grid-wide barrier); what moves
// pages is a kernel of its own behind it, spread over all SMs.
#include "mf/device/mf_shm_device.cuh"
#include "mf_attention.cuh"
#include "mf_copy_device.cuh"
#include "mf_kernels.h"
#include "mf_launch.cuh"
#include "mf_sm100_ptx.cuh"

namespace {

using namespace mf::attn;
using mf::sm100::GridDependency;
using mf::sm100::LaunchDependent;

constexpr int kPlanThreads = 1024;
constexpr int kMaxSeqs = MF_KV_MAX_SEQS;

__device__ __forceinline__ int Pages(int tokens, int pageSize) { return tokens / pageSize + (tokens % pageSize != 0); }

// ---------------------------------------------------------------------------------------------- write
// A thread moves 16 values of a key row and of the value row beside it. Bound by memory: what it reads and writes once.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) mf_kv_write_kernel(const __grid_constant__ mf_kv_write_args_t a)
{
    GridDependency();
    const int chunks = a.dim / 16, perToken = a.kvHeads * chunks;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)a.tokens * perToken) {
        return;
    }
    const int token = (int)(i / perToken), rest = (int)(i % perToken), head = rest / chunks, d = rest % chunks * 16;
    const long long slot = a.slots[token];
    if (slot < 0) {
        return;
    }
    if (slot >= (long long)a.pages * a.pageSize) {
        *a.status = MF_DEV_ERR_BOUNDS;
        return;
    }
    const T *src[2] = {(const T *)a.k + (size_t)token * a.kStride[0] + (size_t)head * a.kStride[1] + d,
                       (const T *)a.v + (size_t)token * a.vStride[0] + (size_t)head * a.vStride[1] + d};
    uint4 x[2][2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        x[w][0] = mf::dev::LdStream16(src[w]);
        x[w][1] = mf::dev::LdStream16(src[w] + 8);
    }
    const size_t page = (size_t)(slot / a.pageSize), off = (size_t)(slot % a.pageSize);
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const size_t at = (((page * 2 + w) * a.kvHeads + head) * a.pageSize + off) * a.dim + d;
        if (E4M3) {
            const float inv = 1.0f / (w == 0 ? a.kScale : a.vScale)[head];
            const uint32_t in[8] = {x[w][0].x, x[w][0].y, x[w][0].z, x[w][0].w, x[w][1].x, x[w][1].y, x[w][1].z, x[w][1].w};
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 lo = Unpack2<T>(in[2 * j]), hi = Unpack2<T>(in[2 * j + 1]);
                unsigned short p, q;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(lo.y * inv), "f"(lo.x * inv));
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(hi.y * inv), "f"(hi.x * inv));
                out[j] = (uint32_t)p | (uint32_t)q << 16;
            }
            *(uint4 *)((unsigned char *)a.data + at) = make_uint4(out[0], out[1], out[2], out[3]);
        } else {
            *(uint4 *)((T *)a.data + at) = x[w][0];
            *(uint4 *)((T *)a.data + at + 8) = x[w][1];
        }
    }
}

// ---------------------------------------------------------------------------------------------- scans of one CTA
// Sums of all threads before this one and of all; two 32-bit counts travel in one 64-bit word.
__device__ __forceinline__ unsigned long long BlockScan(unsigned long long x, unsigned long long *shared, unsigned long long &total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long up = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long y = __shfl_up_sync(~0u, up, d);
        up += lane >= d ? y : 0;
    }
    __syncthreads();  // the words of the scan before have been read
    if (lane == 31) {
        shared[warp] = up;
    }
    __syncthreads();
    unsigned long long w = shared[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long y = __shfl_up_sync(~0u, w, d);
        w += lane >= d ? y : 0;
    }
    total = __shfl_sync(~0u, w, 31);
    const unsigned long long before = __shfl_sync(~0u, w, warp == 0 ? 0 : warp - 1);
    return up - x + (warp == 0 ? 0 : before);
}

// Calls use(page, used, free pages before it, pages in use before it) for the pages [0, pages) in steps of 4096 until `enough` free ones are seen.
template <typename Use>
__device__ __forceinline__ void ScanPages(const int *refs, int pages, int enough, unsigned long long *shared, Use use)
{
    unsigned long long seen = 0;
    for (int base = 0; base < pages && (int)(seen & 0xffffffffu) < enough; base += 4 * kPlanThreads) {
        const int p = base + 4 * (int)threadIdx.x;
        int r[4] = {1, 1, 1, 1};
        if (p + 4 <= pages) {
            const int4 v = *(const int4 *)(refs + p);
            r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
        } else {
            for (int j = 0; j < 4; j++) {
                r[j] = p + j < pages ? refs[p + j] : 1;
            }
        }
        unsigned long long mine = 0, total;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mine += r[j] > 0 ? (p + j < pages ? 1ull << 32 : 0) : 1;
        }
        unsigned long long at = seen + BlockScan(mine, shared, total);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (p + j < pages) {
                use(p + j, r[j] > 0, (int)(at & 0xffffffffu), (int)(at >> 32));
                at += r[j] > 0 ? 1ull << 32 : 1;
            }
        }
        seen += total;
    }
}

// ---------------------------------------------------------------------------------------------- reserve
// The plan that the first kernel leaves for the second, in the workspace: {1 if the call goes through, tokens}, then per request the first
// token's index, the length before, and the page to copy from and to (-1: none); then the free pages.
struct Plan {
    int *head, *firstToken, *old, *from, *to, *need, *free;
    __device__ __forceinline__ Plan(int *ws, int n) : head(ws), firstToken(ws + 4), old(firstToken + n), from(old + n), to(from + n), need(to + n), free(need + n) {}
};
constexpr int kPlanWords = 5;

__global__ void __launch_bounds__(kPlanThreads) mf_kv_reserve_plan_kernel(const __grid_constant__ mf_kv_cache_t c, const int *rows, const int *counts, int n,
                                                                        long long room, int *ws)
{
    extern __shared__ uint32_t named[];  // a bit for each sequence
    __shared__ unsigned long long words[32];
    __shared__ int bad;
    GridDependency();
    const int tid = threadIdx.x, ps = c.pageSize;
    Plan plan(ws, n);
    for (int i = tid; i < (c.seqs + 31) / 32; i += kPlanThreads) {
        named[i] = 0;
    }
    if (tid == 0) {
        bad = 0;
    }
    __syncthreads();
    const int per = (n + kPlanThreads - 1) / kPlanThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    unsigned long long minePages = 0, mineTokens = 0, pages, tokens;
    for (int i = i0; i < i1; i++) {
        const int row = rows[i], count = counts[i];
        int need = 0, from = -1, old = 0;
        if (row < 0 || row >= c.seqs || count < 0 || count > room || (atomicOr(&named[row >> 5], 1u << (row & 31)) >> (row & 31) & 1)) {
            bad = 1;
        } else {
            old = c.lengths[row];
            if (old < 0 || (long long)old + count > (long long)c.tableWidth * ps) {
                bad = 1;
            } else {
                need = Pages(old + count, ps) - Pages(old, ps);
                if (count > 0 && old % ps != 0) {
                    const int last = c.table[(size_t)row * c.tableWidth + old / ps];
                    if (last < 0 || last >= c.pages) {
                        bad = 1;
                    } else if (c.refs[last] > 1) {
                        from = last;
                        need++;
                    }
                }
                minePages += need;
                mineTokens += count;
            }
        }
        plan.old[i] = old;
        plan.from[i] = from;
        plan.need[i] = need;
    }
    const unsigned long long pagesBefore = BlockScan(minePages, words, pages), tokensBefore = BlockScan(mineTokens, words, tokens);
    if ((long long)tokens > room) {
        bad = 1;
    }
    __syncthreads();
    if (!bad) {
        unsigned page = (unsigned)pagesBefore, token = (unsigned)tokensBefore;  // no more than `room`, and two for each request
        for (int i = i0; i < i1; i++) {  // `need` becomes the first of the request's free pages
            const unsigned need = plan.need[i];
            plan.need[i] = page;
            plan.firstToken[i] = token;
            page += need;
            token += counts[i];
        }
        __shared__ int found;
        if (tid == 0) {
            found = 0;
        }
        ScanPages(c.refs, c.pages, (int)pages, words, [&](int p, bool used, int rank, int) {
            if (!used && rank < (int)pages) {
                plan.free[rank] = p;
                if (rank + 1 == (int)pages) {
                    found = 1;
                }
            }
        });
        __syncthreads();
        if (pages != 0 && !found && tid == 0) {
            bad = 1;
        }
        __syncthreads();
    }
    const bool ok = bad == 0;
    if (tid == 0) {
        plan.head[0] = ok;
        plan.head[1] = (int)tokens;
        if (!ok) {
            *c.status = MF_DEV_ERR_BOUNDS;
        }
    }
    if (!ok) {
        return;
    }
    for (int k = tid; k < (int)pages; k += kPlanThreads) {
        int lo = 0, hi = n;  // the last request whose first page is not behind k: requests without pages share their number with the next
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (plan.need[mid] <= k ? lo : hi) = mid;
        }
        const int row = rows[lo], old = plan.old[lo], copied = plan.from[lo] >= 0, j = k - plan.need[lo];
        c.table[(size_t)row * c.tableWidth + Pages(old, ps) + j - copied] = plan.free[k];
        c.refs[plan.free[k]] = 1;
    }
    for (int i = i0; i < i1; i++) {
        plan.to[i] = plan.from[i] >= 0 ? plan.free[plan.need[i]] : -1;
        if (plan.from[i] >= 0) {
            atomicSub(&c.refs[plan.from[i]], 1);
        }
        c.lengths[rows[i]] = plan.old[i] + counts[i];
    }
}

__global__ void __launch_bounds__(256) mf_kv_reserve_apply_kernel(const __grid_constant__ mf_kv_cache_t c, const int *rows, int n, long long room, int *ws,
                                                                  long long *slots)
{
    GridDependency();
    const Plan plan(ws, n);
    const bool ok = plan.head[0] != 0;
    const int tokens = plan.head[1], ps = c.pageSize;
    for (long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x; t < room; t += (long long)gridDim.x * blockDim.x) {
        long long slot = -1;
        if (ok && t < tokens) {
            int lo = 0, hi = n;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                (plan.firstToken[mid] <= t ? lo : hi) = mid;
            }
            const int at = plan.old[lo] + (int)(t - plan.firstToken[lo]);
            slot = (long long)c.table[(size_t)rows[lo] * c.tableWidth + at / ps] * ps + at % ps;
        }
        slots[t] = slot;
    }
    if (!ok) {
        return;
    }
    // the filled rows of the pages that were shared: a warp for each (request, layer, key or value, head)
    const int lane = threadIdx.x & 31, perPage = 2 * c.kvHeads;
    const long long units = (long long)n * c.layers * perPage;
    const size_t run = (size_t)ps * c.rowBytes;
    for (long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; u < units; u += (long long)gridDim.x * blockDim.x >> 5) {
        const int i = (int)(u / (c.layers * perPage)), rest = (int)(u % (c.layers * perPage)), layer = rest / perPage, part = rest % perPage;
        if (plan.from[i] < 0) {
            continue;
        }
        const size_t first = (size_t)layer * c.pages;
        mf::dev::CopyVec<4, 32>((uint4 *)((unsigned char *)c.data + ((first + plan.to[i]) * perPage + part) * run),
                                (const uint4 *)((const unsigned char *)c.data + ((first + plan.from[i]) * perPage + part) * run),
                                (unsigned)(plan.old[i] % ps) * c.rowBytes / 16, lane);
    }
}

// ---------------------------------------------------------------------------------------------- fork, free
// A CTA for each pair. A pair is refused, with the status set, if its numbers are out of range, its destination is in use, was named by
// a pair before it, or is a source of this call: then no CTA reads a length that another one writes.
__global__ void __launch_bounds__(128) mf_kv_fork_kernel(const __grid_constant__ mf_kv_cache_t c, const int *src, const int *dst, int n)
{
    GridDependency();
    const int i = blockIdx.x, from = src[i], to = dst[i], tid = threadIdx.x;
    int bad = from < 0 || from >= c.seqs || to < 0 || to >= c.seqs;
    for (int j = tid; j < n; j += blockDim.x) {
        bad |= (dst[j] == to && j < i) || dst[j] == from || src[j] == to;
    }
    const int length = bad ? 0 : c.lengths[from];
    bad |= !bad && (c.lengths[to] != 0 || length < 0 || length > (long long)c.tableWidth * c.pageSize);
    if (__syncthreads_or(bad)) {  // every thread has read the lengths
        if (tid == 0) {
            *c.status = MF_DEV_ERR_BOUNDS;
        }
        return;
    }
    const int *in = c.table + (size_t)from * c.tableWidth;
    int *out = c.table + (size_t)to * c.tableWidth;
    for (int j = tid; j < Pages(length, c.pageSize); j += blockDim.x) {
        const int p = in[j];
        out[j] = p;
        if (p >= 0 && p < c.pages) {
            atomicAdd(&c.refs[p], 1);
        }
    }
    if (tid == 0) {
        c.lengths[to] = length;
    }
}

// A CTA for each sequence; one that is named twice is free the second time.
__global__ void __launch_bounds__(128) mf_kv_free_kernel(const __grid_constant__ mf_kv_cache_t c, const int *rows)
{
    __shared__ int length;
    GridDependency();
    const int row = rows[blockIdx.x], tid = threadIdx.x;
    if (row < 0 || row >= c.seqs) {
        if (tid == 0) {
            *c.status = MF_DEV_ERR_BOUNDS;
        }
        return;
    }
    if (tid == 0) {
        length = atomicExch(&c.lengths[row], 0);
    }
    __syncthreads();
    int *entry = c.table + (size_t)row * c.tableWidth;
    const int used = length <= 0 ? 0 : min(Pages(length, c.pageSize), c.tableWidth);
    for (int j = tid; j < used; j += blockDim.x) {
        const int p = entry[j];
        entry[j] = -1;
        if (p < 0 || p >= c.pages || atomicSub(&c.refs[p], 1) <= 0) {
            *c.status = MF_DEV_ERR_BOUNDS;  // a table or counts that were not this cache's doing
        }
    }
}

// ---------------------------------------------------------------------------------------------- compact
// Workspace: {moves}, then per move the page it comes from and the place it goes to.
__global__ void __launch_bounds__(kPlanThreads) mf_kv_compact_plan_kernel(const __grid_constant__ mf_kv_cache_t c, int *remap, int *ws)
{
    __shared__ unsigned long long words[32];
    GridDependency();
    unsigned long long mine = 0, total;
    for (int p = threadIdx.x; p < c.pages; p += kPlanThreads) {
        mine += c.refs[p] > 0;
    }
    BlockScan(mine, words, total);
    const int used = (int)total;
    int *from = ws + 4, *to = from + c.pages / 2;
    __shared__ int moves;
    if (threadIdx.x == 0) {
        moves = 0;
    }
    ScanPages(c.refs, c.pages, 0x7fffffff, words, [&](int p, bool live, int freeBefore, int liveBefore) {
        if (p < used) {
            remap[p] = live ? p : -1;
            if (!live) {
                to[freeBefore] = p;
            }
            if (p + 1 == used) {
                moves = freeBefore + !live;
            }
        } else if (live) {
            // the live pages before it are those of [0, used), which lack as many as there are moves, and the sources before it
            from[c.pages / 2 - 1 - (used - 1 - liveBefore)] = p;
        } else {
            remap[p] = -1;
        }
    });
    __syncthreads();
    // sources were counted from the end: they lie in the last `moves` words
    const int m = moves;
    for (int k = threadIdx.x; k < m; k += kPlanThreads) {
        const int s = from[c.pages / 2 - m + k], d = to[k];
        remap[s] = d;
        c.refs[d] = c.refs[s];
        c.refs[s] = 0;
    }
    if (threadIdx.x == 0) {
        ws[0] = m;
    }
}

__global__ void __launch_bounds__(256) mf_kv_compact_move_kernel(const __grid_constant__ mf_kv_cache_t c, const int *remap, const int *ws)
{
    GridDependency();
    const int m = ws[0], *from = ws + 4 + c.pages / 2 - m, *to = ws + 4 + c.pages / 2;
    const size_t bytes = (size_t)2 * c.kvHeads * c.pageSize * c.rowBytes;
    // Eight vectors of a thread in flight and two CTAs per SM: 185 us for 537 MB moved, 197 with four and eight, whose reads and writes mix more.
    constexpr int kTrip = 16 * 256 * 8;
    const int pieces = (int)((bytes + kTrip - 1) / kTrip);
    for (long long u = blockIdx.x; u < (long long)m * c.layers * pieces; u += gridDim.x) {
        const int piece = (int)(u % pieces), layer = (int)(u / pieces % c.layers), k = (int)(u / pieces / c.layers);
        const size_t off = (size_t)piece * kTrip, left = bytes - off, first = (size_t)layer * c.pages;
        mf::dev::CopyVec<8, 256>((uint4 *)((unsigned char *)c.data + (first + to[k]) * bytes + off),
                                 (const uint4 *)((const unsigned char *)c.data + (first + from[k]) * bytes + off),
                                 (unsigned)((left < kTrip ? left : kTrip) / 16), threadIdx.x);
    }
    const long long entries = (long long)c.seqs * c.tableWidth;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < entries; i += (long long)gridDim.x * blockDim.x) {
        const int p = c.table[i];
        if (p >= 0 && p < c.pages) {
            c.table[i] = remap[p];
        }
    }
}

bool Fine(const mf_kv_cache_t *c)
{
    return c != nullptr && c->data != nullptr && c->table != nullptr && c->lengths != nullptr && c->refs != nullptr && c->status != nullptr && c->layers > 0 &&
           c->pages > 0 && c->pageSize > 0 && c->kvHeads > 0 && c->rowBytes > 0 && c->rowBytes % 16 == 0 && c->seqs > 0 && c->seqs <= kMaxSeqs &&
           c->tableWidth >= 0 && (long long)c->tableWidth * c->pageSize <= 0x7fffff00ll && (uintptr_t)c->refs % 16 == 0 && (uintptr_t)c->data % 16 == 0;
}

int Status(cudaError_t e)
{
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return MF_K_LAUNCH_FAILED;
    }
    return MF_K_OK;
}

unsigned Spread(long long ctas, int perSm)
{
    const int sms = mf_k_sm_count();
    const long long most = (long long)perSm * (sms > 0 ? sms : 1);
    return (unsigned)(ctas < 1 ? 1 : ctas < most ? ctas : most);
}

}  // namespace

extern "C" int mf_k_kv_write(const mf_kv_write_args_t *a, int srcType, int cacheType, mf_stream_t stream)
{
    if (a == nullptr || a->tokens < 0 || a->kvHeads <= 0 || a->dim <= 0 || a->dim % 16 != 0 || a->pages <= 0 || a->pageSize <= 0 || a->status == nullptr ||
        (srcType != MF_K_BF16 && srcType != MF_K_FP16) || (cacheType != srcType && cacheType != MF_K_E4M3) ||
        (cacheType == MF_K_E4M3 && (a->kScale == nullptr || a->vScale == nullptr))) {
        return MF_K_INVALID;
    }
    if (a->tokens == 0) {
        return MF_K_OK;
    }
    const long long ctas = ((long long)a->tokens * a->kvHeads * (a->dim / 16) + 255) / 256;
    if (ctas > 0x7fffffffll) {
        return MF_K_TOO_LARGE;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    if (srcType == MF_K_BF16) {
        return Status(cacheType == MF_K_E4M3 ? LaunchDependent(mf_kv_write_kernel<__nv_bfloat16, true>, (unsigned)ctas, 256, 0, s, *a)
                                             : LaunchDependent(mf_kv_write_kernel<__nv_bfloat16, false>, (unsigned)ctas, 256, 0, s, *a));
    }
    return Status(cacheType == MF_K_E4M3 ? LaunchDependent(mf_kv_write_kernel<__half, true>, (unsigned)ctas, 256, 0, s, *a)
                                         : LaunchDependent(mf_kv_write_kernel<__half, false>, (unsigned)ctas, 256, 0, s, *a));
}

extern "C" size_t mf_k_kv_reserve_workspace(int n, long long room, int pageSize)
{
    return n <= 0 || room < 0 || pageSize <= 0 ? 0 : (4 + (size_t)kPlanWords * n + (size_t)(room / pageSize) + 2 * (size_t)n) * sizeof(int);
}

extern "C" int mf_k_kv_reserve(const mf_kv_cache_t *c, const int *rows, const int *counts, int n, long long room, long long *slots, void *workspace,
                               mf_stream_t stream)
{
    if (!Fine(c) || n < 0 || n > c->seqs || room < 0 || room > 0x7fffffffll || (n > 0 && workspace == nullptr)) {
        return MF_K_INVALID;
    }
    if (n == 0) {
        return MF_K_OK;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    const int rc = Status(LaunchDependent(mf_kv_reserve_plan_kernel, 1, kPlanThreads, ((size_t)c->seqs + 31) / 32 * 4, s, *c, rows, counts, n, room, (int *)workspace));
    if (rc != MF_K_OK) {
        return rc;
    }
    const long long ctas = ((long long)n * c->layers * 2 * c->kvHeads + 7) / 8, forSlots = (room + 255) / 256;
    return Status(LaunchDependent(mf_kv_reserve_apply_kernel, Spread(ctas > forSlots ? ctas : forSlots, 8), 256, 0, s, *c, rows, n, room, (int *)workspace, slots));
}

extern "C" int mf_k_kv_fork(const mf_kv_cache_t *c, const int *src, const int *dst, int n, mf_stream_t stream)
{
    if (!Fine(c) || n < 0 || n > c->seqs) {
        return MF_K_INVALID;
    }
    return n == 0 ? (int)MF_K_OK : Status(LaunchDependent(mf_kv_fork_kernel, (unsigned)n, 128, 0, (cudaStream_t)stream, *c, src, dst, n));
}

extern "C" int mf_k_kv_free(const mf_kv_cache_t *c, const int *rows, int n, mf_stream_t stream)
{
    if (!Fine(c) || n < 0) {
        return MF_K_INVALID;
    }
    return n == 0 ? (int)MF_K_OK : Status(LaunchDependent(mf_kv_free_kernel, (unsigned)n, 128, 0, (cudaStream_t)stream, *c, rows));
}

extern "C" size_t mf_k_kv_compact_workspace(int pages) { return pages <= 0 ? 0 : (4 + 2 * (size_t)(pages / 2)) * sizeof(int); }

extern "C" int mf_k_kv_compact(const mf_kv_cache_t *c, int *remap, void *workspace, mf_stream_t stream)
{
    if (!Fine(c) || remap == nullptr || workspace == nullptr) {
        return MF_K_INVALID;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    const int rc = Status(LaunchDependent(mf_kv_compact_plan_kernel, 1, kPlanThreads, 0, s, *c, remap, (int *)workspace));
    if (rc != MF_K_OK) {
        return rc;
    }
    return Status(LaunchDependent(mf_kv_compact_move_kernel, Spread(0x7fffffff, 2), 256, 0, s, *c, remap, (const int *)workspace));
}
