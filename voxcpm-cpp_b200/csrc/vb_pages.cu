// vb_pages.cu -- page operations of a paged K/V cache: extend (with copy on
// write), fork, keep (the accepted path of a draft), truncate, compact.
//
// The bookkeeping lives on the device.  Where rows move (extend, keep,
// compact) a call is a plan, one CTA that checks the requests, works out pages
// and rows and writes the new state, and a copy by all SMs that follows the
// plan's list; both are programmatic dependent launches.  A plan is four
// dependent rounds of loads and a few barriers, so it runs in few threads with
// everything that does not depend on an earlier round loaded in the first.
// (One launch for both, every CTA planning for itself and the last one to
// finish writing the state, took longer: 35 us against 22 for a step of 64
// sequences that extends, keeps and truncates.)  Fork and truncate touch only
// their own requests' table rows and add to the counts atomically (integer
// adds, so the order does not show): a column of CTAs per request.
#include "vb_common.cuh"
#include "vb_kernels.cuh"
#include "vb_tc.cuh"

#include <algorithm>
#include <climits>

namespace vb {

constexpr int PG_PLAN = 1024;        // threads of compact's plan
constexpr int PG_STEP = 256;         // threads of extend's plan: few, as barriers are part of what it costs
constexpr int PG_KEEP = 512;         // threads of keep's plan
constexpr int PG_SCAN = 16;          // counts per thread and scan step
constexpr int PG_COPY = 256;
constexpr int PG_MAX_SEQS = 16384;

// Exclusive sum over the CTA's threads; total: the sum of all.  sh: two rows
// of 32, used in turn (`turn` counts the calls), so one barrier is enough.
template <typename T>
__device__ T block_scan(T v, T (*sh)[32], int turn, T &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    T *row = sh[turn & 1];
    if (lane == 31) row[warp] = x;
    __syncthreads();
    T w = lane < warps ? row[lane] : T(0);
    const T own = __shfl_sync(0xffffffffu, w, warp);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    return __shfl_sync(0xffffffffu, w, warp) - own + x - v;
}

// First error of a call: lowest request, then lowest code.
struct PageError {
    int key;                         // request * 16 + code, INT_MAX: none
    __device__ void at(int request, int code) { atomicMin(&key, request * 16 + code); }
};

__device__ void record(const vb_pages &p, int key) {
    p.status[1] = key >> 4;
    p.status[0] = key & 15;
}

// Whether an error waits to be read, for the CTA as a whole: in a call of many
// CTAs the first may be recording the call's own while others start.  A CTA
// that sees that one leaves; one that does not finds the error itself.
__device__ bool any_error(const vb_pages &p) { return __syncthreads_or(threadIdx.x == 0 && p.status[0] != 0); }

// Which requests came second for a sequence.
__device__ void which_twice(int n, const int32_t *seqs, PageError *err) {
    for (int i = threadIdx.x; i < n; i += blockDim.x)
        for (int j = 0; j < i; j++)
            if (seqs[j] == seqs[i]) {
                err->at(i, VB_PAGES_SEQ);
                break;
            }
}

// Marks the requests' sequences in a bitmap of shared memory and reports
// those out of range or met before.
__device__ void check_seqs(const vb_pages &p, int n, const int32_t *seqs, uint32_t *bits, PageError *err) {
    for (int i = threadIdx.x; i < (p.n_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    bool twice = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i];
        if (s < 0 || s >= p.n_seqs) err->at(i, VB_PAGES_SEQ);
        else twice |= atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u;
    }
    if (__syncthreads_or(twice)) which_twice(n, seqs, err);
}

struct PageJob {                     // rows 0 .. rows-1 of page src, in every layer, to page dst
    int src, dst, rows, pad;
};

// Which of this thread's PG_SCAN pages from `base` on are free.
__device__ __forceinline__ uint32_t free_bits(const vb_pages &p, int base) {
    const int q0 = base + threadIdx.x * PG_SCAN;
    uint32_t bits = 0;
    if (q0 + PG_SCAN <= p.n_pages) {
#pragma unroll
        for (int j = 0; j < PG_SCAN; j += 4) {
            const int4 r = *reinterpret_cast<const int4 *>(p.refs + q0 + j);
            bits |= (uint32_t)(r.x == 0) << j | (uint32_t)(r.y == 0) << (j + 1) | (uint32_t)(r.z == 0) << (j + 2) |
                    (uint32_t)(r.w == 0) << (j + 3);
        }
    } else {
        for (int j = 0; j < PG_SCAN; j++)
            if (q0 + j < p.n_pages && p.refs[q0 + j] == 0) bits |= 1u << j;
    }
    return bits;
}

// Calls take(rank, page) for the first `total` free pages, lowest numbers
// first, and returns how many there are (up to at least total).  here: the
// free_bits of the first step.
template <typename Take>
__device__ int free_pages(const vb_pages &p, int total, uint32_t here, int (*scan)[32], int &turn, Take take) {
    int found = 0;
    for (int base = 0; base < p.n_pages && found < total; base += blockDim.x * PG_SCAN) {
        if (base) here = free_bits(p, base);
        int step;
        int k = found + block_scan(__popc(here), scan, turn++, step);
        const int q0 = base + threadIdx.x * PG_SCAN;
        for (uint32_t b = here; b && k < total; b &= b - 1) take(k++, q0 + __ffs(b) - 1);
        found += step;
    }
    return found;
}

// ws: [0] number of jobs, [4 ..] jobs.
__global__ void __launch_bounds__(PG_STEP) pages_extend_plan(vb_pages p, int n, const int32_t *seqs, const int32_t *rows,
                                                             int *ws) {
    extern __shared__ int sm[];
    __shared__ int scan[2][32];
    __shared__ long long scan2[2][32];
    __shared__ PageError err;
    // per request: the partly filled page that it shares and leaves (-1: none),
    // the rank of its first new page, its length
    int *last = sm, *first = sm + n, *length = sm + 2 * n;
    uint32_t *bits = reinterpret_cast<uint32_t *>(sm + 3 * n);
    PageJob *jobs = reinterpret_cast<PageJob *>(ws + 4);
    const int P = p.page_rows;
    if (threadIdx.x == 0) err.key = INT_MAX;
    for (int i = threadIdx.x; i < (p.n_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
    pdl_trigger();
    pdl_wait();
    const bool held = p.status[0] != 0;                       // an error waits to be read: nothing changes
    const uint32_t free0 = free_bits(p, 0);
    __syncthreads();
    bool twice = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i], r = rows[i];
        last[i] = -1;
        if (s < 0 || s >= p.n_seqs) {
            err.at(i, VB_PAGES_SEQ);
            continue;
        }
        const int len = p.length[s];
        twice |= atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u;
        length[i] = len;
        if (r < 0) err.at(i, VB_PAGES_COUNT);
        else if (len < 0 || (int64_t)len + r > (int64_t)p.max_pages * P) err.at(i, VB_PAGES_LONG);
        else if (r > 0 && len % P) {
            const int pg = p.table[(int64_t)s * p.max_pages + len / P];
            if (pg < 0 || pg >= p.n_pages) err.at(i, VB_PAGES_TABLE);
            else if (p.refs[pg] > 1) last[i] = pg;
        }
    }
    if (__syncthreads_or(twice)) {
        which_twice(n, seqs, &err);
        __syncthreads();
    }
    if (threadIdx.x == 0) ws[0] = 0;
    if (err.key != INT_MAX || held) {
        if (threadIdx.x == 0 && !held) record(p, err.key);
        return;
    }
    // copy on write: a request leaves the shared page unless every other
    // holder has left it before (earlier requests of this call)
    const int per = (n + blockDim.x - 1) / blockDim.x;
    const int i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
    int mine = 0, leave = 0;
    for (int i = i0; i < i1; i++) {
        const int len = length[i];
        int need = (len + rows[i] + P - 1) / P - (len + P - 1) / P;
        const int pg = last[i];
        if (pg >= 0) {
            int left = p.refs[pg];
            for (int j = 0; j < i && left > 1; j++) left -= last[j] == pg;
            if (left > 1) {
                need = (need + 1) | INT_MIN;                  // top bit: the first new page is the copy
                leave++;
            }
        }
        first[i] = need;
        mine += need & INT_MAX;
    }
    long long sums;
    const long long before = block_scan((long long)leave << 32 | mine, scan2, 0, sums);
    const int total = (int)sums, n_leave = (int)(sums >> 32);
    int at = (int)before, k = (int)(before >> 32), turn = 0;
    for (int i = i0; i < i1; i++) {
        const int need = first[i];
        if (need >= 0) last[i] = -1;                          // keeps its page
        else {
            jobs[k] = {last[i], 0, length[i] % P, 0};
            last[i] = k++;                                    // from here on: its job
        }
        first[i] = at;
        at += need & INT_MAX;
    }
    __syncthreads();
    // Two passes over the counts, as nothing may change before it is known
    // that there are pages enough; more than one step only when the pool's
    // first pages are taken.
    const int found = free_pages(p, total, free0, scan, turn, [](int, int) {});
    if (found < total) {
        if (threadIdx.x == 0) {                               // the request that the pages run out at
            int i = 0;
            while (i < n - 1 && first[i + 1] <= found) i++;
            record(p, i * 16 + VB_PAGES_FULL);
        }
        return;
    }
    free_pages(p, total, free0, scan, turn, [&](int rank, int page) {
        int lo = 0, hi = n - 1;                               // the request whose page of this rank it is
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first[mid] <= rank) lo = mid;
            else hi = mid - 1;
        }
        const int begin = (length[lo] + P - 1) / P - (last[lo] >= 0);
        p.table[(int64_t)seqs[lo] * p.max_pages + begin + rank - first[lo]] = page;
        p.refs[page] = 1;
        if (last[lo] >= 0 && rank == first[lo]) jobs[last[lo]].dst = page;
    });
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        if (last[i] >= 0) atomicSub(&p.refs[jobs[last[i]].src], 1);
        p.length[seqs[i]] = length[i] + rows[i];
    }
    if (threadIdx.x == 0) ws[0] = n_leave;
}

// Copies the first rows of pages; a warp takes one (job, layer, k or v, head).
__global__ void __launch_bounds__(PG_COPY) pages_copy_rows(vb_pages p, const int *ws) {
    constexpr int B = 8;
    pdl_trigger();
    pdl_wait();
    const PageJob *jobs = reinterpret_cast<const PageJob *>(ws + 4);
    const int row16 = p.head_dim / 8, head16 = p.page_rows * row16, lane = threadIdx.x & 31;       // 16-byte units
    const int64_t tasks = (int64_t)ws[0] * p.n_layers * 2 * p.n_kv_heads;
    for (int64_t t = (int64_t)blockIdx.x * (PG_COPY / 32) + (threadIdx.x >> 5); t < tasks; t += gridDim.x * (PG_COPY / 32)) {
        const int h = (int)(t % p.n_kv_heads), lay = (int)(t / p.n_kv_heads % (2 * p.n_layers));
        const PageJob j = jobs[t / p.n_kv_heads / (2 * p.n_layers)];
        uint4 *pool = static_cast<uint4 *>((lay & 1) ? p.v : p.k) + ((int64_t)(lay >> 1) * p.n_pages * p.n_kv_heads + h) * head16;
        const uint4 *src = pool + (int64_t)j.src * p.n_kv_heads * head16;
        uint4 *dst = pool + (int64_t)j.dst * p.n_kv_heads * head16;
        const int n16 = j.rows * row16;
        for (int c = lane; c < n16; c += 32 * B) {
            uint4 x[B];
#pragma unroll
            for (int i = 0; i < B; i++)
                if (c + 32 * i < n16) x[i] = src[c + 32 * i];
#pragma unroll
            for (int i = 0; i < B; i++)
                if (c + 32 * i < n16) dst[c + 32 * i] = x[i];
        }
    }
}

// grid (request, column block): every thread owns table columns of one dst.
__global__ void __launch_bounds__(256) pages_fork_kernel(vb_pages p, int n, const int32_t *src, const int32_t *dst) {
    extern __shared__ int sm[];
    __shared__ PageError err;
    pdl_trigger();
    pdl_wait();
    uint32_t *bits = reinterpret_cast<uint32_t *>(sm);
    if (threadIdx.x == 0) err.key = INT_MAX;
    if (any_error(p)) return;
    check_seqs(p, n, dst, bits, &err);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = src[i];
        if (s < 0 || s >= p.n_seqs || (bits[s >> 5] >> (s & 31) & 1u)) err.at(i, VB_PAGES_SEQ);
    }
    __syncthreads();
    if (err.key != INT_MAX) {
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) record(p, err.key);
        return;
    }
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < p.max_pages; c += gridDim.y * blockDim.x) {
        const int now = p.table[(int64_t)s * p.max_pages + c], old = p.table[(int64_t)d * p.max_pages + c];
        if (old >= 0 && old < p.n_pages) atomicSub(&p.refs[old], 1);
        if (now >= 0 && now < p.n_pages) atomicAdd(&p.refs[now], 1);
        if (now >= 0 || old >= 0) p.table[(int64_t)d * p.max_pages + c] = now;
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) p.length[d] = p.length[s];
}

// grid (request, column block).  cut: the new lengths.
__global__ void __launch_bounds__(256) pages_truncate_kernel(vb_pages p, int n, const int32_t *seqs,
                                                             const int32_t *cut) {
    extern __shared__ int sm[];
    __shared__ PageError err;
    pdl_trigger();
    pdl_wait();
    uint32_t *bits = reinterpret_cast<uint32_t *>(sm);
    if (threadIdx.x == 0) err.key = INT_MAX;
    if (any_error(p)) return;
    check_seqs(p, n, seqs, bits, &err);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x)
        if (cut[i] < 0) err.at(i, VB_PAGES_COUNT);
    __syncthreads();
    if (err.key != INT_MAX) {
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) record(p, err.key);
        return;
    }
    const int s = seqs[blockIdx.x], len = cut[blockIdx.x];
    const int keep = len / p.page_rows + (len % p.page_rows != 0);
    for (int c = keep + blockIdx.y * blockDim.x + threadIdx.x; c < p.max_pages; c += gridDim.y * blockDim.x) {
        const int old = p.table[(int64_t)s * p.max_pages + c];
        if (old < 0) continue;
        if (old < p.n_pages) atomicSub(&p.refs[old], 1);
        p.table[(int64_t)s * p.max_pages + c] = -1;
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) p.length[s] = min(p.length[s], len);
}

// ws: [0] requests (0 after an error), [4 ..] moves: [i*ld + j] the pool rows
// (page * page_rows + slot) that row j of request i's path comes from and goes
// to; -1: stays.
__global__ void __launch_bounds__(PG_KEEP) pages_keep_plan(vb_pages p, int n, const int32_t *seqs, const int32_t *drafted,
                                                           const int32_t *kept, const int32_t *path, int ld, int *ws) {
    extern __shared__ int sm[];
    __shared__ PageError err;
    uint32_t *bits = reinterpret_cast<uint32_t *>(sm);
    int2 *moves = reinterpret_cast<int2 *>(ws + 4);
    const int P = p.page_rows, most = p.max_pages * P;
    if (threadIdx.x == 0) err.key = INT_MAX;
    for (int i = threadIdx.x; i < (p.n_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
    pdl_trigger();
    pdl_wait();
    const bool held = p.status[0] != 0;
    __syncthreads();
    bool twice = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i], d = drafted[i], k = kept[i];
        if (s < 0 || s >= p.n_seqs) {
            err.at(i, VB_PAGES_SEQ);
            continue;
        }
        twice |= atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u;
        const int len = p.length[s];
        if (len < 0 || len > most) err.at(i, VB_PAGES_LONG);
        else if (d < 0 || k < 0 || k > d || k > ld || d > len) err.at(i, VB_PAGES_COUNT);
    }
    // the paths, of requests that are in order themselves; by the other warps
    // first, while those above wait for their lengths
    const int busy = min((n + 31) & ~31, PG_KEEP / 2);
    for (int e = (threadIdx.x + PG_KEEP - busy) % PG_KEEP; e < n * ld; e += PG_KEEP) {
        const int i = e / ld, j = e - i * ld, s = seqs[i], d = drafted[i], at = path[e], prev = j ? path[e - 1] : -1;
        moves[e] = make_int2(-1, -1);
        if (j >= kept[i] || s < 0 || s >= p.n_seqs) continue;
        const int len = p.length[s], base = len - d;
        if (d < 0 || kept[i] > d || len < 0 || len > most || base < 0) continue;
        const int32_t *row = p.table + (int64_t)s * p.max_pages;
        if (at < 0 || at >= d || prev >= at) err.at(i, VB_PAGES_PATH);
        else if (at != j) {
            const int ps = row[(base + at) / P], pd = row[(base + j) / P];
            if (ps < 0 || ps >= p.n_pages || pd < 0 || pd >= p.n_pages) err.at(i, VB_PAGES_TABLE);
            else if (p.refs[pd] != 1) err.at(i, VB_PAGES_SHARED);
            else moves[e] = make_int2(ps * P + (base + at) % P, pd * P + (base + j) % P);
        }
    }
    if (__syncthreads_or(twice)) {
        which_twice(n, seqs, &err);
        __syncthreads();
    }
    if (threadIdx.x == 0) ws[0] = err.key == INT_MAX && !held ? n : 0;
    if (err.key != INT_MAX || held) {
        if (threadIdx.x == 0 && !held) record(p, err.key);
        return;
    }
    // pages past the new end
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5) {
        const int s = seqs[i], len = p.length[s], now = len - drafted[i] + kept[i];
        for (int c = (now + P - 1) / P + lane; c < (len + P - 1) / P; c += 32) {
            const int old = p.table[(int64_t)s * p.max_pages + c];
            if (old >= 0 && old < p.n_pages) atomicSub(&p.refs[old], 1);
            p.table[(int64_t)s * p.max_pages + c] = -1;
        }
        __syncwarp();
        if (lane == 0) p.length[s] = now;
    }
}

// A thread owns 16 bytes of every row of one (request, layer, k or v, head)
// and walks the path in order.  A row goes to a place at or before its own and
// later sources lie behind it, so a batch that is loaded before it is stored
// never reads what it wrote.
__global__ void __launch_bounds__(PG_COPY) pages_move_rows(vb_pages p, int ld, const int *ws) {
    constexpr int B = 8;
    pdl_trigger();
    pdl_wait();
    const int row16 = p.head_dim / 8, P = p.page_rows;
    const int cols = p.n_layers * 2 * p.n_kv_heads * row16, blocks = (cols + PG_COPY - 1) / PG_COPY, n = ws[0];
    for (int t = blockIdx.x; t < blocks * n; t += gridDim.x) {
        const int i = t / blocks, col = (t - i * blocks) * PG_COPY + threadIdx.x;
        if (col >= cols) continue;
        const int2 *mv = reinterpret_cast<const int2 *>(ws + 4) + (int64_t)i * ld;
        const int c = col % row16, h = col / row16 % p.n_kv_heads, lay = col / row16 / p.n_kv_heads;
        uint4 *pool = static_cast<uint4 *>((lay & 1) ? p.v : p.k) +
                      ((int64_t)(lay >> 1) * p.n_pages * p.n_kv_heads + h) * P * row16 + c;
        auto at = [&](int r) { return ((int64_t)(r / P) * p.n_kv_heads * P + r % P) * row16; };
        for (int j0 = 0; j0 < ld; j0 += B) {
            uint4 x[B];
            int2 m[B];
#pragma unroll
            for (int j = 0; j < B; j++) m[j] = j0 + j < ld ? mv[j0 + j] : make_int2(-1, -1);
#pragma unroll
            for (int j = 0; j < B; j++)
                if (m[j].x >= 0) x[j] = pool[at(m[j].x)];
#pragma unroll
            for (int j = 0; j < B; j++)
                if (m[j].x >= 0) pool[at(m[j].y)] = x[j];
        }
    }
}

// ws: [0] live pages (0 after an error), [4 ..] the new number of each page,
// then the old number of each new one.
__global__ void __launch_bounds__(PG_PLAN) pages_compact_plan(vb_pages p, vb_pages to, int *ws) {
    __shared__ int scan[2][32];
    __shared__ PageError err;
    pdl_trigger();
    pdl_wait();
    int turn = 0;
    int *number = ws + 4, *live = ws + 4 + p.n_pages;
    if (threadIdx.x == 0) {
        err.key = INT_MAX;
        ws[0] = 0;
        ws[1] = 0;
    }
    if (p.status[0]) return;
    __syncthreads();
    for (int64_t e = threadIdx.x; e < (int64_t)p.n_seqs; e += blockDim.x)
        if (p.length[e] < 0 || (int64_t)p.length[e] > (int64_t)p.max_pages * p.page_rows)
            err.at((int)e, VB_PAGES_LONG);
    int total = 0;
    for (int base = 0; base < p.n_pages; base += blockDim.x * PG_SCAN) {
        const int q0 = base + threadIdx.x * PG_SCAN;
        uint32_t used = 0;
#pragma unroll
        for (int j = 0; j < PG_SCAN; j++)
            if (q0 + j < p.n_pages && p.refs[q0 + j] > 0) used |= 1u << j;
        int here;
        int k = total + block_scan(__popc(used), scan, turn++, here);
#pragma unroll
        for (int j = 0; j < PG_SCAN; j++)
            if (q0 + j < p.n_pages) {
                const bool u = used >> j & 1u;
                number[q0 + j] = u ? k : -1;
                if (u) live[k++] = q0 + j;
            }
        total += here;
    }
    __syncthreads();
    if (threadIdx.x == 0 && total > to.n_pages) err.at(0, VB_PAGES_FULL);
    __syncthreads();
    if (err.key != INT_MAX) {
        if (threadIdx.x == 0) record(p, err.key);
        return;
    }
    for (int i = threadIdx.x; i < to.n_pages; i += blockDim.x) to.refs[i] = i < total ? p.refs[live[i]] : 0;
    for (int i = threadIdx.x; i < p.n_seqs; i += blockDim.x) to.length[i] = p.length[i];
    if (threadIdx.x < 4) to.status[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        ws[0] = total;
        ws[1] = 1;
    }
}

// Page contents (a unit: the K or V of one page of one layer, contiguous)
// and the table, over all CTAs.  Bound by HBM: 1000 pages of 64 rows in 28
// layers of 2 heads (3.76 GB read and written) take 569 to 574 us, the copy rate.
__global__ void __launch_bounds__(PG_COPY) pages_compact_copy(vb_pages p, vb_pages to, const int *ws) {
    constexpr int B = 4;
    pdl_trigger();
    pdl_wait();
    if (!ws[1]) return;
    const int total = ws[0];
    const int *number = ws + 4, *live = ws + 4 + p.n_pages;
    const int64_t page16 = (int64_t)p.n_kv_heads * p.page_rows * (p.head_dim / 8);
    const int64_t units = (int64_t)total * p.n_layers * 2;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int j = (int)(u % total), lay = (int)(u / total);
        const uint4 *src = static_cast<const uint4 *>((lay & 1) ? p.v : p.k) +
                           ((int64_t)(lay >> 1) * p.n_pages + live[j]) * page16;
        uint4 *dst = static_cast<uint4 *>((lay & 1) ? to.v : to.k) + ((int64_t)(lay >> 1) * to.n_pages + j) * page16;
        for (int64_t i = threadIdx.x; i < page16; i += B * PG_COPY) {
            uint4 x[B];
#pragma unroll
            for (int b = 0; b < B; b++)
                if (i + b * PG_COPY < page16) x[b] = src[i + b * PG_COPY];
#pragma unroll
            for (int b = 0; b < B; b++)
                if (i + b * PG_COPY < page16) dst[i + b * PG_COPY] = x[b];
        }
    }
    const int64_t entries = (int64_t)to.n_seqs * to.max_pages;
    for (int64_t e = (int64_t)blockIdx.x * PG_COPY + threadIdx.x; e < entries; e += (int64_t)gridDim.x * PG_COPY) {
        const int64_t s = e / to.max_pages, c = e % to.max_pages;
        const int old = c < p.max_pages ? p.table[s * p.max_pages + c] : -1;
        to.table[e] = old >= 0 && old < p.n_pages ? number[old] : -1;
    }
}

// -------------------------------------------------------------------- host
int check_pages(vb_ctx *ctx, const vb_pages *p, const char *who) {
    if (!p || !p->k || !p->v || !p->table || !p->length || !p->refs || !p->status)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: null cache or cache pointer", who);
    if (p->type != VB_TYPE_BF16 && p->type != VB_TYPE_F16)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: cache rows are BF16 or F16", who);
    if (p->n_layers <= 0 || p->n_pages <= 0 || p->n_kv_heads <= 0 || p->n_seqs <= 0 || p->max_pages <= 0 ||
        p->n_seqs > PG_MAX_SEQS)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: cache sizes out of range", who);
    if (p->page_rows < 16 || p->page_rows > 1024 || (p->page_rows & (p->page_rows - 1)))
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: page_rows must be a power of two, 16 to 1024", who);
    if (p->head_dim < 8 || p->head_dim > 256 || p->head_dim % 8)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: head_dim must be a multiple of 8, at most 256", who);
    // row numbers of one layer, and rows of one sequence, are 32-bit; a length
    // is rounded up to pages of up to 1024 rows and to tiles of 128
    if ((int64_t)p->n_pages * p->n_kv_heads * p->page_rows > INT_MAX || (int64_t)p->max_pages * p->page_rows > INT_MAX - 1024)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: cache too large", who);
    if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->table | (uintptr_t)p->length | (uintptr_t)p->refs |
         (uintptr_t)p->status) & 15)
        return set_error(ctx, VB_ERR_INVALID_ARG, "%s: cache pointers must be 16-byte aligned", who);
    return VB_OK;
}

static int check_call(vb_ctx *ctx, const vb_pages *p, int n, const char *who, bool pointers) {
    int rc = check_pages(ctx, p, who);
    if (rc) return rc;
    if (n < 0 || n > p->n_seqs) return set_error(ctx, VB_ERR_INVALID_ARG, "%s: 0 to n_seqs requests", who);
    if (n > 0 && !pointers) return set_error(ctx, VB_ERR_INVALID_ARG, "%s: null pointer", who);
    return VB_OK;
}

// CTAs for a call that may copy so many bytes: one for each 16 KB, four per SM at most.
static unsigned share_out(const vb_ctx *ctx, int64_t bytes) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(4 * ctx->sm_count, bytes >> 14));
}

static size_t seq_bits(const vb_pages *p) { return (size_t)((p->n_seqs + 31) / 32) * 4; }

int init_pages(vb_ctx *ctx) {
    VB_CHECK(ctx, cudaFuncSetAttribute(pages_extend_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       3 * PG_MAX_SEQS * 4 + PG_MAX_SEQS / 8));
    return VB_OK;
}

}  // namespace vb

using namespace vb;

extern "C" int vb_pages_init(vb_ctx *ctx, const vb_pages *p) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_pages(ctx, p, "vb_pages_init");
    if (rc) return rc;
    VB_CHECK(ctx, cudaMemsetAsync(p->table, 0xff, (size_t)p->n_seqs * p->max_pages * 4, ctx->stream));
    VB_CHECK(ctx, cudaMemsetAsync(p->length, 0, (size_t)p->n_seqs * 4, ctx->stream));
    VB_CHECK(ctx, cudaMemsetAsync(p->refs, 0, (size_t)p->n_pages * 4, ctx->stream));
    VB_CHECK(ctx, cudaMemsetAsync(p->status, 0, 16, ctx->stream));
    return VB_OK;
}

extern "C" int vb_pages_extend(vb_ctx *ctx, const vb_pages *p, int n, const int32_t *seqs, const int32_t *rows) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_call(ctx, p, n, "vb_pages_extend", seqs && rows);
    if (rc || n == 0) return rc;
    rc = arena_reserve(ctx, ctx->pages_ws, 16 + (size_t)n * sizeof(PageJob));
    if (rc) return rc;
    int *ws = static_cast<int *>(ctx->pages_ws.ptr);
    VB_CHECK(ctx, pdl_launch(ctx, pages_extend_plan, dim3(1), dim3(PG_STEP), (size_t)3 * n * 4 + seq_bits(p), *p, n, seqs, rows,
                             ws));
    VB_LAUNCH_CHECK(ctx, "pages_extend_plan");
    // (as if every request left its page)
    const int64_t bytes = (int64_t)n * 2 * p->n_layers * p->n_kv_heads * p->page_rows * p->head_dim * 2;
    VB_CHECK(ctx, pdl_launch(ctx, pages_copy_rows, dim3(share_out(ctx, bytes)), dim3(PG_COPY), 0, *p,
                             static_cast<const int *>(ws)));
    VB_LAUNCH_CHECK(ctx, "pages_copy_rows");
    return VB_OK;
}

static dim3 column_grid(const vb_pages *p, int n) {
    return dim3(n, std::min(16, (p->max_pages + 255) / 256));
}

extern "C" int vb_pages_fork(vb_ctx *ctx, const vb_pages *p, int n, const int32_t *src, const int32_t *dst) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_call(ctx, p, n, "vb_pages_fork", src && dst);
    if (rc || n == 0) return rc;
    VB_CHECK(ctx, pdl_launch(ctx, pages_fork_kernel, column_grid(p, n), dim3(256), seq_bits(p), *p, n, src, dst));
    VB_LAUNCH_CHECK(ctx, "pages_fork");
    return VB_OK;
}

extern "C" int vb_pages_truncate(vb_ctx *ctx, const vb_pages *p, int n, const int32_t *seqs, const int32_t *length) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_call(ctx, p, n, "vb_pages_truncate", seqs && length);
    if (rc || n == 0) return rc;
    VB_CHECK(ctx, pdl_launch(ctx, pages_truncate_kernel, column_grid(p, n), dim3(256), seq_bits(p), *p, n, seqs,
                             length));
    VB_LAUNCH_CHECK(ctx, "pages_truncate");
    return VB_OK;
}

extern "C" int vb_pages_keep(vb_ctx *ctx, const vb_pages *p, int n, const int32_t *seqs, const int32_t *drafted,
                             const int32_t *kept, const int32_t *path, int ld_path) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_call(ctx, p, n, "vb_pages_keep", seqs && drafted && kept && (path || !ld_path));
    if (rc) return rc;
    const int64_t cols = (int64_t)p->n_layers * 2 * p->n_kv_heads * (p->head_dim / 8);
    if (ld_path < 0 || (int64_t)n * ld_path > INT_MAX || cols > INT_MAX || (cols / PG_COPY + 1) * n > INT_MAX)
        return set_error(ctx, VB_ERR_INVALID_ARG, "vb_pages_keep: path length or cache out of range");
    if (n == 0) return VB_OK;
    rc = arena_reserve(ctx, ctx->pages_ws, 16 + (size_t)n * ld_path * sizeof(int2));
    if (rc) return rc;
    int *ws = static_cast<int *>(ctx->pages_ws.ptr);
    VB_CHECK(ctx, pdl_launch(ctx, pages_keep_plan, dim3(1), dim3(PG_KEEP), seq_bits(p), *p, n, seqs, drafted, kept, path,
                             ld_path, ws));
    VB_LAUNCH_CHECK(ctx, "pages_keep_plan");
    const int64_t bytes = (int64_t)n * 2 * p->n_layers * p->n_kv_heads * ld_path * p->head_dim * 2;
    VB_CHECK(ctx, pdl_launch(ctx, pages_move_rows, dim3(share_out(ctx, bytes)), dim3(PG_COPY), 0, *p, ld_path,
                             static_cast<const int *>(ws)));
    VB_LAUNCH_CHECK(ctx, "pages_move_rows");
    return VB_OK;
}

extern "C" int vb_pages_compact(vb_ctx *ctx, const vb_pages *p, const vb_pages *to) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_pages(ctx, p, "vb_pages_compact");
    if (rc) return rc;
    rc = check_pages(ctx, to, "vb_pages_compact");
    if (rc) return rc;
    if (p->type != to->type || p->n_layers != to->n_layers || p->n_kv_heads != to->n_kv_heads ||
        p->page_rows != to->page_rows || p->head_dim != to->head_dim || p->n_seqs != to->n_seqs ||
        to->max_pages < p->max_pages)
        return set_error(ctx, VB_ERR_INVALID_ARG, "vb_pages_compact: the caches hold different rows");
    if (p->k == to->k || p->v == to->v || p->table == to->table || p->length == to->length || p->refs == to->refs ||
        p->status == to->status)
        return set_error(ctx, VB_ERR_INVALID_ARG, "vb_pages_compact: the caches share memory");
    rc = arena_reserve(ctx, ctx->pages_ws, 16 + (size_t)p->n_pages * 8);
    if (rc) return rc;
    int *ws = static_cast<int *>(ctx->pages_ws.ptr);
    VB_CHECK(ctx, pdl_launch(ctx, pages_compact_plan, dim3(1), dim3(PG_PLAN), 0, *p, *to, ws));
    VB_LAUNCH_CHECK(ctx, "pages_compact_plan");
    // one CTA for every four units that there can be, 128 per SM at most: CTAs
    // that come and go keep the copy even where resident ones fall out of step
    // (3.8 GB with 8 | 32 | 128 per SM: 625 | 587 | 569 us; 70 MB of small pages
    // with 16 | 128: 18 | 32, the empty ones cost)
    const int64_t units = (int64_t)std::min(p->n_pages, to->n_pages) * p->n_layers * 2;
    const unsigned ctas = (unsigned)std::max<int64_t>(ctx->sm_count, std::min<int64_t>(units / 4, 128 * ctx->sm_count));
    VB_CHECK(ctx, pdl_launch(ctx, pages_compact_copy, dim3(ctas), dim3(PG_COPY), 0, *p, *to,
                             static_cast<const int *>(ws)));
    VB_LAUNCH_CHECK(ctx, "pages_compact_copy");
    return VB_OK;
}

extern "C" int vb_pages_status(vb_ctx *ctx, const vb_pages *p, int *error, int *request, int *free_pages) {
    if (!ctx) return VB_ERR_INVALID_ARG;
    int rc = check_pages(ctx, p, "vb_pages_status");
    if (rc) return rc;
    int32_t st[4] = {0, 0, 0, 0};
    VB_CHECK(ctx, cudaMemcpyAsync(st, p->status, sizeof(st), cudaMemcpyDeviceToHost, ctx->stream));
    VB_CHECK(ctx, cudaStreamSynchronize(ctx->stream));
    if (free_pages) {
        try {
            std::vector<int32_t> refs((size_t)p->n_pages);
            VB_CHECK(ctx, cudaMemcpyAsync(refs.data(), p->refs, refs.size() * 4, cudaMemcpyDeviceToHost, ctx->stream));
            VB_CHECK(ctx, cudaStreamSynchronize(ctx->stream));
            int n = 0;
            for (int32_t r : refs) n += r == 0;
            *free_pages = n;
        } catch (...) {
            return set_error(ctx, VB_ERR_OOM, "vb_pages_status: out of host memory");
        }
    }
    if (error) *error = st[0];
    if (request) *request = st[0] ? st[1] : 0;
    if (!st[0]) return VB_OK;
    VB_CHECK(ctx, cudaMemsetAsync(p->status, 0, sizeof(st), ctx->stream));
    return set_error(ctx, VB_ERR_BACKEND, "paged cache: error %d at request %d", st[0], st[1]);
}
