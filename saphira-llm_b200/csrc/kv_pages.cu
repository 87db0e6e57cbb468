// kv_pages.cu -- the paged KV cache: forking, reserving (with copy on write),
// releasing and compacting pages, and the store of new tokens.
//
// The cache is the caller's memory: pools of pages, one reference count per
// page (0 = free), one table row and one length per slot (sequence). Every
// operator first checks all that it will use (slots, lengths, page ids,
// counts) and changes nothing when something is wrong, so the bookkeeping
// runs in one CTA or one cluster: a phase ends at a barrier, not at a launch.
// What it decides to copy goes into a list in the caller's workspace, and a
// second launch over the whole device (overlapped with the first by
// programmatic dependent launch) moves the bytes.
//
// A page is given out lowest id first, in the order of the call's slots, so
// the tables a call leaves are the same every time; the reference counts are
// integer atomics, whose order does not matter.

#include <cooperative_groups.h>

#include "../../include/sllm_cuda_testing.h"
#include "serve.cuh"

namespace cg = cooperative_groups;

namespace sllm {
namespace {

constexpr int kClCtas = 8;          // CTAs of a bookkeeping cluster
constexpr int kClThreads = 512;
constexpr int kResThreads = 1024;   // the reserving CTA
constexpr int kHead = 16;           // ints before the workspace's arrays; [0] is the number of copies

struct Work {                       // the caller's workspace, as ints
    int* count;
    int* mark;                      // [n_slots] how often a slot is named
    int* slot_page;                 // [n_slots] the last page a slot will write to, or -1
    int* slot_need;                 // [n_slots] first page of its share of the free list; bit 31: copies
    int* list;                      // [n_pages] free pages, or compact's map from old to new ids
    int4* pairs;                    // [max(n_slots, n_pages)] copies: source, destination, rows
    int* rows;                      // [n_slots][width] tables being forked
};

__host__ __device__ inline size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

__host__ __device__ inline size_t work_ints(int n_pages, int n_slots, int width) {
    const size_t pairs = (size_t)(n_pages > n_slots ? n_pages : n_slots);
    return kHead + 3 * align16(n_slots) + align16(n_pages) + 4 * pairs + align16((size_t)n_slots * width);
}

__host__ __device__ inline Work work_of(void* base, int n_pages, int n_slots, int width) {
    const size_t pairs = (size_t)(n_pages > n_slots ? n_pages : n_slots);
    Work w;
    int* p = static_cast<int*>(base);
    w.count = p;
    p += kHead;
    w.mark = p;
    p += align16(n_slots);
    w.slot_page = p;
    p += align16(n_slots);
    w.slot_need = p;
    p += align16(n_slots);
    w.list = p;
    p += align16(n_pages);
    w.pairs = reinterpret_cast<int4*>(p);
    p += 4 * pairs;
    w.rows = p;
    return w;
}

__device__ __forceinline__ int used_of(int len, int page) { return (len + page - 1) / page; }

// the used entries of a slot's table name live pages (threads t, t + nt, ...)
__device__ __forceinline__ bool row_ok(const PagesDev& p, int slot, int t, int nt) {
    const int len = p.lens[slot];
    if (len < 0 || len > p.cap) return false;
    const int used = used_of(len, p.page);
    bool ok = true;
    for (int j = t; j < used; j += nt) {
        const int id = p.tables[(size_t)slot * p.width + j];
        ok = ok && id >= 0 && id < p.n_pages && p.refs[id] > 0;
    }
    return ok;
}

// The threads of a bookkeeping cluster that share a slot: a whole CTA's, or so
// many fewer, down to a warp's, that one round takes all slots. 1024 slots of
// 32 pages with a CTA each, one after the other: fork 176 us, release 231 us;
// with a warp each 18 and 17 us. Fork of 32 slots of 256 pages: a
// warp each 22.9 us, a CTA each 14.7 us, 128 threads each 10.8 us.
struct Team {
    int t, size, first, step;       // this thread, threads; the first slot and the way to the next
    __device__ __forceinline__ Team(int n, int rank) {
        size = kClThreads;
        while (size > 32 && kClCtas * (kClThreads / size) < n) size /= 2;
        t = threadIdx.x % size;
        first = rank * (kClThreads / size) + threadIdx.x / size;
        step = kClCtas * (kClThreads / size);
    }
    __device__ __forceinline__ void sync() const {
        if (size == 32) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / size), "r"(size) : "memory");
    }
};

// exclusive sum over the block; *total gets the sum. NT threads, all of them.
template <int NT>
__device__ __forceinline__ int block_scan(int v, int* total) {
    __shared__ int part[NT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
    #pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        const int y = part[w];
        before += w < warp ? y : 0;
        all += y;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// ---------------------------------------------------------------------------
// fork: dst[i] becomes what src[i] holds, for all i at once. The tables of
// the sources are staged first, so a slot may be a source and a destination
// (a beam search's reordering); every page a destination held loses one
// reference, every page of a source gains one. No page is copied here: a
// shared last page is copied when a slot next reserves tokens in it.
// ---------------------------------------------------------------------------
__global__ void __cluster_dims__(kClCtas, 1, 1) __launch_bounds__(kClThreads)
kv_fork_kernel(const PagesDev p, const int32_t* src, const int32_t* dst, int n, void* work, int32_t* status) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ int bad;
    const Work w = work_of(work, p.n_pages, p.n_slots, p.width);
    const int rank = (int)cl.block_rank(), t = threadIdx.x;
    const Team team(n, rank);
    if (t == 0) bad = 0;
    for (int i = rank * kClThreads + t; i < p.n_slots; i += kClCtas * kClThreads) w.mark[i] = 0;
    cl.sync();
    int* const bad0 = cl.map_shared_rank(&bad, 0);
    for (int i = team.first; i < n; i += team.step) {
        const int s = src[i], d = dst[i];
        bool ok = s >= 0 && s < p.n_slots && d >= 0 && d < p.n_slots;
        if (ok) ok = row_ok(p, s, team.t, team.size) && row_ok(p, d, team.t, team.size);
        if (team.t == 0 && d >= 0 && d < p.n_slots && atomicAdd(&w.mark[d], 1) > 0) ok = false;
        if (!ok) atomicExch(bad0, 1);
    }
    cl.sync();
    const int any = *bad0;
    cl.sync();                      // nobody leaves before all have read CTA 0's word
    if (any != 0) {
        if (rank == 0 && t == 0) raise(status, SLLM_CUDA_ERR_ARG);
        return;
    }
    for (int i = team.first; i < n; i += team.step) {
        const int s = src[i], len = p.lens[s], used = used_of(len, p.page);
        for (int j = team.t; j < used; j += team.size) {
            const int id = p.tables[(size_t)s * p.width + j];
            w.rows[(size_t)i * p.width + j] = id;
            atomicAdd(&p.refs[id], 1);
        }
        if (team.t == 0) w.slot_page[i] = len;
    }
    cl.sync();
    for (int i = team.first; i < n; i += team.step) {
        const int d = dst[i], len = w.slot_page[i], used = used_of(len, p.page);
        const int was = used_of(p.lens[d], p.page);
        for (int j = team.t; j < max(used, was); j += team.size) {
            int32_t* e = p.tables + (size_t)d * p.width + j;
            if (j < was) atomicSub(&p.refs[*e], 1);
            if (j < used) *e = w.rows[(size_t)i * p.width + j];
        }
        team.sync();                // every thread has read the old length
        if (team.t == 0) p.lens[d] = len;
    }
}

// ---------------------------------------------------------------------------
// release: slots[i] keeps its first new_len[i] tokens (none without new_len)
// ---------------------------------------------------------------------------
__global__ void __cluster_dims__(kClCtas, 1, 1) __launch_bounds__(kClThreads)
kv_release_kernel(const PagesDev p, const int32_t* slots, const int32_t* new_len, int n, void* work,
                  int32_t* status) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ int bad;
    const Work w = work_of(work, p.n_pages, p.n_slots, p.width);
    const int rank = (int)cl.block_rank(), t = threadIdx.x;
    const Team team(n, rank);
    if (t == 0) bad = 0;
    for (int i = rank * kClThreads + t; i < p.n_slots; i += kClCtas * kClThreads) w.mark[i] = 0;
    cl.sync();
    int* const bad0 = cl.map_shared_rank(&bad, 0);
    for (int i = team.first; i < n; i += team.step) {
        const int s = slots[i];
        bool ok = s >= 0 && s < p.n_slots;
        if (ok) {
            ok = row_ok(p, s, team.t, team.size);
            const int nl = new_len != nullptr ? new_len[i] : 0;
            if (nl < 0 || nl > p.lens[s]) ok = false;
            if (team.t == 0 && atomicAdd(&w.mark[s], 1) > 0) ok = false;
        }
        if (!ok) atomicExch(bad0, 1);
    }
    cl.sync();
    const int any = *bad0;
    cl.sync();
    if (any != 0) {
        if (rank == 0 && t == 0) raise(status, SLLM_CUDA_ERR_ARG);
        return;
    }
    for (int i = team.first; i < n; i += team.step) {
        const int s = slots[i], nl = new_len != nullptr ? new_len[i] : 0;
        const int keep = used_of(nl, p.page), was = used_of(p.lens[s], p.page);
        for (int j = keep + team.t; j < was; j += team.size) atomicSub(&p.refs[p.tables[(size_t)s * p.width + j]], 1);
        team.sync();
        if (team.t == 0) p.lens[s] = nl;
    }
}

// ---------------------------------------------------------------------------
// reserve: pages for n_new[i] more tokens of slots[i], and its length moved
// on. A last page that is partly filled, will be written and has other
// owners is replaced by a copy: slot by slot in the call's order, so of r
// owners named in one call that are all its owners the last keeps the page.
// One CTA: the call's slots are few as a rule, and the free pages are found by
// one pass over the counts, 16 per thread in flight. A page's writers are counted
// in the page's own words of the workspace.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kResThreads)
kv_reserve_kernel(const PagesDev p, const int32_t* slots, const int32_t* n_new, int n, void* work, int32_t* status) {
    __shared__ int err, n_pairs;
    pdl_trigger();
    const Work w = work_of(work, p.n_pages, p.n_slots, p.width);
    const int t = threadIdx.x;
    if (t == 0) {
        err = 0;
        n_pairs = 0;
        *w.count = 0;
    }
    for (int i = t; i < n; i += kResThreads) {
        const int s = slots[i];
        if (s >= 0 && s < p.n_slots) w.mark[s] = 0;
    }
    __syncthreads();
    // what each slot asks for: its new pages, and its last page if it writes there
    int fresh = 0, last = -1, owners = 0;       // of this thread's last slot
    bool shared = false;
    for (int base = 0; base < n; base += kResThreads) {
        const int i = base + t;
        fresh = owners = 0;
        last = -1;
        if (i < n) {
            const int s = slots[i], nn = n_new[i];
            int e = 0;
            if (s < 0 || s >= p.n_slots || nn < 0 || atomicAdd(&w.mark[s], 1) > 0) {
                e = SLLM_CUDA_ERR_ARG;
            } else {
                const int cur = p.lens[s];
                if (cur < 0 || cur > p.cap) {
                    e = SLLM_CUDA_ERR_ARG;
                } else if (nn > p.cap - cur) {
                    e = SLLM_CUDA_ERR_TOO_LARGE;
                } else {
                    fresh = used_of(cur + nn, p.page) - used_of(cur, p.page);
                    if (nn > 0 && cur % p.page != 0) {
                        last = p.tables[(size_t)s * p.width + cur / p.page];
                        if (last < 0 || last >= p.n_pages || (owners = p.refs[last]) <= 0) {
                            e = SLLM_CUDA_ERR_ARG;
                            last = -1;
                        }
                    }
                }
            }
            if (e != 0) atomicCAS(&err, 0, e);
            if (owners > 1 && n > 32) {     // x: how many slots of this call write to the page, y: the last of them
                shared = true;
                w.pairs[last].x = 0;
                w.pairs[last].y = -1;
            }
            w.slot_page[i] = last;
            w.slot_need[i] = fresh;
        }
    }
    const bool one = n <= kResThreads;          // this thread's slot is still at hand
    // (all in one warp: the lanes compare; the words and two more barriers took 0.4 us)
    const unsigned alike = n <= 32 ? __match_any_sync(0xffffffffu, last) : 0u;
    if (__syncthreads_or(shared)) {
        for (int i = t; i < n; i += kResThreads) {
            const int page = one ? last : w.slot_page[i];
            if (page >= 0 && (one ? owners : p.refs[page]) > 1) {
                atomicAdd(&w.pairs[page].x, 1);
                atomicMax(&w.pairs[page].y, i);
            }
        }
        shared = true;
        __syncthreads();
    }
    int total = 0;
    for (int base = 0; base < n; base += kResThreads) {
        const int i = base + t;
        if (!one) {
            last = i < n ? w.slot_page[i] : -1;
            fresh = i < n ? w.slot_need[i] : 0;
            owners = shared && last >= 0 ? p.refs[last] : 0;
        }
        // where all owners write, the last of them keeps the page
        int cow = 0;
        if (owners > 1) {
            const int writers = n <= 32 ? __popc(alike) : w.pairs[last].x;
            const int end = n <= 32 ? 31 - __clz(alike) : w.pairs[last].y;
            cow = writers == owners && end == i ? 0 : 1;
            if (writers > owners) atomicCAS(&err, 0, SLLM_CUDA_ERR_ARG);        // more entries than the count says
        }
        int sum;
        const int at = block_scan<kResThreads>(cow + fresh, &sum);
        if (i < n) w.slot_need[i] = (total + at) | (cow << 31);
        total += sum;
    }
    __syncthreads();
    if (err != 0) {                 // the same for every thread
        if (t == 0) raise(status, err);
        return;
    }
    // the `total` lowest free pages
    constexpr int PER = 16;
    int found = 0;
    for (int base = 0; base < p.n_pages && found < total; base += kResThreads * PER) {
        const int b = base + t * PER;
        int r[PER];
        if (b + PER <= p.n_pages) {
            #pragma unroll
            for (int k = 0; k < PER / 4; ++k) {
                const int4 v = *reinterpret_cast<const int4*>(p.refs + b + 4 * k);
                r[4 * k] = v.x; r[4 * k + 1] = v.y; r[4 * k + 2] = v.z; r[4 * k + 3] = v.w;
            }
        } else {
            #pragma unroll
            for (int k = 0; k < PER; ++k) r[k] = b + k < p.n_pages ? p.refs[b + k] : 1;
        }
        int c = 0;
        #pragma unroll
        for (int k = 0; k < PER; ++k) c += r[k] == 0 ? 1 : 0;
        int sum;
        int at = found + block_scan<kResThreads>(c, &sum);
        #pragma unroll
        for (int k = 0; k < PER; ++k)
            if (r[k] == 0) {
                if (at < total) w.list[at] = b + k;
                ++at;
            }
        found += sum;
    }
    __syncthreads();
    if (found < total) {
        if (t == 0) raise(status, SLLM_CUDA_ERR_NOMEM);
        return;
    }
    // hand them out: a thread per slot, and a warp for a slot that gets many
    const int lane = t & 31;
    for (int base = 0; base < n; base += kResThreads) {
        const int i = base + t;
        int s = 0, from = 0, first = 0, fresh = 0;
        if (i < n) {
            s = slots[i];
            const int nn = n_new[i], cur = p.lens[s], need = w.slot_need[i], cow = need < 0 ? 1 : 0, at = need & 0x7fffffff;
            first = used_of(cur, p.page);
            fresh = used_of(cur + nn, p.page) - first;
            from = at + cow;
            if (cow) {
                const int id = w.list[at], last = w.slot_page[i];
                p.tables[(size_t)s * p.width + cur / p.page] = id;
                p.refs[id] = 1;
                atomicSub(&p.refs[last], 1);
                w.pairs[atomicAdd(&n_pairs, 1)] = make_int4(last, id, cur % p.page, 0);
            }
            p.lens[s] = cur + nn;
        }
        const bool many = fresh > 2;
        for (int x = 0; x < fresh && !many; ++x) {
            const int id = w.list[from + x];
            p.tables[(size_t)s * p.width + first + x] = id;
            p.refs[id] = 1;
        }
        for (unsigned m = __ballot_sync(0xffffffffu, many); m != 0; m &= m - 1) {
            const int l = __ffs(m) - 1, f = __shfl_sync(0xffffffffu, fresh, l), a = __shfl_sync(0xffffffffu, from, l);
            int32_t* const row = p.tables + (size_t)__shfl_sync(0xffffffffu, s, l) * p.width +
                                 __shfl_sync(0xffffffffu, first, l);
            for (int x = lane; x < f; x += 32) {
                const int id = w.list[a + x];
                row[x] = id;
                p.refs[id] = 1;
            }
        }
    }
    __syncthreads();
    if (t == 0) *w.count = n_pairs;
}

// ---------------------------------------------------------------------------
// compact: with L live pages, every live page at or above L moves into a free
// page below L (both in ascending order). Sources and destinations are
// disjoint, so the copies need no order among themselves.
// ---------------------------------------------------------------------------
__global__ void __cluster_dims__(kClCtas, 1, 1) __launch_bounds__(kClThreads)
kv_compact_kernel(const PagesDev p, void* work, int32_t* status) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ int bad, live_cnt, src_cnt;
    pdl_trigger();
    const Work w = work_of(work, p.n_pages, p.n_slots, p.width);
    const int rank = (int)cl.block_rank(), t = threadIdx.x;
    if (t == 0) {
        bad = 0;
        live_cnt = 0;
        src_cnt = 0;
    }
    cl.sync();
    int* const bad0 = cl.map_shared_rank(&bad, 0);
    // the tables first: nothing moves when one is wrong
    {
        const int lane = t & 31;
        bool ok = true;
        for (int s = rank * (kClThreads / 32) + (t >> 5); s < p.n_slots; s += kClCtas * (kClThreads / 32))
            ok = row_ok(p, s, lane, 32) && ok;
        if (!ok) atomicExch(bad0, 1);
    }
    // this CTA's share of the pages: a contiguous run, 512 at a time
    const int per = ((p.n_pages + kClCtas - 1) / kClCtas + kClThreads - 1) / kClThreads * kClThreads;
    const int lo = min(rank * per, p.n_pages), hi = min(lo + per, p.n_pages);
    int c = 0;
    for (int i = lo + t; i < hi; i += kClThreads) c += p.refs[i] > 0 ? 1 : 0;
    if (c > 0) atomicAdd(&live_cnt, c);
    cl.sync();
    const int any = *bad0;
    int live = 0;
    for (int r = 0; r < kClCtas; ++r) live += *cl.map_shared_rank(&live_cnt, r);
    // sources of this share: live pages at or above `live`
    int cs = 0;
    for (int i = max(lo, live) + t; i < hi; i += kClThreads) cs += p.refs[i] > 0 ? 1 : 0;
    if (cs > 0) atomicAdd(&src_cnt, cs);
    cl.sync();
    int src0 = 0, total = 0;        // sources before this share, and all of them
    for (int r = 0; r < kClCtas; ++r) {
        const int x = *cl.map_shared_rank(&src_cnt, r);
        src0 += r < rank ? x : 0;
        total += x;
    }
    // free pages below `live` before this share = pages below it that are not live
    int live_before = 0;
    for (int r = 0; r < rank; ++r) live_before += *cl.map_shared_rank(&live_cnt, r);
    cl.sync();                      // all remote reads are done
    if (any != 0) {
        if (rank == 0 && t == 0) {
            *w.count = 0;
            raise(status, SLLM_CUDA_ERR_ARG);
        }
        return;
    }
    int dst0 = min(lo, live) - (live_before - src0);    // live pages below `live` before this share
    for (int base = lo; base < hi; base += kClThreads) {
        const int i = base + t;
        const int ref = i < hi ? p.refs[i] : 0;
        const int is_src = i < hi && i >= live && ref > 0 ? 1 : 0;
        const int is_dst = i < hi && i < live && ref <= 0 ? 1 : 0;
        int sums;                   // both ranks in one scan: 16 bits each suffice for 512 threads
        const int at = block_scan<kClThreads>(is_src | (is_dst << 16), &sums);
        if (is_src) {
            w.pairs[src0 + (at & 0xffff)].x = i;
            w.pairs[src0 + (at & 0xffff)].w = ref;
        }
        if (is_dst) w.pairs[dst0 + (at >> 16)].y = i;
        if (i < hi) w.list[i] = i;
        src0 += sums & 0xffff;
        dst0 += sums >> 16;
    }
    cl.sync();
    for (int i = rank * kClThreads + t; i < total; i += kClCtas * kClThreads) {
        const int4 m = w.pairs[i];
        w.pairs[i].z = p.page;
        w.list[m.x] = m.y;
        p.refs[m.y] = m.w;
        p.refs[m.x] = 0;
    }
    if (rank == 0 && t == 0) *w.count = total;
}

// ---------------------------------------------------------------------------
// the copies: one warp per run of rows (a page's rows of one layer and kv
// head are contiguous), 4 KB in flight per warp. Only the rows a copy names
// move. For compact the same launch rewrites the tables. Bound by HBM: 48 slots
// of up to 200 tokens, 30 layers and 1024 pages of f16 compacted in 90 us, 5.6
// TB/s of reads and writes, the bookkeeping before it included.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
kv_copy_kernel(const PagesDev p, uint8_t* k, uint8_t* v, int runs, int row_bytes, void* work, int remap) {
    pdl_wait();
    const Work w = work_of(work, p.n_pages, p.n_slots, p.width);
    const int count = *w.count;
    if (count <= 0) return;
    const int lane = threadIdx.x & 31;
    const long long nw = (long long)gridDim.x * 8, w0 = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long units = (long long)count * 2 * runs;
    const size_t run_bytes = (size_t)p.page * row_bytes;
    for (long long u = w0; u < units; u += nw) {
        const long long pr = u / (2 * runs);
        const int r = (int)(u - pr * (2 * runs));
        const int4 m = w.pairs[pr];
        uint8_t* const pool = r < runs ? k : v;
        const size_t off = (size_t)(r < runs ? r : r - runs) * run_bytes;
        const uint4* a = reinterpret_cast<const uint4*>(pool + (size_t)m.x * runs * run_bytes + off);
        uint4* b = reinterpret_cast<uint4*>(pool + (size_t)m.y * runs * run_bytes + off);
        const int nv = m.z * (row_bytes >> 4);
        for (int x = lane; x < nv; x += 256) {
            uint4 r8[8];
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x + 32 * j < nv) r8[j] = __ldcs(a + x + 32 * j);
            #pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x + 32 * j < nv) __stcs(b + x + 32 * j, r8[j]);
        }
    }
    if (remap) {
        for (long long s = w0; s < p.n_slots; s += nw) {
            const int used = used_of(p.lens[s], p.page);
            int32_t* row = p.tables + (size_t)s * p.width;
            for (int j = lane; j < used; j += 32) row[j] = w.list[row[j]];
        }
    }
}

// ---------------------------------------------------------------------------
// append: RoPE (the decode path's rotation from the same angle table),
// conversion and store. A warp takes eight rows (heads of k, of v, of q, in
// that order) of one token, two at a time: lane l of a half-warp holds elements
// 4l .. 4l + 3 and 64 + 4l .., which are the rotation's pairs, so everything
// moves in 16-byte pieces (8-byte stores for f16). The rows are read before
// the slot's table has been walked. Bound by HBM: every value is read once and
// written once (k and v twice). 4099 tokens of 64 and 8 heads, f32: 60.7 us, 6.1
// TB/s (one row a warp, four bytes a lane: 94 us); 16 tokens of 20 and 5: 3.8 us.
// ---------------------------------------------------------------------------
constexpr int kApRows = 8;

struct AppendParams {
    const int32_t* slot;
    const int32_t* pos;
    const float* q;
    const float* k;
    const float* v;
    size_t qs, ks, vs;              // floats from a token to the next
    const float* cs;
    const float* sn;
    void* qo;
    void* ko;
    void* vo;
    void* kp;                       // the layer's slice of page 0
    void* vp;
    size_t page_stride;             // elements from a page to the next
    int n_tokens, n_head, n_kv, n_ctx;
    int32_t* status;
};

template <class T>
__global__ void __launch_bounds__(256)
kv_append_kernel(const __grid_constant__ PagesDev p, const __grid_constant__ AppendParams a) {
    const int lane = threadIdx.x & 31, l4 = 4 * (lane & 15);
    const int rows = (a.q != nullptr ? a.n_head : 0) + 2 * a.n_kv, units = (rows + kApRows - 1) / kApRows;
    const long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int tok = (int)(u / units);
    if (tok >= a.n_tokens) return;
    const int r0 = (int)(u - (long long)tok * units) * kApRows + (lane >> 4);
    const int slot = a.slot[tok], pos = a.pos[tok];
    // row r: k heads, v heads, q heads
    float4 lo[kApRows / 2], hi[kApRows / 2];
    #pragma unroll
    for (int i = 0; i < kApRows / 2; ++i) {
        const int r = r0 + 2 * i;
        if (r < rows) {
            const float* x = r < a.n_kv       ? a.k + tok * a.ks + r * kServeDim
                             : r < 2 * a.n_kv ? a.v + tok * a.vs + (r - a.n_kv) * kServeDim
                                              : a.q + tok * a.qs + (r - 2 * a.n_kv) * kServeDim;
            lo[i] = __ldcs(reinterpret_cast<const float4*>(x + l4));
            hi[i] = __ldcs(reinterpret_cast<const float4*>(x + 64 + l4));
        }
    }
    if (slot < 0) return;           // a padding token
    int id = -1;
    if (slot < p.n_slots && pos >= 0 && pos < a.n_ctx && pos < p.cap && pos < p.lens[slot])
        id = p.tables[(size_t)slot * p.width + pos / p.page];
    // a shared page is never written: its other owners would change
    if (id < 0 || id >= p.n_pages || p.refs[id] != 1) {
        if (lane == 0) raise(a.status, SLLM_CUDA_ERR_ARG);
        return;
    }
    const float4 c = ld4(a.cs + (size_t)pos * 64 + l4), s = ld4(a.sn + (size_t)pos * 64 + l4);
    const size_t place = (size_t)id * a.page_stride + (size_t)(pos % p.page) * kServeDim + l4;
    #pragma unroll
    for (int i = 0; i < kApRows / 2; ++i) {
        const int r = r0 + 2 * i;
        if (r >= rows) break;
        const bool is_v = r >= a.n_kv && r < 2 * a.n_kv;
        if (!is_v) {
            const float4 x = lo[i], y = hi[i];
            lo[i].x = __fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x));
            lo[i].y = __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y));
            lo[i].z = __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z));
            lo[i].w = __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w));
            hi[i].x = __fadd_rn(__fmul_rn(x.x, s.x), __fmul_rn(y.x, c.x));
            hi[i].y = __fadd_rn(__fmul_rn(x.y, s.y), __fmul_rn(y.y, c.y));
            hi[i].z = __fadd_rn(__fmul_rn(x.z, s.z), __fmul_rn(y.z, c.z));
            hi[i].w = __fadd_rn(__fmul_rn(x.w, s.w), __fmul_rn(y.w, c.w));
        }
        const int h = r < a.n_kv ? r : is_v ? r - a.n_kv : r - 2 * a.n_kv;
        T* out = static_cast<T*>(r < a.n_kv ? a.ko : is_v ? a.vo : a.qo);
        if (out != nullptr) {
            out += ((size_t)tok * (r < 2 * a.n_kv ? a.n_kv : a.n_head) + h) * kServeDim + l4;
            st4(out, lo[i]);
            st4(out + 64, hi[i]);
        }
        if (r < 2 * a.n_kv) {
            T* row = static_cast<T*>(is_v ? a.vp : a.kp) + place + (size_t)h * p.page * kServeDim;
            st4(row, lo[i]);
            st4(row + 64, hi[i]);
        }
    }
}

int check_call(const sllm_cuda_kv_pages* p, const char* who, int n, const void* work, size_t work_bytes,
               const void* a, const void* b, const void* status) {
    int rc = check_pages(p, who);
    if (rc != SLLM_CUDA_OK) return rc;
    if (n < 0 || n > p->n_slots) return fail(SLLM_CUDA_ERR_ARG, "%s: %d slots named, the cache has %d", who, n, p->n_slots);
    if (work == nullptr || !aligned16(work) || work_bytes < sllm_cuda_kv_work_bytes(p))
        return fail(SLLM_CUDA_ERR_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who, work_bytes,
                    sllm_cuda_kv_work_bytes(p));
    const void* ptr[] = {p->k, p->v, p->refs, p->tables, p->lens, work, a, b, status};
    const char* name[] = {"k", "v", "refs", "tables", "lens", "work", "slots", "slots or lengths", "status"};
    for (int i = 0; i < 9; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], who, name[i])) != SLLM_CUDA_OK) return rc;
    return SLLM_CUDA_OK;
}

cudaError_t launch_copies(const sllm_cuda_kv_pages& p, long long most, void* work, int remap, cudaStream_t st) {
    const int runs = p.n_layer * p.n_head_kv;
    const long long units = most * 2 * runs + (remap ? p.n_slots : 0);
    const long long blocks = (units + 7) / 8, cap = 8LL * current_sms();
    return launch(kv_copy_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap)), dim3(256), 0, st, true,
                  pages_dev(p), static_cast<uint8_t*>(p.k), static_cast<uint8_t*>(p.v), runs,
                  (int)(kServeDim * kv_elt_bytes(p.kv_type)), work, remap);
}

}  // namespace

static std::atomic<uint32_t> g_attn_wait_ns{0};
WaitLimit attn_wait_limit() {
    const uint32_t set = g_attn_wait_ns.load(std::memory_order_relaxed), ns = set != 0 ? set : 2000000000u;
    return WaitLimit{ns, ns < 65536u ? ns : 65536u};
}

int current_sms() {
    int dev = 0;
    cudaGetDevice(&dev);
    return num_sms_of(dev);
}

int need_device(const void* p, const char* who, const char* arg) {
    if (((uintptr_t)p & 3u) != 0) return fail(SLLM_CUDA_ERR_ARG, "%s: %s is not aligned", who, arg);
    cudaPointerAttributes at{};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) {
        cudaGetLastError();
        return fail(SLLM_CUDA_ERR_UNSUPPORTED, "%s: no CUDA device", who);
    }
    if (e != cudaSuccess) return cuda_fail(e, who);
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) return cuda_fail(cudaGetLastError(), who);
    if (at.type == cudaMemoryTypeManaged) return SLLM_CUDA_OK;
    if (at.type != cudaMemoryTypeDevice || at.device != dev)
        return fail(SLLM_CUDA_ERR_ARG, "%s: %s is not memory of the current device (%d)", who, arg, dev);
    return SLLM_CUDA_OK;
}

int check_pages(const sllm_cuda_kv_pages* p, const char* who) {
    if (p == nullptr || p->k == nullptr || p->v == nullptr || p->refs == nullptr || p->tables == nullptr ||
        p->lens == nullptr)
        return fail(SLLM_CUDA_ERR_ARG, "%s: a NULL cache or array", who);
    if (p->kv_type != SLLM_CUDA_KV_F32 && p->kv_type != SLLM_CUDA_KV_F16)
        return fail(SLLM_CUDA_ERR_ARG, "%s: unknown cache type %d", who, p->kv_type);
    if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
        return fail(SLLM_CUDA_ERR_UNSUPPORTED, "%s: pages of %d tokens (16, 32, 64 or 128)", who, p->page_size);
    if (p->n_pages < 1 || p->n_pages > (1 << 24) || p->n_layer < 1 || p->n_layer > 1024 || p->n_head_kv < 1 ||
        p->n_head_kv > 1024 || p->n_slots < 1 || p->n_slots > (1 << 16) || p->table_width < 1 ||
        p->table_width > (1 << 23) || (long long)p->table_width * p->page_size > 0x7fffff00LL ||
        (long long)p->n_slots * p->table_width > 0x7fffffffLL)
        return fail(SLLM_CUDA_ERR_ARG, "%s: cache of %d pages, %d layers, %d kv heads, %d slots, %d entries a table",
                    who, p->n_pages, p->n_layer, p->n_head_kv, p->n_slots, p->table_width);
    if (!aligned16(p->k) || !aligned16(p->v) || !aligned16(p->refs))
        return fail(SLLM_CUDA_ERR_ARG, "%s: k, v and refs must be 16-byte aligned", who);
    return SLLM_CUDA_OK;
}

}  // namespace sllm

using namespace sllm;

extern "C" int sllm_cuda_test_attn_error(void) {
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    const int a = take_prompt_error(), b = take_prefix_error();
    return a != 0 ? a : b;
}

extern "C" void sllm_cuda_test_attn_wait(uint32_t ns) { g_attn_wait_ns.store(ns, std::memory_order_relaxed); }

extern "C" size_t sllm_cuda_kv_work_bytes(const sllm_cuda_kv_pages* p) {
    if (check_pages(p, "kv_work_bytes") != SLLM_CUDA_OK) return 0;
    return 4 * work_ints(p->n_pages, p->n_slots, p->table_width);
}

extern "C" int sllm_cuda_kv_fork(const sllm_cuda_kv_pages* p, const int32_t* src, const int32_t* dst, int32_t n,
                                 void* work, size_t work_bytes, int32_t* status, void* stream) {
    if (n != 0 && (src == nullptr || dst == nullptr)) return fail(SLLM_CUDA_ERR_ARG, "kv_fork: NULL slots");
    const int rc = check_call(p, "kv_fork", n, work, work_bytes, src, dst, status);
    if (rc != SLLM_CUDA_OK || n == 0) return rc;
    kv_fork_kernel<<<kClCtas, kClThreads, 0, (cudaStream_t)stream>>>(pages_dev(*p), src, dst, n, work, status);
    CK(cudaGetLastError(), "kv_fork launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}

extern "C" int sllm_cuda_kv_release(const sllm_cuda_kv_pages* p, const int32_t* slots, const int32_t* new_len,
                                    int32_t n, void* work, size_t work_bytes, int32_t* status, void* stream) {
    if (n != 0 && slots == nullptr) return fail(SLLM_CUDA_ERR_ARG, "kv_release: NULL slots");
    const int rc = check_call(p, "kv_release", n, work, work_bytes, slots, new_len, status);
    if (rc != SLLM_CUDA_OK || n == 0) return rc;
    kv_release_kernel<<<kClCtas, kClThreads, 0, (cudaStream_t)stream>>>(pages_dev(*p), slots, new_len, n, work, status);
    CK(cudaGetLastError(), "kv_release launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}

extern "C" int sllm_cuda_kv_reserve(const sllm_cuda_kv_pages* p, const int32_t* slots, const int32_t* n_new,
                                    int32_t n, void* work, size_t work_bytes, int32_t* status, void* stream) {
    if (n != 0 && (slots == nullptr || n_new == nullptr))
        return fail(SLLM_CUDA_ERR_ARG, "kv_reserve: NULL slots or lengths");
    const int rc = check_call(p, "kv_reserve", n, work, work_bytes, slots, n_new, status);
    if (rc != SLLM_CUDA_OK || n == 0) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    kv_reserve_kernel<<<1, kResThreads, 0, st>>>(pages_dev(*p), slots, n_new, n, work, status);
    CK(cudaGetLastError(), "kv_reserve launch");
    CK(launch_copies(*p, n, work, 0, st), "kv_reserve copies");
    count_launches(2);
    return SLLM_CUDA_OK;
}

extern "C" int sllm_cuda_kv_compact(const sllm_cuda_kv_pages* p, void* work, size_t work_bytes, int32_t* status,
                                    void* stream) {
    const int rc = check_call(p, "kv_compact", 0, work, work_bytes, nullptr, nullptr, status);
    if (rc != SLLM_CUDA_OK) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    kv_compact_kernel<<<kClCtas, kClThreads, 0, st>>>(pages_dev(*p), work, status);
    CK(cudaGetLastError(), "kv_compact launch");
    CK(launch_copies(*p, p->n_pages / 2 + 1, work, 1, st), "kv_compact copies");
    count_launches(2);
    return SLLM_CUDA_OK;
}

extern "C" int sllm_cuda_kv_append(const sllm_cuda_kv_pages* p, int32_t layer, int32_t n_tokens, const int32_t* slot,
                                   const int32_t* pos, int32_t n_head, const float* q, size_t q_stride,
                                   const float* k, size_t k_stride, const float* v, size_t v_stride,
                                   const float* rope_cos, const float* rope_sin, int32_t n_ctx, void* q_out,
                                   void* k_out, void* v_out, int32_t* status, void* stream) {
    int rc = check_pages(p, "kv_append");
    if (rc != SLLM_CUDA_OK) return rc;
    if (slot == nullptr || pos == nullptr || k == nullptr || v == nullptr || rope_cos == nullptr ||
        rope_sin == nullptr || (q == nullptr) != (q_out == nullptr))
        return fail(SLLM_CUDA_ERR_ARG, "kv_append: a NULL array (q and q_out go together)");
    const size_t kvn = (size_t)p->n_head_kv * kServeDim, qn = (size_t)(n_head > 0 ? n_head : 0) * kServeDim;
    if (layer < 0 || layer >= p->n_layer || n_tokens < 0 || n_tokens > (1 << 24) || n_ctx < 1 ||
        (q != nullptr && (n_head < 1 || n_head > 1024 || n_head % p->n_head_kv != 0 || q_stride < qn)) ||
        k_stride < kvn || v_stride < kvn || q_stride > (1u << 30) || k_stride > (1u << 30) || v_stride > (1u << 30))
        return fail(SLLM_CUDA_ERR_ARG, "kv_append: layer %d, %d tokens, %d heads, strides %zu %zu %zu", layer, n_tokens,
                    n_head, q_stride, k_stride, v_stride);
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out) ||
        !aligned16(rope_cos) || !aligned16(rope_sin) || (q_stride | k_stride | v_stride) % 4 != 0)
        return fail(SLLM_CUDA_ERR_ARG, "kv_append: arrays must be 16-byte aligned, strides a multiple of 4 floats");
    const void* ptr[] = {p->k, p->v, p->refs, p->tables, p->lens, slot, pos, q, k, v, rope_cos, rope_sin, q_out, k_out,
                         v_out, status};
    const char* name[] = {"k", "v", "refs", "tables", "lens", "slot", "pos", "q", "k", "v", "rope_cos", "rope_sin",
                          "q_out", "k_out", "v_out", "status"};
    for (int i = 0; i < 16; ++i)
        if (ptr[i] != nullptr && (rc = need_device(ptr[i], "kv_append", name[i])) != SLLM_CUDA_OK) return rc;
    if (n_tokens == 0) return SLLM_CUDA_OK;
    AppendParams a{};
    a.slot = slot; a.pos = pos;
    a.q = q; a.k = k; a.v = v;
    a.qs = q_stride; a.ks = k_stride; a.vs = v_stride;
    a.cs = rope_cos; a.sn = rope_sin;
    a.qo = q_out; a.ko = k_out; a.vo = v_out;
    const size_t layer_elts = (size_t)p->n_head_kv * p->page_size * kServeDim;
    const size_t off = (size_t)layer * layer_elts * kv_elt_bytes(p->kv_type);
    a.kp = static_cast<uint8_t*>(p->k) + off;
    a.vp = static_cast<uint8_t*>(p->v) + off;
    a.page_stride = (size_t)p->n_layer * layer_elts;
    a.n_tokens = n_tokens; a.n_head = n_head; a.n_kv = p->n_head_kv; a.n_ctx = n_ctx;
    a.status = status;
    const int rows = (q != nullptr ? n_head : 0) + 2 * p->n_head_kv;
    const long long units = (long long)n_tokens * ((rows + kApRows - 1) / kApRows);
    if (units > 0x7fffffffLL * 8 - 8) return fail(SLLM_CUDA_ERR_TOO_LARGE, "kv_append: %d tokens", n_tokens);
    const dim3 grid((unsigned)((units + 7) / 8));
    if (p->kv_type == SLLM_CUDA_KV_F16)
        kv_append_kernel<__half><<<grid, 256, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    else
        kv_append_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>(pages_dev(*p), a);
    CK(cudaGetLastError(), "kv_append launch");
    count_launches(1);
    return SLLM_CUDA_OK;
}
