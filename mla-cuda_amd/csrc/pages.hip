// Pages of a cache that requests share: forking requests (their tables, and which pages need a copy),
// making a pool dense again, and the copies themselves.  Tables and the ring of free pages are those
// of cache8.hip's extend; a page is held by every table row that names it among its request's pages,
// so that who holds what follows from the tables alone and nothing is counted between calls.
//
// A small pool is done by one workgroup in one launch, with a word a page in LDS; a large one in launches
// over parts of it, with the words in memory.  No order of atomics or of writers shows in a result.
// Bound by launches and by loads that wait on one another (lengths, entries, words), some tens of KB of them: a fork of
// 8 requests over 90 pages 5.6 us, compaction of 522 pages 8.0; 256 requests over 42,000 pages 14.6 us in four
// launches, compaction of 113,000 pages 17.7 in five.

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace mla {

namespace {

typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kRange = kPageRange;            // pages a workgroup owns
constexpr int kPer = kRange / kThreads;       // consecutive ones a thread
// a large pool's parts: few pages a thread, whose stores lie apart (moves and ring of 111,000 pages 10.1 us with 16
// of them, 5.4 with 4)
constexpr int kPartThreads = 256, kPartWaves = kPartThreads / 64, kPartPer = 4, kPart = kPartThreads * kPartPer;
constexpr int kSmall = kPartThreads * kPer;   // pages that so many threads keep in LDS

// Sum over the threads in front of this one of a workgroup of W waves; *total that over all.
template <int W = kWaves>
__device__ __forceinline__ int block_scan(int v, int* waves, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
    s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xF, 0xF, true);    // row_shr:1, 2, 4, 8
    s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xA, 0xF, false);   // row_bcast:15, 31
    s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xC, 0xF, false);
    __syncthreads();                          // the last use of `waves` is over
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    int before = s - v, all = 0;
    #pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < wave) before += waves[w];
        all += waves[w];
    }
    *total = all;
    return before;
}

__global__ void __launch_bounds__(256) pages_clear_kernel(v4u_t* p, int64_t n) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) p[i] = v4u_t{0, 0, 0, 0};
}
hipError_t clear_pages(void* p, int64_t bytes, hipStream_t stream) {   // 16-byte aligned, a multiple of 16
    const int64_t n = bytes / 16;
    hipLaunchKernelGGL(pages_clear_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 8 * kNumCUs)), dim3(256), 0,
                       stream, static_cast<v4u_t*>(p), n);
    return hipGetLastError();
}

__device__ __forceinline__ int pages_of(int tokens, int page) { return (int)(((int64_t)tokens + page - 1) / page); }
// place i past the ring's head, for head < n and i < n (or i = n: head again)
__device__ __forceinline__ int ring_at(int head, int i, int n) {
    const uint32_t p = (uint32_t)head + (uint32_t)i;
    return (int)(p >= (uint32_t)n ? p - (uint32_t)n : p);
}
// this thread's N consecutive words of a range
template <int N> struct Words { uint32_t w[N]; };
template <int N>
__device__ __forceinline__ Words<N> own_words(const uint32_t* words) {
    Words<N> x;
    #pragma unroll
    for (int i = 0; i < N; i += 4) {
        const v4u_t v = *reinterpret_cast<const v4u_t*>(words + threadIdx.x * N + i);
        #pragma unroll
        for (int k = 0; k < 4; ++k) x.w[i + k] = v[k];
    }
    return x;
}

// ---- fork -----------------------------------------------------------------------------------
// Request b continues the first n = min(keep_lens[b], L[p]) tokens of request p = parents[b].  A
// page's word says how it is held: not (0), before the call only (1), as the open page of request b
// and of none in front (kOpen - b), as a whole page (kWhole).  A larger word wins, so that the word
// does not depend on the order of its holders.  An open page stays with the request that its word
// names; the others that would write it, all of them if it is somebody's whole page, take a copy.
constexpr uint32_t kHeld = 1u, kOpen = 0x7fffffffu, kWhole = 0xffffffffu;
constexpr int kNoCopy = -0x7fffffff - 1;      // no free page (whatever a ring may hold)

struct ForkArgs {
    const int* parents;
    const int* keep;
    const int* lens;
    const int* table;
    const int* state;        // {head, count}
    int* ring;
    int* lens_out;
    int* table_out;
    int* state_out;
    int* copies;             // [B][2]
    uint32_t* words;         // [parts * kPart] (a large pool)
    int* freed;              // [parts]
    int B, page, max_pages, num_pages, parts;
};

struct ForkRow { int src, n; };
__device__ __forceinline__ int fork_len(const ForkArgs& a, int b) {
    return (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
}
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int b) {
    const int p = a.parents[b];
    if (p < 0 || p >= a.B) return {0, 0};
    return {p, min(max(a.keep[b], 0), fork_len(a, p))};
}

// The marks of rows wave, wave + waves, .. of a.B, kRows of them at a time, 128 entries of each: all loads
// before the first mark.
struct ForkMark { int src, have, whole, held; };
__device__ __forceinline__ ForkMark fork_mark(const ForkArgs& a, int b) {
    const ForkRow r = fork_row(a, b);
    return {r.src, pages_of(fork_len(a, b), a.page), r.n / a.page, pages_of(r.n, a.page)};
}
template <int kRows, class Row>
__device__ __forceinline__ void fork_marks(const ForkArgs& a, uint32_t* words, int b0, int nb, int wave, int waves, Row row) {
    const int lane = threadIdx.x & 63;
    auto mark = [&](int page, uint32_t w) __attribute__((always_inline)) {
        if (page >= 0 && page < a.num_pages) atomicMax(&words[page], w);
    };
    for (int r0 = wave; r0 < nb; r0 += kRows * waves) {
        ForkMark m[kRows];
        int most = 0;
        #pragma unroll
        for (int k = 0; k < kRows; ++k) {
            m[k] = r0 + k * waves < nb ? row(r0 + k * waves) : ForkMark{0, 0, 0, 0};
            most = max(most, max(m[k].have, m[k].held));
        }
        for (int j0 = lane; j0 < most; j0 += 128) {
            int own[kRows][2], from[kRows][2];
            #pragma unroll
            for (int k = 0; k < kRows; ++k)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = j0 + 64 * i;
                    own[k][i] = j < m[k].have ? a.table[(int64_t)(b0 + r0 + k * waves) * a.max_pages + j] : -1;
                    from[k][i] = j < m[k].held ? a.table[(int64_t)m[k].src * a.max_pages + j] : -1;
                }
            #pragma unroll
            for (int k = 0; k < kRows; ++k)
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mark(own[k][i], kHeld);
                    mark(from[k][i], j0 + 64 * i < m[k].whole ? kWhole : kOpen - (uint32_t)(b0 + r0 + k * waves));
                }
        }
    }
}

// The plan of all requests: each one's copy, if it needs one and a free page is left for it.
// put(b, row, old page, fresh page or kNoCopy, whether it is cut back to its whole pages)
template <int W, class Word, class Put>
__device__ __forceinline__ int fork_plan(const ForkArgs& a, int head, int count, int* waves, Word word, Put put) {
    const int per = (a.B + 64 * W - 1) / (64 * W);
    const int b0 = min(a.B, (int)threadIdx.x * per), b1 = min(a.B, b0 + per);
    auto needs = [&](int b, ForkRow r, int* old) __attribute__((always_inline)) {
        if (r.n % a.page == 0) return false;
        *old = a.table[(int64_t)r.src * a.max_pages + r.n / a.page];
        return *old >= 0 && *old < a.num_pages && word(*old) != kOpen - (uint32_t)b;
    };
    int n = 0, old = -1, total;
    for (int b = b0; b < b1; ++b) n += needs(b, fork_row(a, b), &old);
    int order = block_scan<W>(n, waves, &total);
    for (int b = b0; b < b1; ++b) {
        const ForkRow r = fork_row(a, b);
        const bool need = needs(b, r, &old), given = need && order < count;
        put(b, r, old, given ? a.ring[ring_at(head, order, a.num_pages)] : kNoCopy, need && !given);
        order += need;
    }
    return min(total, count);
}

// This request's new table row, by a wave.
__device__ __forceinline__ void fork_write(const ForkArgs& a, int b, int src, int n, int fresh) {
    const int whole = n / a.page, held = pages_of(n, a.page);
    const int* from = a.table + (int64_t)src * a.max_pages;
    int* to = a.table_out + (int64_t)b * a.max_pages;
    for (int j = threadIdx.x & 63; j < a.max_pages; j += 64)
        to[j] = j >= held ? 0 : j < whole || fresh == kNoCopy ? from[j] : fresh;
}

// The pages of `x`, from lo on, that nobody holds any more, behind the ring's tail: `before` of them come
// first.  Their number.
template <int W, int N>
__device__ __forceinline__ int fork_free(const ForkArgs& a, int lo, const Words<N>& x, int before, int head, int count, int* waves) {
    int n = 0, total;
    #pragma unroll
    for (int i = 0; i < N; ++i) n += x.w[i] == kHeld;
    int k = before + block_scan<W>(n, waves, &total);
    #pragma unroll
    for (int i = 0; i < N; ++i)
        if (x.w[i] == kHeld) {
            if (k < a.num_pages - count) a.ring[ring_at(head, count + k, a.num_pages)] = lo + threadIdx.x * N + i;
            ++k;
        }
    return total;
}

__device__ __forceinline__ void ring_state(const int* state, int n, int* head, int* count) {
    *head = state[0] % n;
    if (*head < 0) *head += n;
    *count = min(max(state[1], 0), n);
}

struct ForkInfo { int src, n, fresh; };

// What a request's plan leaves behind, and its numbers for its row.
__device__ __forceinline__ ForkInfo fork_put(const ForkArgs& a, int b, const ForkRow& r, int old, int fresh, bool cut) {
    const int n = cut ? r.n / a.page * a.page : r.n;
    a.lens_out[b] = n;
    a.copies[2 * b] = fresh == kNoCopy ? -1 : old;
    a.copies[2 * b + 1] = fresh == kNoCopy ? -1 : fresh;
    return {r.src, n, fresh};
}

// A pool that a workgroup of W waves holds (kPer pages a thread) and at most a request a thread: few waves, where
// that is enough, meet sooner (beams of 8 requests 6.0 us with 16 of them).
template <int W>
__global__ void __launch_bounds__(64 * W) fork_one_kernel(ForkArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t words[64 * W * kPer];
    __shared__ int waves[W];
    __shared__ ForkMark rows[64 * W];
    __shared__ ForkInfo info[64 * W];
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int i = tid; i < 64 * W * kPer / 4; i += 64 * W) reinterpret_cast<v4u_t*>(words)[i] = v4u_t{0, 0, 0, 0};
    if (tid < a.B) rows[tid] = fork_mark(a, tid);
    int head, count;
    ring_state(a.state, a.num_pages, &head, &count);
    __syncthreads();
    fork_marks<4>(a, words, 0, a.B, wave, W, [&](int b) { return rows[b]; });
    __syncthreads();
    const int taken = fork_plan<W>(a, head, count, waves, [&](int page) { return words[page]; },
                                        [&](int b, const ForkRow& r, int old, int fresh, bool cut) __attribute__((always_inline)) {
        info[b] = fork_put(a, b, r, old, fresh, cut);
    });
    const int freed = fork_free<W>(a, 0, own_words<kPer>(words), 0, head, count, waves);
    if (tid == 0) {
        a.state_out[0] = ring_at(head, taken, a.num_pages);
        a.state_out[1] = min(count - taken + freed, a.num_pages);
    }
    __syncthreads();
    for (int b = wave; b < a.B; b += W) fork_write(a, b, info[b].src, info[b].n, info[b].fresh);
}

// A large pool or batch: words in memory (cleared), the parts' freed pages, then those to the ring and the rows.
__global__ void __launch_bounds__(256) fork_mark_kernel(ForkArgs a) {
    const int wave = blockIdx.x * 4 + (threadIdx.x >> 6);
    fork_marks<1>(a, a.words, 0, a.B, wave, gridDim.x * 4, [&](int b) { return fork_mark(a, b); });
}
__device__ __forceinline__ Words<kPartPer> fork_part(const ForkArgs& a, int g) {
    return own_words<kPartPer>(a.words + (int64_t)g * kPart);
}

__global__ void __launch_bounds__(kPartThreads) fork_freed_kernel(ForkArgs a) {
    __shared__ int waves[kPartWaves];
    const Words<kPartPer> x = fork_part(a, blockIdx.x);
    int n = 0, total;
    #pragma unroll
    for (int i = 0; i < kPartPer; ++i) n += x.w[i] == kHeld;
    block_scan<kPartWaves>(n, waves, &total);
    if (threadIdx.x == 0) a.freed[blockIdx.x] = total;
}

// Workgroups [0, parts) free pages, the others write kPartWaves rows each.
__global__ void __launch_bounds__(kPartThreads) fork_emit_kernel(ForkArgs a) {
    __shared__ int waves[kPartWaves];
    __shared__ ForkInfo info[kPartWaves];
    const int tid = threadIdx.x, g = blockIdx.x;
    int head, count;
    ring_state(a.state, a.num_pages, &head, &count);
    if (g < a.parts) {
        const Words<kPartPer> x = fork_part(a, g);
        int n = 0, before;
        for (int r = tid; r < g; r += kPartThreads) n += a.freed[r];
        block_scan<kPartWaves>(n, waves, &before);
        fork_free<kPartWaves>(a, g * kPart, x, before, head, count, waves);
        return;
    }
    const int r0 = (g - a.parts) * kPartWaves;
    const int taken = fork_plan<kPartWaves>(a, head, count, waves, [&](int page) { return a.words[page]; },
                                            [&](int b, const ForkRow& r, int old, int fresh, bool cut) __attribute__((always_inline)) {
        if (b >= r0 && b < r0 + kPartWaves) info[b - r0] = fork_put(a, b, r, old, fresh, cut);
    });
    if (r0 == 0) {
        int n = 0, freed;
        for (int r = tid; r < a.parts; r += kPartThreads) n += a.freed[r];
        block_scan<kPartWaves>(n, waves, &freed);
        if (tid == 0) {
            a.state_out[0] = ring_at(head, taken, a.num_pages);
            a.state_out[1] = (int)min((int64_t)count - taken + freed, (int64_t)a.num_pages);
        }
    }
    __syncthreads();
    const int b = r0 + (tid >> 6);
    if (b < a.B) fork_write(a, b, info[tid >> 6].src, info[tid >> 6].n, info[tid >> 6].fresh);
}

// ---- compact --------------------------------------------------------------------------------
// The pages that tables hold (U of them) and the free ones of the ring, in the order of their
// numbers: the first U are to be held, the others free.  A held page past the first U moves to a free
// one among them, both in order.  Pages that are neither (a program's own) stay out of it.
constexpr uint32_t kUsed = 1u, kFree = 2u;   // a page's word

struct CompactArgs {
    const int* lens;
    const int* table;
    const int* ring;
    const int* state;
    int* table_out;
    int* ring_out;
    int* state_out;
    int* copies;             // [room][2]
    uint8_t* used;           // [ranges * kPart] past one workgroup's range: whether a page is held,
    uint8_t* free;           // and whether the ring has it
    int2* sums;              // [ranges] {held, free} pages of each kPart
    int* to;                 // [num_pages] which move a page is
    int* cut;                // the first page that is not among the first U
    int B, page, max_pages, num_pages, ranges, room;
};

// How many of a thread's pages are held and free, as one number for one sum over a workgroup (whose range's counts
// are below 2^16 each).
template <int N>
__device__ __forceinline__ int held_free(const Words<N>& x) {
    int n = 0;
    #pragma unroll
    for (int i = 0; i < N; ++i) n += (x.w[i] & kUsed) != 0 ? 1 : x.w[i] == kFree ? 1 << 16 : 0;
    return n;
}
static_assert(kRange < 1 << 15, "two counts a number");

// Held and free pages in front of this thread's, of a range with `front` before it; `all` of the range alone.
template <int W, int N>
__device__ __forceinline__ int2 in_front(const Words<N>& x, int2 front, int* waves, int2* all) {
    int total;
    const int n = block_scan<W>(held_free(x), waves, &total);
    *all = make_int2(total & 0xffff, total >> 16);
    return make_int2(front.x + (n & 0xffff), front.y + (n >> 16));
}

// The words of a pool that a workgroup of W waves holds.
template <int W>
__device__ __forceinline__ void compact_words(const CompactArgs& a, uint32_t* words) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < 64 * W * kPer / 4; i += 64 * W) reinterpret_cast<v4u_t*>(words)[i] = v4u_t{0, 0, 0, 0};
    int head, count;
    ring_state(a.state, a.num_pages, &head, &count);
    __syncthreads();
    auto mark = [&](int page, uint32_t w) __attribute__((always_inline)) {
        if (page >= 0 && page < a.num_pages) atomicOr(&words[page], w);
    };
    constexpr int kRun = 8;
    for (int b0 = wave; b0 < a.B; b0 += 4 * W) {     // four rows at a time, 128 entries of each
        int have[4], most = 0;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int b = min(b0 + k * W, a.B - 1);
            const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
            have[k] = b0 + k * W < a.B ? pages_of(len, a.page) : 0;
            most = max(most, have[k]);
        }
        for (int j0 = lane; j0 < most; j0 += 128) {
            int p[kRun];
            #pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const int j = j0 + 64 * (k & 1);
                p[k] = j < have[k >> 1] ? a.table[(int64_t)(b0 + (k >> 1) * W) * a.max_pages + j] : -1;
            }
            #pragma unroll
            for (int k = 0; k < kRun; ++k) mark(p[k], kUsed);
        }
    }
    for (int i = tid; i < count; i += kRun * (64 * W)) {
        int p[kRun];
        #pragma unroll
        for (int k = 0; k < kRun; ++k)
            p[k] = i + k * (64 * W) < count ? a.ring[ring_at(head, i + k * (64 * W), a.num_pages)] : -1;
        #pragma unroll
        for (int k = 0; k < kRun; ++k) mark(p[k], kFree);
    }
    __syncthreads();
}

// The cut, with U pages held in all, if it is among this thread's pages (from p0 on, `front` held and free ones in
// front of them): the page, and the held pages in front of it.
template <int N>
__device__ __forceinline__ bool compact_cut(int U, int p0, const Words<N>& x, int2 front, int* page, int* used) {
    const int c = held_free(x), n = (c & 0xffff) + (c >> 16);
    int held = front.x, rank = front.x + front.y;
    if (rank > U || rank + n <= U) return false;
    #pragma unroll
    for (int i = 0; i < N; ++i) {
        if (x.w[i] == 0) continue;
        if (rank == U) {
            *page = p0 + i;
            *used = held;
        }
        ++rank;
        held += (x.w[i] & kUsed) != 0;
    }
    return true;
}

// Moves and free pages among this thread's: hold(page, move) for a page that moves, hole(page, move) for one
// that is moved to.
template <int N, class Hold, class Hole>
__device__ __forceinline__ void compact_emit(const CompactArgs& a, int U, int p0, const Words<N>& x, int2 front,
                                             int used_below, Hold hold, Hole hole) {
    int used = front.x, free = front.y;
    #pragma unroll
    for (int i = 0; i < N; ++i) {
        if (x.w[i] == 0) continue;
        const int rank = used + free, p = p0 + i;
        if (rank >= U) a.ring_out[rank - U] = p;     // free after the call
        if (x.w[i] & kUsed) {
            if (rank >= U) hold(p, used - used_below);
            ++used;
        } else {
            if (rank < U) hole(p, free);
            ++free;
        }
    }
}
// A row's entries j0, j0 + step, .. through the moves.
template <class To>
__device__ __forceinline__ void compact_row(const CompactArgs& a, int b, int j0, int end, int step, int cut, To to) {
    const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
    const int have = pages_of(len, a.page);
    for (int j = j0; j < end; j += step) {
        int p = 0;
        if (j < have) {
            p = a.table[(int64_t)b * a.max_pages + j];
            if (p >= cut && p < a.num_pages) p = to(p);
        }
        a.table_out[(int64_t)b * a.max_pages + j] = p;
    }
}

// A large pool: bytes a page, cleared and written plainly (all writers write 1), then the parts' sums, then the
// moves, then the table.
// A wave marks a row of the table, and a workgroup its share of the ring.
__global__ void __launch_bounds__(256) compact_mark_kernel(CompactArgs a) {
    const int lane = threadIdx.x & 63;
    constexpr int kRun = 8;
    for (int b = blockIdx.x * 4 + (threadIdx.x >> 6); b < a.B; b += gridDim.x * 4) {
        const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
        const int have = pages_of(len, a.page);
        for (int j = lane; j < have; j += kRun * 64) {
            int p[kRun];
            #pragma unroll
            for (int k = 0; k < kRun; ++k) p[k] = j + 64 * k < have ? a.table[(int64_t)b * a.max_pages + j + 64 * k] : -1;
            #pragma unroll
            for (int k = 0; k < kRun; ++k)
                if (p[k] >= 0 && p[k] < a.num_pages) a.used[p[k]] = 1;
        }
    }
    int head, count;
    ring_state(a.state, a.num_pages, &head, &count);
    for (int i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) {
        const int p = a.ring[ring_at(head, i, a.num_pages)];
        if (p >= 0 && p < a.num_pages) a.free[p] = 1;
    }
}

// this thread's words of part g
__device__ __forceinline__ Words<kPartPer> part_words(const CompactArgs& a, int g) {
    static_assert(kPartPer == 4, "4 bytes a thread");
    const int64_t at = (int64_t)g * kPartThreads + threadIdx.x;
    const uint32_t u = reinterpret_cast<const uint32_t*>(a.used)[at], f = reinterpret_cast<const uint32_t*>(a.free)[at];
    Words<kPartPer> x;
    #pragma unroll
    for (int i = 0; i < kPartPer; ++i) x.w[i] = u >> (8 * i) & 1u ? kUsed : (f >> (8 * i) & 1u) * kFree;
    return x;
}

__global__ void __launch_bounds__(kPartThreads) compact_sums_kernel(CompactArgs a) {
    __shared__ int waves[kPartWaves];
    const Words<kPartPer> x = part_words(a, blockIdx.x);
    int all;
    block_scan<kPartWaves>(held_free(x), waves, &all);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = make_int2(all & 0xffff, all >> 16);
}

__global__ void __launch_bounds__(kPartThreads) compact_emit_kernel(CompactArgs a) {
    __shared__ int waves[kPartWaves];
    __shared__ int cut_at[2];    // the cut: page, held pages in front of it
    const int tid = threadIdx.x, lane = tid & 63, g = blockIdx.x;
    const Words<kPartPer> own = part_words(a, g);
    // sums in front of this part and of all, then the part of the cut: in every wave, 64 parts at a time
    int u = 0, f = 0, uu = 0, ff = 0;
    for (int r = lane; r < a.ranges; r += 64) {
        const int2 x = a.sums[r];
        uu += x.x;
        ff += x.y;
        if (r < g) { u += x.x; f += x.y; }
    }
    const int2 front = make_int2(wave_sum(u), wave_sum(f));
    const int U = wave_sum(uu), left = wave_sum(ff);
    int2 cut_front = make_int2(0, 0), all;
    int base = 0, used = 0, at = -1;
    for (int r0 = 0; r0 < a.ranges && at < 0; r0 += 64) {
        const int2 x = r0 + lane < a.ranges ? a.sums[r0 + lane] : make_int2(0, 0);
        int both = x.x + x.y, held = x.x;
        for (int i = 1; i < 64; i *= 2) {
            const int p = __shfl_up(both, i), q = __shfl_up(held, i);
            if (lane >= i) { both += p; held += q; }
        }
        const int before = base + both - x.x - x.y;
        const uint64_t m = __builtin_amdgcn_ballot_w64(before <= U && U < before + x.x + x.y);
        if (m) {
            const int k = __builtin_ctzll(m);
            at = r0 + k;
            cut_front.x = used + __shfl(held - x.x, k);
            cut_front.y = __shfl(before, k) - cut_front.x;
        }
        base += __shfl(both, 63);
        used += __shfl(held, 63);
    }
    int cut = a.num_pages, used_below = U;       // without a free page nothing is past the first U
    if (at >= 0) {
        const Words<kPartPer> x = part_words(a, at);
        const int2 n = in_front<kPartWaves>(x, cut_front, waves, &all);
        int p, held;
        if (compact_cut(U, at * kPart + tid * kPartPer, x, n, &p, &held)) {
            cut_at[0] = p;
            cut_at[1] = held;
        }
        __syncthreads();
        cut = cut_at[0];
        used_below = cut_at[1];
    }
    compact_emit(a, U, g * kPart + tid * kPartPer, own, in_front<kPartWaves>(own, front, waves, &all), used_below,
                 [&](int p, int k) { a.to[p] = k; if (k < a.room) a.copies[2 * k] = p; },
                 [&](int p, int k) { if (k < a.room) a.copies[2 * k + 1] = p; });
    // what is past the moves and the free pages
    const int moves = U - used_below;
    for (int64_t k = moves + (int64_t)g * kPartThreads + tid; k < a.room; k += (int64_t)a.ranges * kPartThreads)
        a.copies[2 * k] = a.copies[2 * k + 1] = -1;
    for (int64_t k = left + (int64_t)g * kPartThreads + tid; k < a.num_pages; k += (int64_t)a.ranges * kPartThreads)
        a.ring_out[k] = -1;
    if (g == 0 && tid == 0) {
        a.state_out[0] = 0;
        a.state_out[1] = left;
        *a.cut = cut;
    }
}

// An entry a thread: its loads wait on one another (a wave a row 7.4 us at 256 rows of 512 entries, 3.3 so).
__global__ void __launch_bounds__(256) compact_table_kernel(CompactArgs a) {
    const int cut = *a.cut, runs = (a.max_pages + 255) / 256;
    for (int64_t i = blockIdx.x; i < (int64_t)a.B * runs; i += gridDim.x) {
        const int b = (int)(i / runs), j = (int)(i - (int64_t)b * runs) * 256 + threadIdx.x;
        compact_row(a, b, j, min(a.max_pages, j + 1), 1, cut, [&](int p) { return a.copies[2 * a.to[p] + 1]; });
    }
}

// A pool that a workgroup holds: all of it here, the moves in LDS.
template <int W>
__global__ void __launch_bounds__(64 * W) compact_one_kernel(CompactArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t words[64 * W * kPer];
    __shared__ int waves[W], cut_at[2], holes[64 * W * kPer / 2];
    const int tid = threadIdx.x;
    compact_words<W>(a, words);
    const Words<kPer> own = own_words<kPer>(words);
    int2 all;
    const int2 front = in_front<W>(own, make_int2(0, 0), waves, &all);
    const int U = all.x, left = all.y;
    if (tid == 0 && left == 0) {
        cut_at[0] = a.num_pages;
        cut_at[1] = U;
    }
    int p, held;
    if (compact_cut(U, tid * kPer, own, front, &p, &held)) {
        cut_at[0] = p;
        cut_at[1] = held;
    }
    __syncthreads();
    const int cut = cut_at[0], used_below = cut_at[1];
    // a page that moves keeps its move's number in its word, above the two bits
    compact_emit(a, U, tid * kPer, own, front, used_below,
                 [&](int p, int k) { words[p] |= (uint32_t)k << 2; a.copies[2 * k] = p; },
                 [&](int p, int k) { holes[k] = p; a.copies[2 * k + 1] = p; });
    for (int k = U - used_below + tid; k < a.room; k += 64 * W) a.copies[2 * k] = a.copies[2 * k + 1] = -1;
    for (int k = left + tid; k < a.num_pages; k += 64 * W) a.ring_out[k] = -1;
    if (tid == 0) {
        a.state_out[0] = 0;
        a.state_out[1] = left;
    }
    __syncthreads();
    for (int b = tid >> 6; b < a.B; b += W)
        compact_row(a, b, tid & 63, a.max_pages, 64, cut, [&](int q) { return holes[words[q] >> 2]; });
}

// ---- copies ---------------------------------------------------------------------------------
// Workgroup (x, y) copies pairs [x per, (x + 1) per), and so on a grid further, in part y, a layer of a pool.  Bound by the bytes: 460 MB read
// and written 102 us, 4.5 TB/s, 113 MB 24.8 us (a large copy 4.7 TB/s).
constexpr int kCopyThreads = 256;

struct CopyArgs {
    const int* copies;       // [n][2] {source, destination}
    int64_t n;
    int num_pages, per, pools;
    int first[kMaxPools + 1];    // part that a pool begins with
    uint8_t* data[kMaxPools];
    int64_t page_bytes[kMaxPools], layer_bytes[kMaxPools];
    int width[kMaxPools];    // bytes a lane: 16, 4 or 1
};

template <typename T>
__device__ __forceinline__ void copy_page(uint8_t* dst, const uint8_t* src, int64_t bytes) {
    const int64_t n = bytes / (int64_t)sizeof(T);
    const T* s = reinterpret_cast<const T*>(src);
    T* d = reinterpret_cast<T*>(dst);
    constexpr int kRun = 8;
    for (int64_t i = threadIdx.x; i < n; i += kRun * kCopyThreads) {
        T x[kRun];
        #pragma unroll
        for (int k = 0; k < kRun; ++k) x[k] = s[min(i + k * kCopyThreads, n - 1)];
        #pragma unroll
        for (int k = 0; k < kRun; ++k)
            if (i + k * kCopyThreads < n) d[i + k * kCopyThreads] = x[k];
    }
}

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(CopyArgs a) {
    int pool = 0;
    while (pool + 1 < a.pools && (int)blockIdx.y >= a.first[pool + 1]) ++pool;
    uint8_t* base = a.data[pool] + ((int)blockIdx.y - a.first[pool]) * a.layer_bytes[pool];
    const int64_t bytes = a.page_bytes[pool];
    const int lane = threadIdx.x & 63;
    for (int64_t i0 = (int64_t)blockIdx.x * a.per; i0 < a.n; i0 += (int64_t)gridDim.x * a.per) {
        // up to 64 pairs, a lane each; the same in every wave
        const int64_t i = i0 + lane;
        int2 mine = make_int2(-1, -1);
        if (lane < a.per && i < a.n) mine = reinterpret_cast<const int2*>(a.copies)[i];
        const bool in = mine.x >= 0 && mine.x < a.num_pages && mine.y >= 0 && mine.y < a.num_pages && mine.x != mine.y;
        uint64_t todo = __builtin_amdgcn_ballot_w64(in);
        while (todo) {
            const int k = __builtin_ctzll(todo);
            todo &= todo - 1;
            const uint8_t* src = base + (int64_t)__builtin_amdgcn_readlane(mine.x, k) * bytes;
            uint8_t* dst = base + (int64_t)__builtin_amdgcn_readlane(mine.y, k) * bytes;
            if (a.width[pool] == 16) copy_page<v4u_t>(dst, src, bytes);
            else if (a.width[pool] == 4) copy_page<uint32_t>(dst, src, bytes);
            else copy_page<uint8_t>(dst, src, bytes);
        }
    }
}

int parts_of(int num_pages) { return (int)(((int64_t)num_pages + kPart - 1) / kPart); }
bool fork_in_one(int B, int num_pages) { return B <= kThreads && num_pages <= kRange; }

}  // namespace

size_t cache_fork_workspace(int B, int num_pages) {
    if (fork_in_one(B, num_pages)) return 0;
    return (size_t)parts_of(num_pages) * (kPart + 1) * 4;
}

hipError_t launch_cache_fork(const CacheFork& p, void* workspace, hipStream_t stream) {
    ForkArgs a;
    a.parents = p.parents; a.keep = p.keep_lens; a.lens = p.seq_lens; a.table = p.block_table;
    a.state = p.free_state; a.ring = p.free_pages;
    a.lens_out = p.seq_lens_out; a.table_out = p.block_table_out; a.state_out = p.free_state_out;
    a.copies = p.copies;
    a.parts = parts_of(p.num_pages);
    a.words = static_cast<uint32_t*>(workspace);
    a.freed = static_cast<int*>(workspace) + (size_t)a.parts * kPart;
    a.B = p.B; a.page = p.page_size; a.max_pages = p.max_pages; a.num_pages = p.num_pages;
    if (fork_in_one(p.B, p.num_pages)) {
        if (p.B <= kPartThreads && p.num_pages <= kSmall)
            hipLaunchKernelGGL(fork_one_kernel<kPartWaves>, dim3(1), dim3(kPartThreads), 0, stream, a);
        else
            hipLaunchKernelGGL(fork_one_kernel<kWaves>, dim3(1), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    const hipError_t e = clear_pages(workspace, (int64_t)a.parts * kPart * 4, stream);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(fork_mark_kernel, dim3((unsigned)std::min((p.B + 3) / 4, 8 * kNumCUs)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(fork_freed_kernel, dim3((unsigned)a.parts), dim3(kPartThreads), 0, stream, a);
    hipLaunchKernelGGL(fork_emit_kernel, dim3((unsigned)(a.parts + (p.B + kPartWaves - 1) / kPartWaves)), dim3(kPartThreads),
                       0, stream, a);
    return hipGetLastError();
}

size_t cache_compact_workspace(int num_pages) {
    if (num_pages <= kRange) return 0;
    const size_t parts = parts_of(num_pages);
    return 2 * parts * kPart + parts * 8 + (size_t)num_pages * 4 + 4;
}

hipError_t launch_cache_compact(const CacheCompact& p, void* workspace, hipStream_t stream) {
    CompactArgs a;
    a.lens = p.seq_lens; a.table = p.block_table; a.ring = p.free_pages; a.state = p.free_state;
    a.table_out = p.block_table_out; a.ring_out = p.free_pages_out; a.state_out = p.free_state_out;
    a.copies = p.copies;
    a.B = p.B; a.page = p.page_size; a.max_pages = p.max_pages; a.num_pages = p.num_pages;
    a.room = std::max(1, p.num_pages / 2);
    a.ranges = parts_of(p.num_pages);
    const size_t bytes = (size_t)a.ranges * kPart;
    a.used = static_cast<uint8_t*>(workspace);
    a.free = a.used + bytes;
    a.sums = reinterpret_cast<int2*>(a.free + bytes);
    a.to = reinterpret_cast<int*>(a.sums + a.ranges);
    a.cut = a.to + p.num_pages;
    if (p.num_pages <= kRange) {
        if (p.num_pages <= kSmall) hipLaunchKernelGGL(compact_one_kernel<kPartWaves>, dim3(1), dim3(kPartThreads), 0, stream, a);
        else hipLaunchKernelGGL(compact_one_kernel<kWaves>, dim3(1), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    const unsigned rows = (unsigned)std::min((p.B + 3) / 4, 8 * kNumCUs);
    const unsigned ring = (unsigned)std::min<int64_t>(((int64_t)p.num_pages + 1023) / 1024, 8 * kNumCUs);
    const hipError_t e = clear_pages(workspace, 2 * (int64_t)bytes, stream);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(compact_mark_kernel, dim3(std::max(rows, ring)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(compact_sums_kernel, dim3((unsigned)a.ranges), dim3(kPartThreads), 0, stream, a);
    hipLaunchKernelGGL(compact_emit_kernel, dim3((unsigned)a.ranges), dim3(kPartThreads), 0, stream, a);
    const int64_t runs = (int64_t)p.B * ((p.max_pages + 255) / 256);
    hipLaunchKernelGGL(compact_table_kernel, dim3((unsigned)std::min<int64_t>(runs, 8 * kNumCUs)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_copy_pages(const CopyPages& p, hipStream_t stream) {
    if (p.n <= 0) return hipSuccess;
    CopyArgs a;
    a.copies = p.copies; a.n = p.n; a.num_pages = p.num_pages; a.pools = p.pools;
    int parts = 0;
    for (int i = 0; i < p.pools; ++i) {
        a.first[i] = parts;
        parts += p.pool[i].layers;
        a.data[i] = static_cast<uint8_t*>(p.pool[i].data);
        a.page_bytes[i] = p.pool[i].page_bytes;
        a.layer_bytes[i] = p.pool[i].layer_bytes;
        const uint64_t low = reinterpret_cast<uintptr_t>(p.pool[i].data) | (uint64_t)a.page_bytes[i] |
                             (p.pool[i].layers > 1 ? (uint64_t)a.layer_bytes[i] : 0);
        a.width[i] = low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : 1;
    }
    a.first[p.pools] = parts;
    // about 4,096 workgroups: of a long list, whose places may be empty, each takes several pairs
    int per = 1;
    while (per < 64 && p.n * parts / per > 4096) per *= 2;
    a.per = per;
    const int64_t groups = std::min<int64_t>((p.n + per - 1) / per, 1 << 20);   // (2^32 threads would be none)
    if (parts > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)groups, (unsigned)parts), dim3(kCopyThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
