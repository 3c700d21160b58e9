// The paged cache in 8 bits with a power-of-two scale for each block of tokens: block tables,
// positions and slots from request lengths (extend), the append that writes it and the reader
// of its rows.  Attention over it is flash16x8_kernel (flash.hip).
//
// Format: pools of pages of page_size rows, e4m3 codes [num_pages, page_size, 512] (latent) and
// [num_pages, page_size, 64] (rope key), and E8M0 scale bytes [num_pages, page_size / G, 2], one
// for each block of G tokens and each part: value = code * 2^(byte - 127).  The two parts have a
// scale each because a latent row is RMS-normalised and a rope key is not.  Powers of two cost an
// e4m3 code no precision (it has an exponent of its own), and they let a block whose scale grows
// be coded again without error but for values that become subnormal.

#include "common.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace mla {

namespace {

typedef uint32_t v2u_t __attribute__((ext_vector_type(2)));
typedef float v2f_t __attribute__((ext_vector_type(2)));

// Inclusive sum over the lanes up to this one, and the wave's maximum (of values >= 0).
__device__ __forceinline__ int lanes_sum_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ int lanes_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

// ---- extend ---------------------------------------------------------------------------------
// Request b holds L = seq_lens[b] tokens and asks for new_lens[b] more (or fewer).  What it needs,
// pages(L + n) - pages(L), is summed over the requests in order, and a request is granted while
// the running sum stays within the free pages; the same sums place its pages in the ring of free
// ones.  So the whole plan is two prefix sums over the requests (pages asked for, pages given
// back), made by one workgroup; then every table entry, ring entry, position and slot follows from
// its request's four numbers {L, granted, first page taken, first page given back} alone, in any
// order: taken pages come from the ring's free ones and given ones go to places that hold none, and
// a new token's page is an old table entry or a free one, so nothing written here is read here.
// It is bound by latency: a decode step of 128 requests takes 6.2 us, its tables a few KB; 32 requests of
// up to 4,096 new tokens 3.2 + 4.7 (2.1 MB of positions and slots), 256 of up to 60,000 tokens, some of them
// ending, 11.4 (33 with a page a thread in turn and divisions by the compiler).
constexpr int kExtendThreads = 1024;   // at most
constexpr int kExtendWaves = kExtendThreads / 64;

// x / d for 0 <= x < 2^31 and a d that the host knows (a division takes forty instructions, and each
// request's plan has five), by the method of Granlund and Montgomery (1994): with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// x / d = (floor(m x / 2^32) + x) / 2^s, where the sum stays below 2^32.
struct FastDiv {
    uint32_t d, m;
    int s;
    static FastDiv of(uint32_t d) {
        int s = 0;
        while ((1ull << s) < d) ++s;
        return {d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return (__umulhi(m, x) + x) >> s; }
    __device__ __forceinline__ uint32_t mod(uint32_t x) const { return x - div(x) * d; }
};

struct ExtendArgs {
    int B, Sq, page_size, max_pages, num_pages;
    FastDiv by_page, by_sq;
    const int* new_lens;
    const int* seq_lens;
    const int* free_state;   // {head, count}
    int* table;
    int* ring;
    int* lens_out;
    int* state_out;
    int* granted;
    int64_t* positions;
    int64_t* slots;
    int4* info;              // [B + 1]: the requests' four numbers, then {head, count, long runs, 0}
};

__device__ __forceinline__ int extend_pages(const ExtendArgs& a, int tokens) {
    const uint32_t q = a.by_page.div((uint32_t)tokens);
    return (int)(q + (q * a.by_page.d != (uint32_t)tokens));
}
// Place `at` places past the ring's head (at < 2 num_pages <= 2^31).
__device__ __forceinline__ int ring_place(const ExtendArgs& a, int head, int at) {
    uint32_t p = (uint32_t)head + (uint32_t)at;
    if (p >= (uint32_t)a.num_pages) p -= (uint32_t)a.num_pages;
    return (int)(p >= (uint32_t)a.num_pages ? p - (uint32_t)a.num_pages : p);
}

// The part that follows from `info` (in LDS or memory), by `threads` threads of which this is number
// `t`: a thread for each request's first page in or out, a wave for the pages behind it where a
// request has any (`runs`), a thread for each position.
__device__ __forceinline__ void extend_fill(const ExtendArgs& a, const int4* info, int head, int count,
                                            int runs, int t, int threads) {
    // pages k0, k0 + step, .. of request b's move, kRun of them together: free pages into the table, or
    // table entries to the ring, as far as there are places behind the tail (else they are in the ring)
    auto move = [&](int b, int k0, int step, auto run) __attribute__((always_inline)) {
        constexpr int kRun = decltype(run)::value;
        const int4 r = info[b];
        const int have = extend_pages(a, r.x), end = extend_pages(a, r.x + r.y);
        int* row = a.table + (int64_t)b * a.max_pages;
        const bool in = have < end;
        const int n = in ? end - have : min(have - end, a.num_pages - count - r.w);
        const int from = in ? r.z : count + r.w;   // past the ring's head
        row += in ? have : end;
        for (int k = k0; k < n; k += kRun * step) {
            int page[kRun];
            #pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const int m = min(k + i * step, n - 1);
                page[i] = in ? a.ring[ring_place(a, head, from + m)] : row[m];
            }
            #pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const int m = k + i * step;
                if (m < n) (in ? row[m] : a.ring[ring_place(a, head, from + m)]) = page[i];
            }
            if (step == 0) break;
        }
    };
    for (int b = t; b < a.B; b += threads) move(b, 0, 0, std::integral_constant<int, 1>{});
    if (runs)
        for (int b = t >> 6; b < a.B; b += threads >> 6)
            move(b, 1 + (t & 63), 64, std::integral_constant<int, 4>{});
    const int total = a.B * a.Sq;
    for (int i = t; i < total; i += threads) {
        const int b = (int)a.by_sq.div((uint32_t)i), s = i - b * a.Sq;
        const int4 r = info[b];
        int64_t pos = -1, slot = -1;
        if (s >= a.Sq - r.y) {
            const int p = r.x + r.y - a.Sq + s, j = (int)a.by_page.div((uint32_t)p), have = extend_pages(a, r.x);
            const int page = j < have ? a.table[(int64_t)b * a.max_pages + j]
                                      : a.ring[ring_place(a, head, r.z + j - have)];
            pos = p;
            slot = (int64_t)page * a.page_size + (p - j * a.page_size);
        }
        a.positions[i] = pos;
        a.slots[i] = slot;
    }
}

// ONE: `info` stays in LDS (B <= kExtendThreads) and this workgroup does the rest too.
template <bool ONE>
__global__ void __launch_bounds__(kExtendThreads) cache_extend_kernel(ExtendArgs a) {
    __shared__ int w_ask[kExtendWaves], w_back[kExtendWaves], w_take[kExtendWaves], w_runs[kExtendWaves];
    __shared__ int4 info_lds[ONE ? kExtendThreads : 1];
    int4* info = ONE ? info_lds : a.info;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int threads = blockDim.x, waves = threads >> 6;
    const int N = a.num_pages, span = a.max_pages * a.page_size;
    const int per = (a.B + threads - 1) / threads;   // ONE: 1
    const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    // pages asked for by a request that its own limits allow, and given back by one that shrinks
    struct Plan { int L, n, ask, back; };
    auto plan = [&](int b) __attribute__((always_inline)) {
        Plan p = {min(max(a.seq_lens[b], 0), span), a.new_lens[b], 0, 0};
        const int have = extend_pages(a, p.L);
        if (p.n > 0) {
            if (p.n > a.Sq || p.n > span - p.L) p.n = 0;
            else p.ask = extend_pages(a, p.L + p.n) - have;
        } else {
            p.n = max(p.n, -p.L);
            p.back = have - extend_pages(a, p.L + p.n);
        }
        return p;
    };
    const int head_in = a.free_state[0], count_in = a.free_state[1];
    Plan own = {0, 0, 0, 0};   // of request b0, where the thread has one alone
    int ask = 0, back = 0;
    for (int b = b0; b < b1; ++b) {
        own = plan(b);
        ask += own.ask;
        back += own.back;
    }
    const int ia = lanes_sum_scan(ask), ib = lanes_sum_scan(back);
    if (lane == 63) { w_ask[wave] = ia; w_back[wave] = ib; }
    __syncthreads();
    int head = head_in % N;
    if (head < 0) head += N;
    const int count = min(max(count_in, 0), N);
    int asked = ia - ask, pushed = ib - back, all_back = 0;
    for (int w = 0; w < waves; ++w) {
        if (w < wave) { asked += w_ask[w]; pushed += w_back[w]; }
        all_back += w_back[w];
    }
    int taken = 0;   // pages taken by the requests up to this thread's last granted one
    bool runs = false;
    for (int b = b0; b < b1; ++b) {
        Plan p = per == 1 ? own : plan(b);
        const int first = asked;
        asked += p.ask;
        if (p.ask > 0) {
            if (asked <= count) taken = asked;
            else p.n = 0;
        }
        runs |= max(p.ask, p.back) > 1;
        info[b] = make_int4(p.L, p.n, first, pushed);
        pushed += p.back;
        a.lens_out[b] = p.L + p.n;
        a.granted[b] = p.n;
    }
    const int most = lanes_max(taken);
    const int any = __builtin_amdgcn_ballot_w64(runs) != 0;
    if (lane == 0) { w_take[wave] = most; w_runs[wave] = any; }
    __syncthreads();
    int all_runs = 0;
    for (int w = 0; w < waves; ++w) {
        taken = max(taken, w_take[w]);
        all_runs |= w_runs[w];
    }
    if (tid == 0) {
        a.state_out[0] = ring_place(a, head, taken);
        a.state_out[1] = count - taken + min(all_back, N - count);
        if (!ONE) info[a.B] = make_int4(head, count, all_runs, 0);
    }
    if (ONE) extend_fill(a, info, head, count, all_runs, tid, threads);
}

__global__ void __launch_bounds__(256) cache_extend_fill_kernel(ExtendArgs a) {
    const int4 s = a.info[a.B];
    extend_fill(a, a.info, s.x, s.y, s.z, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- append ---------------------------------------------------------------------------------
// A workgroup owns one block of G tokens of one sequence: it forms the block's new rows from the
// product x @ W_kv_a (or its split-K partials), takes the largest magnitude of each part over
// them, and codes them.  Nothing of a block is shared between workgroups, so the scale needs no
// atomics and the result no order.  A wave makes a row at a time (8 latent columns and, in the
// lower half, one rope pair a lane: the norm is a wave reduction) and keeps up to four across the
// barrier that the block's maxima need.  Few new rows leave waves over: those share the rows' splits
// (up to 16 of them, whose loads a wave alone would wait for four times), the sums in wave order.
// Bound by latency in decode (128 rows in 13 splits 5.7 us), by the partials' bytes in
// prefill (4,096 rows in 3 splits, 28 MB, 14 us: 2 TB/s, a row's loads waiting on one another).
//   scale: 2^e with the smallest e >= -100 such that every finite magnitude is <= 448 * 2^e (448,
//     e4m3's largest value, is 1.75 * 2^8: e from the exponent and one comparison); where the block
//     keeps rows written before, at least the scale that they have.  If that grew, they are
//     coded again: code * 2^(e_old - e), exact but for values that become subnormal.
//   codes: v * 2^-e rounded once, to nearest even, from the fp32 row; a value that is not finite
//     becomes the NaN code and has no part in the scale.
struct AppendBlkArgs {
    const float* in;         // [nsplit][B*Sq][576], split_stride floats apart
    int nsplit;
    int64_t split_stride;
    const void* gain;
    const float* inv_freq;
    const int* seq_lens;     // after the append
    const int* new_lens;
    const int* table;
    uint8_t* c_kv;
    uint8_t* pe;
    uint8_t* scales;
    int B, Sq, page_size, max_pages, num_pages, blocks;
    float eps;
};

constexpr int kA8R = 512, kA8D = 64, kA8Row = kA8R + kA8D;
constexpr int kA8Waves = 16, kA8Threads = 64 * kA8Waves;
constexpr int kScaleMin = 127 - 100;

__device__ __forceinline__ float finite_abs(float v) {
    const float m = fabsf(v);
    return m < INFINITY ? m : 0.f;
}
// the E8M0 byte of the smallest scale that holds magnitudes up to amax (finite, >= 0)
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t u = __float_as_uint(amax);
    return max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u), kScaleMin);
}
__device__ __forceinline__ float scale_value(int byte) { return __uint_as_float((uint32_t)byte << 23); }
// 1 / scale_value(byte) for bytes 1 .. 254 (the last one's, 2^-127, is subnormal)
__device__ __forceinline__ float scale_inverse(int byte) {
    return __uint_as_float(byte < 254 ? (uint32_t)(254 - byte) << 23 : 0x00400000u);
}
__device__ __forceinline__ float code_input(float v, float inv) {
    return fabsf(v) < INFINITY ? v * inv : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// four codes to the values that they have under `scale`, a power of two
__device__ __forceinline__ v4f decode4(uint32_t w, float scale) {
    const v2f_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    const v2f_t hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
    return v4f{lo[0], lo[1], hi[0], hi[1]};
}

// A row's product as a wave holds it: latent columns 8 lane .. +7, and rope pair lane % 32.
struct RowSums { v4f a, b; v2f_t r; };

// The sum of splits i0, i0 + step, .. of the row at `row`.
__device__ __forceinline__ RowSums sum_splits(const float* row, int nsplit, int64_t split_stride, int i0,
                                              int step) {
    const int lane = threadIdx.x & 63;
    const float* lp = row + 8 * lane;
    const float* rp = row + kA8R + 2 * (lane & 31);
    RowSums s = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}, v2f_t{0.f, 0.f}};
    constexpr int kWin = 4;   // splits' loads in flight
    for (int i = i0; i < nsplit; i += kWin * step) {
        v4f x0[kWin], x1[kWin];
        v2f_t xr[kWin];
        #pragma unroll
        for (int k = 0; k < kWin; ++k) {
            const int64_t o = (int64_t)min(i + k * step, nsplit - 1) * split_stride;
            x0[k] = *reinterpret_cast<const v4f*>(lp + o);
            x1[k] = *reinterpret_cast<const v4f*>(lp + o + 4);
            xr[k] = *reinterpret_cast<const v2f_t*>(rp + o);
        }
        #pragma unroll
        for (int k = 0; k < kWin; ++k)
            if (i + k * step < nsplit) { s.a += x0[k]; s.b += x1[k]; s.r += xr[k]; }
    }
    return s;
}
// The same through LDS, for the waves after this one to add to theirs.
__device__ __forceinline__ void store_sums(float* part, const RowSums& s) {
    const int lane = threadIdx.x & 63;
    *reinterpret_cast<v4f*>(part + 8 * lane) = s.a;
    *reinterpret_cast<v4f*>(part + 8 * lane + 4) = s.b;
    if (lane < 32) *reinterpret_cast<v2f_t*>(part + kA8R + 2 * lane) = s.r;
}
__device__ __forceinline__ void add_sums(RowSums* s, const float* part) {
    const int lane = threadIdx.x & 63;
    s->a += *reinterpret_cast<const v4f*>(part + 8 * lane);
    s->b += *reinterpret_cast<const v4f*>(part + 8 * lane + 4);
    s->r += *reinterpret_cast<const v2f_t*>(part + kA8R + 2 * (lane & 31));
}

template <int OUT>
__device__ __forceinline__ void load_gain(const void* gain, float (&g)[8]) {
    const int lane = threadIdx.x & 63;
    #pragma unroll
    for (int k = 0; k < 8; ++k) {
        if constexpr (OUT == kOutF32) g[k] = static_cast<const float*>(gain)[8 * lane + k];
        else g[k] = Store16<OUT>::to_f32(static_cast<const uint16_t*>(gain)[8 * lane + k]);
    }
}
// The cache row of the product `s` at position pos: normalised latent, rotated rope pair.
__device__ __forceinline__ void make_row(const RowSums& s, const float (&gain)[8], float eps, int pos,
                                         float freq, float* lat, float* rot) {
    float ss = 0.f;
    #pragma unroll
    for (int k = 0; k < 4; ++k) ss += s.a[k] * s.a[k] + s.b[k] * s.b[k];
    const float inv = rsqrtf(wave_reduce(ss, OpSum()) / (float)kA8R + eps);
    #pragma unroll
    for (int k = 0; k < 8; ++k) lat[k] = (k < 4 ? s.a[k] : s.b[k - 4]) * inv * gain[k];
    float c, sn;
    rope_cos_sin(rope_angle(pos, freq), &c, &sn);
    rot[0] = rope_even(s.r[0], s.r[1], c, sn);
    rot[1] = rope_odd(s.r[0], s.r[1], c, sn);
}

// The rows alone, into the place of the first split: where many rows of a block come in many splits,
// one CU per block would read them all (64 rows in 16 splits: 2.4 MB, 30 us); a workgroup per row
// spreads that over the chip, and the blocks then read a row once.  Its four waves share the splits.
template <int OUT>
__global__ void __launch_bounds__(256) kv_rows_kernel(AppendBlkArgs a) {
    __shared__ float part[4][kA8Row];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.Sq, i = blockIdx.x % a.Sq;
    const int L = min(max(a.seq_lens[b], 0), a.max_pages * a.page_size);
    const int n = min(max(a.new_lens[b], 0), min(a.Sq, L));
    if (i < a.Sq - n) return;   // padding
    float* row = const_cast<float*>(a.in) + (int64_t)blockIdx.x * kA8Row;
    float gain[8];
    load_gain<OUT>(a.gain, gain);
    const float freq = a.inv_freq[lane & 31];
    RowSums s = sum_splits(row, a.nsplit, a.split_stride, wave, 4);
    store_sums(part[wave], s);
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; ++w) add_sums(&s, part[w]);
    float lat[8], rot[2];
    make_row(s, gain, a.eps, L - a.Sq + i, freq, lat, rot);
    store_sums(row, RowSums{v4f{lat[0], lat[1], lat[2], lat[3]}, v4f{lat[4], lat[5], lat[6], lat[7]},
                            v2f_t{rot[0], rot[1]}});
}

// READY: `in` holds the rows themselves (kv_rows_kernel's).
template <int OUT, int G, bool READY>
__global__ void __launch_bounds__(kA8Threads) kv_append_blk_kernel(AppendBlkArgs a) {
    constexpr int kRows = G / kA8Waves;   // rows a wave
    __shared__ float red[2][kA8Waves];
    __shared__ float part[kA8Waves][kA8Row];   // a team's sums
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.blocks, t = blockIdx.x % a.blocks;
    const int L = min(max(a.seq_lens[b], 0), a.max_pages * a.page_size);
    const int n = min(max(a.new_lens[b], 0), min(a.Sq, L));
    const int first = L - n, p0 = (first / G + t) * G;
    if (n == 0 || p0 >= L) return;
    const int page = a.table[(int64_t)b * a.max_pages + p0 / a.page_size];
    float gain[8], freq = 0.f;
    if constexpr (!READY) {
        load_gain<OUT>(a.gain, gain);
        freq = a.inv_freq[lane & 31];
    }

    // new rows lo .. hi-1 of the block: with as many waves as rows or fewer, wave w makes rows
    // w, w + 16, ..; with more, a team of waves shares a row's splits and its first wave goes on
    const int lo = max(first - p0, 0), hi = min(L - p0, G);
    int team = 1;
    while (2 * team * (hi - lo) <= kA8Waves) team *= 2;
    if (READY || a.nsplit <= 4) team = 1;   // one wave's loads at once
    auto row_of = [&](int q) __attribute__((always_inline)) {   // -1: none
        const int r = team > 1 ? (q ? G : lo + wave / team) : wave + kA8Waves * q;
        return r >= lo && r < hi ? r : -1;
    };
    auto in_row = [&](int r) __attribute__((always_inline)) {
        return a.in + ((int64_t)b * a.Sq + (p0 + r - L + a.Sq)) * kA8Row;
    };
    RowSums shared_row;
    if (team > 1) {
        const int r = row_of(0);
        if (r >= 0) {
            shared_row = sum_splits(in_row(r), a.nsplit, a.split_stride, wave % team, team);
            store_sums(part[wave], shared_row);
        }
        __syncthreads();
        if (r >= 0 && wave % team == 0)
            for (int w = wave + 1; w < wave + team; ++w) add_sums(&shared_row, part[w]);
    }
    const bool mine = team == 1 || wave % team == 0;
    float lat[kRows][8], rot[kRows][2];
    float top = 0.f, top_r = 0.f;
    #pragma unroll
    for (int q = 0; q < kRows; ++q) {
        const int r = row_of(q);
        if (r < 0 || !mine) continue;   // wave-uniform
        const RowSums s = team > 1 ? shared_row : sum_splits(in_row(r), READY ? 1 : a.nsplit, a.split_stride, 0, 1);
        if constexpr (READY) {
            #pragma unroll
            for (int k = 0; k < 8; ++k) lat[q][k] = k < 4 ? s.a[k] : s.b[k - 4];
            rot[q][0] = s.r[0];
            rot[q][1] = s.r[1];
        } else {
            make_row(s, gain, a.eps, p0 + r, freq, lat[q], rot[q]);
        }
        #pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, finite_abs(lat[q][k]));
        top_r = fmaxf(top_r, fmaxf(finite_abs(rot[q][0]), finite_abs(rot[q][1])));
    }
    if (page < 0 || page >= a.num_pages) return;   // not a page of the pool: skipped
    const int64_t row0 = (int64_t)page * a.page_size + p0 % a.page_size;
    uint8_t* sc = a.scales + 2 * (row0 / G);
    int old[2] = {0, 0};
    if (lo > 0) { old[0] = sc[0]; old[1] = sc[1]; }
    top = wave_reduce(top, OpMax());
    top_r = wave_reduce(top_r, OpMax());
    if (lane == 0) { red[0][wave] = top; red[1][wave] = top_r; }
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kA8Waves; ++w) {
        top = fmaxf(top, red[0][w]);
        top_r = fmaxf(top_r, red[1][w]);
    }
    const int e_lat = max(scale_byte(top), old[0]), e_rot = max(scale_byte(top_r), old[1]);
    if (threadIdx.x == 0) { sc[0] = (uint8_t)e_lat; sc[1] = (uint8_t)e_rot; }
    const float inv_l = scale_inverse(e_lat), inv_r = scale_inverse(e_rot);
    auto at_lat = [&](int r) __attribute__((always_inline)) { return a.c_kv + (row0 + r) * kA8R + 8 * lane; };
    auto at_rot = [&](int r) __attribute__((always_inline)) { return a.pe + (row0 + r) * kA8D + 2 * (lane & 31); };
    #pragma unroll
    for (int q = 0; q < kRows; ++q) {
        const int r = row_of(q);
        if (r < 0 || !mine) continue;
        auto in = [&](int k) __attribute__((always_inline)) { return code_input(lat[q][k], inv_l); };
        *reinterpret_cast<v2u_t*>(at_lat(r)) =
            v2u_t{code4(in(0), in(1), in(2), in(3)), code4(in(4), in(5), in(6), in(7))};
        if (lane < 32)
            *reinterpret_cast<uint16_t*>(at_rot(r)) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(
                code_input(rot[q][0], inv_r), code_input(rot[q][1], inv_r), 0, false);
    }
    // rows of before, where the scale grew: times 2^(e_old - e), at least 2^-100 (which leaves nothing)
    if (lo > 0 && e_lat != old[0]) {
        const float f = scale_value(127 - min(e_lat - old[0], 100));
        for (int r = wave; r < lo; r += kA8Waves) {
            const v2u_t w = *reinterpret_cast<const v2u_t*>(at_lat(r));
            const v4f x = decode4(w[0], f), y = decode4(w[1], f);
            *reinterpret_cast<v2u_t*>(at_lat(r)) =
                v2u_t{code4(x[0], x[1], x[2], x[3]), code4(y[0], y[1], y[2], y[3])};
        }
    }
    if (lo > 0 && e_rot != old[1] && lane < 32) {
        const float f = scale_value(127 - min(e_rot - old[1], 100));
        for (int r = wave; r < lo; r += kA8Waves) {
            const v2f_t x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(
                (uint32_t)*reinterpret_cast<const uint16_t*>(at_rot(r)), f, false);
            *reinterpret_cast<uint16_t*>(at_rot(r)) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        }
    }
}

// ---- read -----------------------------------------------------------------------------------
// Rows by slot, decoded: a wave takes four rows at a time (their 8 codes a lane, then the rope
// codes of all four by 16 lanes each), all loads before the first store.  Bound by the bytes: 58,415 rows
// to bf16 17.6 us, 101 MB at 5.8 TB/s (in part from the last-level cache); 4,989 rows 4.3 us, of which most
// is the launch.
struct ReadBlkArgs {
    const int64_t* slots;
    int64_t n, rows;         // slots asked for; rows of the pool
    const uint8_t* c_kv;
    const uint8_t* pe;
    const uint8_t* scales;
    void* lat;               // [n, 512]
    void* rot;               // [n, 64]
    int block_shift;         // log2 of the tokens a block
};

template <int OUT>
__device__ __forceinline__ void store4(void* dst, int64_t at, v4f v) {
    if constexpr (OUT == kOutF32)
        *reinterpret_cast<v4f*>(static_cast<float*>(dst) + at) = v;
    else
        *reinterpret_cast<v2u_t*>(static_cast<uint16_t*>(dst) + at) =
            v2u_t{Store16<OUT>::pack2(v[0], v[1]), Store16<OUT>::pack2(v[2], v[3])};
}

template <int OUT>
__global__ void __launch_bounds__(256) kv_read_blk_kernel(ReadBlkArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * 4;
    for (int64_t r0 = 4 * ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)); r0 < a.n; r0 += 4 * waves) {
        v2u_t c[4];
        float f[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t s = r0 + i < a.n ? a.slots[r0 + i] : -1;
            const bool in = s >= 0 && s < a.rows;
            c[i] = in ? reinterpret_cast<const v2u_t*>(a.c_kv + s * kA8R)[lane] : v2u_t{0, 0};
            f[i] = in ? scale_value(a.scales[2 * (s >> a.block_shift)]) : 1.f;
        }
        const int64_t rr = r0 + (lane >> 4);
        const int64_t s = rr < a.n ? a.slots[rr] : -1;
        const bool in = s >= 0 && s < a.rows;
        const uint32_t p = in ? reinterpret_cast<const uint32_t*>(a.pe + s * kA8D)[lane & 15] : 0;
        const float fp = in ? scale_value(a.scales[2 * (s >> a.block_shift) + 1]) : 1.f;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r0 + i >= a.n) break;
            store4<OUT>(a.lat, (r0 + i) * kA8R + 8 * lane, decode4(c[i][0], f[i]));
            store4<OUT>(a.lat, (r0 + i) * kA8R + 8 * lane + 4, decode4(c[i][1], f[i]));
        }
        if (rr < a.n) store4<OUT>(a.rot, rr * kA8D + 4 * (lane & 15), decode4(p, fp));
    }
}

}  // namespace

// Up to this many positions one workgroup does everything; past it a second, wide launch fills.
constexpr int kExtendOneFill = 8192;

static bool extend_in_one(int B, int Sq) {
    return B <= kExtendThreads && (int64_t)B * Sq <= kExtendOneFill;
}
size_t cache_extend_workspace(int B, int Sq) {
    return extend_in_one(B, Sq) ? 0 : ((size_t)B + 1) * sizeof(int4);
}

hipError_t launch_cache_extend(const CacheExtend& p, void* workspace, hipStream_t stream) {
    ExtendArgs a;
    a.B = p.B; a.Sq = p.Sq; a.page_size = p.page_size; a.max_pages = p.max_pages; a.num_pages = p.num_pages;
    a.new_lens = p.new_lens; a.seq_lens = p.seq_lens; a.free_state = p.free_state;
    a.table = p.block_table; a.ring = p.free_pages;
    a.lens_out = p.seq_lens_out; a.state_out = p.free_state_out; a.granted = p.granted;
    a.positions = p.positions; a.slots = p.slots;
    a.info = static_cast<int4*>(workspace);
    a.by_page = FastDiv::of((uint32_t)p.page_size);
    a.by_sq = FastDiv::of((uint32_t)p.Sq);
    if (extend_in_one(p.B, p.Sq)) {
        // fewer waves, and with them a shorter way through the barriers, where they have work enough
        const int threads = p.B <= 32 && p.B * p.Sq <= 256 ? 256 : kExtendThreads;
        hipLaunchKernelGGL(cache_extend_kernel<true>, dim3(1), dim3(threads), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(cache_extend_kernel<false>, dim3(1), dim3(kExtendThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t wgs = std::max<int64_t>(((int64_t)p.B * p.Sq + 1023) / 1024, (p.B + 3) / 4);
    hipLaunchKernelGGL(cache_extend_fill_kernel, dim3((unsigned)std::min<int64_t>(wgs, 8 * kNumCUs)),
                       dim3(256), 0, stream, a);
    return hipGetLastError();
}

namespace {
template <int OUT, int G>
void launch_append_g(const AppendBlkArgs& a, bool rows_first, hipStream_t stream) {
    const dim3 grid((unsigned)(a.B * a.blocks)), threads(kA8Threads);
    if (!rows_first) {
        hipLaunchKernelGGL((kv_append_blk_kernel<OUT, G, false>), grid, threads, 0, stream, a);
        return;
    }
    hipLaunchKernelGGL(kv_rows_kernel<OUT>, dim3((unsigned)(a.B * a.Sq)), dim3(256), 0, stream, a);
    // the rows are float32 whatever the gain's type
    hipLaunchKernelGGL((kv_append_blk_kernel<kOutF32, G, true>), grid, threads, 0, stream, a);
}
template <int OUT>
hipError_t launch_append_blk(const AppendBlkArgs& a, int block, hipStream_t stream) {
    // Rows in a launch of their own where a block's are many partial rows and each is more than one
    // round of loads (one launch / two, with the product, us: 160 tokens in 16 splits, blocks of 64
    // 49.0 / 24.9; 1,024 in 6, blocks of 64 40.1 / 32.8, of 16 29.6 / 30.7; 16 tokens of 8 sequences
    // in 14 24.3 / 22.0; 4 of 33 21.0 / 21.7; 4,096 in 3, blocks of 64 67.1 / 69.3).
    const bool rows_first = a.nsplit > 4 && std::min(a.Sq, block) * a.nsplit >= 160;
    if (block == 16) launch_append_g<OUT, 16>(a, rows_first, stream);
    else if (block == 32) launch_append_g<OUT, 32>(a, rows_first, stream);
    else launch_append_g<OUT, 64>(a, rows_first, stream);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_kv_append_blk(const KvAppendBlk& p, hipStream_t stream) {
    if ((p.block != 16 && p.block != 32 && p.block != 64) || p.page_size % p.block != 0)
        return hipErrorInvalidValue;
    AppendBlkArgs a;
    a.in = p.in; a.nsplit = p.nsplit; a.split_stride = p.split_stride;
    a.gain = p.gain; a.inv_freq = p.inv_freq; a.seq_lens = p.seq_lens; a.new_lens = p.new_lens;
    a.table = p.block_table;
    a.c_kv = static_cast<uint8_t*>(p.c_kv); a.pe = static_cast<uint8_t*>(p.pe);
    a.scales = static_cast<uint8_t*>(p.scales);
    a.B = p.B; a.Sq = p.Sq; a.page_size = p.page_size; a.max_pages = p.max_pages;
    a.num_pages = p.num_pages; a.eps = p.eps;
    a.blocks = (p.Sq + p.block - 2) / p.block + 1;   // blocks that Sq tokens in a row can touch
    if ((int64_t)a.B * a.blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (p.gain_type == kOutF32) return launch_append_blk<kOutF32>(a, p.block, stream);
    if (p.gain_type == kOutBF16) return launch_append_blk<kOutBF16>(a, p.block, stream);
    return launch_append_blk<kOutF16>(a, p.block, stream);
}

hipError_t launch_kv_read_blk(const KvReadBlk& p, hipStream_t stream) {
    if (p.n <= 0) return hipSuccess;
    ReadBlkArgs a;
    a.slots = p.slots; a.n = p.n; a.rows = p.rows;
    a.c_kv = static_cast<const uint8_t*>(p.c_kv); a.pe = static_cast<const uint8_t*>(p.pe);
    a.scales = static_cast<const uint8_t*>(p.scales);
    a.lat = p.lat; a.rot = p.rot;
    a.block_shift = p.block == 16 ? 4 : p.block == 32 ? 5 : 6;
    const unsigned grid = (unsigned)std::min<int64_t>((p.n + 15) / 16, 16 * kNumCUs);
    if (p.out_type == kOutF32)
        hipLaunchKernelGGL(kv_read_blk_kernel<kOutF32>, dim3(grid), dim3(256), 0, stream, a);
    else if (p.out_type == kOutBF16)
        hipLaunchKernelGGL(kv_read_blk_kernel<kOutBF16>, dim3(grid), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(kv_read_blk_kernel<kOutF16>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace mla
