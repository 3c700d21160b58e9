// Attention in the expanded form, for chunks of many new tokens: every head has keys and values of
// its own, made from the cache's latent rows,
//   k[h] = W_uk[h] c (128),  v[h] = W_uv[h] c (128),
//   out[h] = softmax((q_nope[h] . k[h] + q_rope[h] . pe) / scale) v[h],
// the same function as the absorbed pass (flash.hip) at 2 * 320 operations a pair and head instead of
// 2 * 1,088, for 2 * 256 * 512 a key and head once.  In launches:
//   expand_plan_kernel    which 64-row units of the cache the batch holds, shared pages once
//   expand_gather_kernel  their rows side by side in 16 bits: latent [rows, 512], rope [rows, 64]
//   bgemm_kernel<EXPAND>  the heads' keys and values [heads][rows][128 | 128] (bgemm.hip)
//   heads_kernel          the attention
// the last two for as many heads at a time as the workspace holds.

#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "kernels.h"
#include "mma.h"
#include "stage.h"

namespace mla {

namespace {

typedef uint32_t v2u_t __attribute__((ext_vector_type(2)));
typedef float v2f_t __attribute__((ext_vector_type(2)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

constexpr int kUnit = kExpandUnit;            // rows a unit (and keys a step of the attention)
constexpr int kR = 512, kD = 64, kN = 128;    // latent, rope, nope / value widths
constexpr int kHead = 6;                      // log2 of a bf16 unit's largest value as it is stored
constexpr int kSpread = 12;                   // log2 of how far a row's largest may lie below it
constexpr int kMixed = 4096;                  // added to a mixed unit's exponent

// ---- units ----------------------------------------------------------------------------------
// Unit j of sequence b is its keys [64 j, 64 j + 64).  Sequences that continue one prompt hold the
// same page there; such a unit is expanded once, for the lowest of them (only where it is full in
// both: the rows past a sequence's end are zeros, and the others' are not).  A sequence is only
// compared with those that share its first page, which is what a shared prefix begins with.
struct PlanArgs {
    const int* seq_lens;     // null, with the table: a dense cache, nothing to plan
    const int* table;
    int* owner;      // [B][units] the sequence that the unit is made for
    int* rank;       // [B][units] how many own units it has in front
    int* count;      // [B] own units
    int* order;      // [B] the sequences, longest first
    int* any_bad;
    int B, Sk, units, max_pages, per_page;   // per_page: units a page
};

constexpr int kPlanThreads = 256, kPlanList = 1024;

__global__ void __launch_bounds__(kPlanThreads) expand_plan_kernel(PlanArgs a) {
    __shared__ int list[kPlanList], n_list, w_own[kPlanThreads / 64];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (b == 0 && tid == 0) *a.any_bad = 0;
    if (!a.table) return;
    const int len = min(max(a.seq_lens[b], 0), a.Sk);
    const int* row = a.table + (int64_t)b * a.max_pages;
    // longer sequences, and those as long in front of this one
    int longer = 0;
    for (int c = tid; c < a.B; c += kPlanThreads) {
        const int n = min(max(a.seq_lens[c], 0), a.Sk);
        longer += n > len || (n == len && c < b);
    }
    longer = wave_sum(longer);
    if (lane == 0) w_own[wave] = longer;
    // sequences in front of this one with the same first page, in order
    if (tid == 0) n_list = 0;
    __syncthreads();
    if (tid == 0) a.order[w_own[0] + w_own[1] + w_own[2] + w_own[3]] = b;
    if (len >= kUnit && wave == 0) {
        const int page = row[0];
        int n = 0;
        for (int c0 = 0; c0 < b && n < kPlanList; c0 += 64) {
            const int c = min(c0 + lane, b);
            const bool same = c < b && a.table[(int64_t)c * a.max_pages] == page && a.seq_lens[c] >= kUnit;
            const uint64_t m = __builtin_amdgcn_ballot_w64(same);
            const int at = n + __popcll(m & ((1ull << lane) - 1));
            if (same && at < kPlanList) list[at] = c;
            n += __popcll(m);
        }
        if (lane == 0) n_list = min(n, kPlanList);
    }
    __syncthreads();
    const int units = (len + kUnit - 1) / kUnit;
    int base = 0;
    for (int j0 = 0; j0 < units; j0 += kPlanThreads) {
        const int j = j0 + tid;
        int own = b;
        if (j < units && (j + 1) * kUnit <= len) {
            const int pg = j / a.per_page, page = row[pg];
            for (int i = 0; i < n_list; ++i) {
                const int c = list[i];
                if (a.table[(int64_t)c * a.max_pages + pg] == page && a.seq_lens[c] >= (j + 1) * kUnit) {
                    own = c;
                    break;
                }
            }
        }
        const bool mine = j < units && own == b;
        const uint64_t m = __builtin_amdgcn_ballot_w64(mine);
        if (lane == 0) w_own[wave] = __popcll(m);
        __syncthreads();
        int before = base;
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) before += w_own[w];
            base += w_own[w];
        }
        if (j < units) {
            a.owner[(int64_t)b * a.units + j] = own;
            a.rank[(int64_t)b * a.units + j] = before + __popcll(m & ((1ull << lane) - 1));
        }
        __syncthreads();
    }
    if (tid == 0) a.count[b] = base;
}

// ---- gather ---------------------------------------------------------------------------------
// A workgroup copies a unit's rows, or only notes where its owner's are.  Few units are bound by the way to
// memory and back, many by their bytes: 512 rows 7.1 us, 4,096 9.1, 32,768 16.8 (4.5 TB/s), 13,216 of the 8-bit
// cache 14.4 (with four waves instead of eight and loads behind tests of their own 9.3, 11.5, 19.5 and 22.2); with the
// weights of 128 heads (16 in the third) beside them 10.8, 14.3, 20.0 and 17.6.
// Keys, values and weights are fp16 from here on, in bf16 too: 11 bits instead of 8 bring the outputs'
// distance from the exact ones from 1.6 to 2.3 times that of their own rounding down to about it (bf16).
// A bf16 cache is fitted into fp16's range by a power of two for each unit, 2^e: its rows are stored
// under it, the largest value in [2^kHead, 2^(kHead+1)), and the attention puts it back.  kHead leaves
// 2^9 above for keys and values, sums of 512 products with weights (below 1 they cannot reach fp16's
// end), and 2^20 below down to its subnormals.  Where a latent row (where that is zeros: a rope row) is more than
// 2^kSpread below the largest value the unit is `mixed`: each latent and each rope row has a power of two of its own, so
// that no row, hidden or not, costs another its bits.
// An fp16 cache is as it is (e = 0).  The latent rows keep the type of W_uk and W_uv, which they are
// multiplied with; the rope rows are fp16.
// A latent row with a value that is not finite makes every key and value of it NaN or infinite, and
// with it every output of a query that sees it NaN (also under a weight of 0); the row is written as
// zeros, so that queries in front of it are not touched by 0 * NaN, and the unit's first such row is
// noted for the queries behind it.  Rope values need no such care: they only reach their own key's
// scores.
struct GatherArgs {
    const void* c_kv;
    const void* pe;
    const uint8_t* scales;
    const int* seq_lens;     // null: every sequence has Sk keys
    const int* table;        // null: [B, Sk] rows
    int planned;             // whether the plan ran (else every sequence has its units in its own places)
    const int* owner;
    const int* rank;
    const int* count;
    int* unit;               // [B][units] the unit's place in lat / rot
    int* bad;                // [places] first row that is not finite, or 64
    int* exps;               // [places] e (its largest row's, plus kMixed)
    int* row_exps;           // [places][2][64] the latent and the rope rows' own, of mixed units
    int* any_bad;
    int* rows;               // rows in all
    uint16_t* lat;
    uint16_t* rot;
    const uint16_t* W_uk;    // [H][128][512]
    const uint16_t* W_uv;
    int* w_flag;             // [H][2] of W_uk and W_uv: kScaled, kOdd
    int* w_exps;             // [H][2][128] their rows' powers of two, or kOddRow (where flagged)
    uint16_t* w_copy;        // [H][2][128][512] rows under them (where scaled)
    int B, Sk, units, max_pages, page_size, num_pages, block_shift, H, w_groups;
};

template <typename TL>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = Half<TL>::kF16 ? 0x7c00u : 0x7f80u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// 2^k, for k in [-126, 127]
__device__ __forceinline__ float two_to(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
// the exponent of a positive float; zero and what is below 2^-100 count as 2^-100 (so that values under
// 2^-e, and outputs under 2^e, stay in float32's range)
__device__ __forceinline__ int exponent_of(float x) { return max((int)(__float_as_uint(x) >> 23) - 127, -100); }

// two 16-bit values, or two of four e4m3 codes under a power of two in the 16-bit type
template <typename TL>
__device__ __forceinline__ v2f_t halves(uint32_t w) {
    return v2f_t{Half<TL>::to_f32(w & 0xffffu), Half<TL>::to_f32(w >> 16)};
}
template <typename TL>
__device__ __forceinline__ v2u_t decode_half4(uint32_t w, float scale) {
    const v2f_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
    const v2f_t hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
    return v2u_t{Half<TL>::pack2(lo[0], lo[1]), Half<TL>::pack2(hi[0], hi[1])};
}
__device__ __forceinline__ float finite_max(float m, float x) {
    x = fabsf(x);
    return x < INFINITY ? fmaxf(m, x) : m;
}

constexpr int kGatherThreads = 512, kGatherWaves = kGatherThreads / 64;
constexpr int kWaveRows = kUnit / kGatherWaves;

// ---- weights --------------------------------------------------------------------------------
// fp16 keys and values have bf16's range only as far as the weights are of ordinary size.  Where the largest weight of
// every row (of a head's W_uk or W_uv, zeros aside) is in [2^-9, 1) they are: 512 products with latents below 2^(kHead+1)
// stay below 65504, and a latent row as far below its unit's largest as kSpread lets it be still leaves 11 bits.  A head's
// W_uk or W_uv with a row outside is `scaled`: the product reads a copy whose rows are each brought to [1/2, 1) by
// a power of two, which the attention puts into the query's columns (W_uk) or into the output's (W_uv); so the function
// stays what it is, and the head's numbers do not depend on the weights' unit.  A row with a weight that is not
// finite is `odd` (in fp16 too, whose weights are otherwise as they are): its output column, or for W_uk all of the head,
// is NaN where a query sees a key.  A workgroup has 128 rows, beside the gather's: 128 heads' 33.5 MB make that
// launch 7.4 -> 10.8 us at 512 rows and 9.5 -> 14.0 at 3,400, and the product behind it 23.9 -> 24.9 and (weights on the
// chip by then) 138 -> 121; 16 rows of a wave in flight instead of 8 are not faster (+0.9 us).
constexpr int kScaled = 1, kOdd = 2;          // flags
constexpr int kOddRow = 1 << 16, kZeroRow = -400;   // (zeros count as so small that their query columns weigh nothing)
constexpr float kSmallRow = 1.f / 512;        // rows from here to 1 are as they are

typedef uint16_t v2h_t __attribute__((ext_vector_type(2)));
template <typename TL>
__device__ __forceinline__ void expand_weights(const GatherArgs& a, int h, int half) {
    __shared__ int row_e[kN], w_flags[kGatherWaves];
    constexpr uint32_t kInf = Half<TL>::kF16 ? 0x7c00u : 0x7f80u;
    constexpr int kRows = kN / kGatherWaves, kRun = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const v4u* const src = reinterpret_cast<const v4u*>((half ? a.W_uv : a.W_uk) + (int64_t)h * kN * kR) + kRows * wave * 64 + lane;
    int flag = 0;
    #pragma unroll 1
    for (int r0 = 0; r0 < kRows; r0 += kRun) {
        v4u x[kRun];
        #pragma unroll
        for (int i = 0; i < kRun; ++i) x[i] = src[(r0 + i) * 64];
        #pragma unroll
        for (int i = 0; i < kRun; ++i) {
            v2h_t m = {0, 0};
            #pragma unroll
            for (int k = 0; k < 4; ++k) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2h_t, x[i][k] & 0x7fff7fffu));
            const uint32_t u = min((uint32_t)max(m[0], m[1]), kInf);      // magnitudes, NaN as infinity
            const float top = wave_reduce(Half<TL>::to_f32(u), OpMax());
            int e = Half<TL>::kF16 ? 0 : kZeroRow;
            if (!(top < INFINITY)) {
                e = kOddRow;
                flag |= kOdd | (Half<TL>::kF16 ? 0 : kScaled);
            } else if (!Half<TL>::kF16 && top > 0.f) {
                e = exponent_of(top) + 1;
                if (!(top >= kSmallRow && top < 1.f)) flag |= kScaled;
            }
            if (lane == 0) row_e[kRows * wave + r0 + i] = e;
        }
    }
    if (lane == 0) w_flags[wave] = flag;
    __syncthreads();
    flag = 0;
    for (int w = 0; w < kGatherWaves; ++w) flag |= w_flags[w];
    flag = __builtin_amdgcn_readfirstlane(flag);
    const int at = 2 * h + half;
    if (tid == 0) a.w_flag[at] = flag;
    if (flag == 0) return;
    if (tid < kN) a.w_exps[at * kN + tid] = row_e[tid];
    if constexpr (!Half<TL>::kF16) {
        v4u* const dst = reinterpret_cast<v4u*>(a.w_copy + (int64_t)at * kN * kR) + kRows * wave * 64 + lane;
        #pragma unroll 1
        for (int i = 0; i < kRows; ++i) {
            const int e = row_e[kRows * wave + i];
            v4u x = src[i * 64];
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(x[k]);
                x[k] = e == kOddRow ? 0u : Half<TL>::pack2(ldexpf(v[0], -e), ldexpf(v[1], -e));
            }
            dst[i * 64] = x;
        }
    }
}

template <typename TL, bool F8>
__global__ void __launch_bounds__(kGatherThreads) expand_gather_kernel(GatherArgs a) {
    __shared__ int part[kGatherWaves], w_bad[kGatherWaves];
    __shared__ float row_top[2][kUnit];     // latent, rope
    const int j = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (j >= a.units) {
        const int i = b * a.w_groups + j - a.units;
        if (i < 2 * a.H) expand_weights<TL>(a, i >> 1, i & 1);
        return;
    }
    const int k0 = j * kUnit;
    // (with the length, not behind it; the table spans all units)
    const int page = a.table ? load_uniform(a.table + (int64_t)b * a.max_pages + k0 / a.page_size) : 0;
    const int len = a.seq_lens ? min(max(load_uniform(a.seq_lens + b), 0), a.Sk) : a.Sk;
    const bool first = j == 0 && b == 0;
    const bool here = j * kUnit < len;
    if (!here && !first) return;     // the first workgroup leaves the number of rows, whatever it has
    int place = b * a.units + j, own = b;
    if (a.planned) {
        const int at = place;
        own = here ? a.owner[at] : 0;
        // units of the sequences in front of the owner; the first workgroup also adds up all of them
        int sum = 0, all = 0;
        for (int c = tid; c < (first ? a.B : own); c += kGatherThreads) {
            const int n = a.count[c];
            all += n;
            sum += c < own ? n : 0;
        }
        sum = wave_sum(sum);
        if (lane == 0) part[wave] = sum;
        __syncthreads();
        auto total = [&]() __attribute__((always_inline)) {
            int n = 0;
            for (int w = 0; w < kGatherWaves; ++w) n += part[w];
            return n;
        };
        sum = total();
        if (first) {
            __syncthreads();
            all = wave_sum(all);
            if (lane == 0) part[wave] = all;
            __syncthreads();
            if (tid == 0) *a.rows = kUnit * total();
        }
        if (!here) return;
        place = sum + a.rank[(int64_t)own * a.units + j];
        if (tid == 0) a.unit[at] = place;
        if (own != b) return;
    } else if (tid == 0) {
        if (here) a.unit[place] = place;
        if (first) *a.rows = a.B == 1 ? (len + kUnit - 1) / kUnit * kUnit : kUnit * a.B * a.units;
    }

    if (!here) return;

    // where the unit's rows lie (a page is a whole number of units)
    int64_t r0 = (int64_t)b * a.Sk + k0;
    bool in = true;
    if (a.table) {
        in = page >= 0 && page < a.num_pages;
        r0 = (int64_t)page * a.page_size + k0 % a.page_size;
    }
    const int n = in ? min(kUnit, len - k0) : 0;
    uint16_t* lat = a.lat + (int64_t)place * kUnit * kR;
    uint16_t* rot = a.rot + (int64_t)place * kUnit * kD;
    // latent rows: 8 columns a lane; rope rows: 8 lanes a row.  All loads before their first use: rows behind the end
    // read the last one, and are zeros.  A wave's rows, of both, are in one block of scales.
    static_assert(kWaveRows == 8, "a wave's latent and rope rows are the same 8");
    v4u x[kWaveRows], y;
    const int w0 = kWaveRows * wave, yr = tid >> 3;
    #pragma unroll
    for (int i = 0; i < kWaveRows; ++i) x[i] = v4u{0, 0, 0, 0};
    y = v4u{0, 0, 0, 0};
    if (n > 0) {
        typedef std::conditional_t<F8, v2u_t, v4u> Raw;
        constexpr int kSize = F8 ? 1 : 2;
        const uint8_t* lat_in = static_cast<const uint8_t*>(a.c_kv) + r0 * (kR * kSize);
        const uint8_t* rot_in = static_cast<const uint8_t*>(a.pe) + r0 * (kD * kSize);
        Raw u[kWaveRows], v;
        float f = 1.f, g = 1.f;
        if constexpr (F8) {
            const uint8_t* s = a.scales + 2 * ((r0 + w0) >> a.block_shift);
            f = __uint_as_float((uint32_t)s[0] << 23);
            g = __uint_as_float((uint32_t)s[1] << 23);
        }
        #pragma unroll
        for (int i = 0; i < kWaveRows; ++i) u[i] = reinterpret_cast<const Raw*>(lat_in + min(w0 + i, n - 1) * (kR * kSize))[lane];
        v = reinterpret_cast<const Raw*>(rot_in + min(yr, n - 1) * (kD * kSize))[tid & 7];
        #pragma unroll
        for (int i = 0; i < kWaveRows; ++i) {
            if (w0 + i >= n) continue;
            if constexpr (F8) {
                const v2u_t lo = decode_half4<TL>(u[i][0], f), hi = decode_half4<TL>(u[i][1], f);
                x[i] = v4u{lo[0], lo[1], hi[0], hi[1]};
            } else {
                x[i] = u[i];
            }
        }
        if (yr < n) {
            if constexpr (F8) {
                const v2u_t lo = decode_half4<TL>(v[0], g), hi = decode_half4<TL>(v[1], g);
                y = v4u{lo[0], lo[1], hi[0], hi[1]};
            } else {
                y = v;
            }
        }
    }
    int worst = kUnit;
    if constexpr (!Half<TL>::kF16) {
        float top = 0.f;
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const v2f_t v = halves<TL>(y[k]);
            top = finite_max(finite_max(top, v[0]), v[1]);
        }
        #pragma unroll
        for (int k = 1; k < 8; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
        if ((tid & 7) == 0) row_top[1][yr] = top;
    }
    #pragma unroll
    for (int i = 0; i < kWaveRows; ++i) {
        const bool odd = not_finite2<TL>(x[i][0]) || not_finite2<TL>(x[i][1]) || not_finite2<TL>(x[i][2]) ||
                         not_finite2<TL>(x[i][3]);
        if (__builtin_amdgcn_ballot_w64(odd) != 0) {
            worst = min(worst, w0 + i);
            x[i] = v4u{0, 0, 0, 0};
        }
        if constexpr (!Half<TL>::kF16) {
            float top = 0.f;
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(x[i][k]);
                top = fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1])));
            }
            top = wave_reduce(top, OpMax());
            if (lane == 0) row_top[0][w0 + i] = top;
        }
    }
    if (lane == 0) w_bad[wave] = worst;
    __syncthreads();
    for (int w = 0; w < kGatherWaves; ++w) worst = min(worst, w_bad[w]);
    // the unit's exponent, and whether its latent rows (those that are not zero) keep near it; in a mixed unit
    // those that are zero count as its largest latent row
    int e = 0, lat_e = 0, rope_e = 0;
    bool mixed = false;
    if constexpr (!Half<TL>::kF16) {
        const float top = row_top[0][lane], rope = row_top[1][lane];
        e = exponent_of(wave_reduce(fmaxf(top, rope), OpMax())) - kHead;
        lat_e = exponent_of(top > 0.f ? top : wave_reduce(top, OpMax())) - kHead;      // of row `lane`
        rope_e = rope > 0.f ? exponent_of(rope) - kHead : e;
        mixed = __builtin_amdgcn_ballot_w64(e - (top > 0.f ? lat_e : rope_e) > kSpread) != 0;
        if (!mixed) rope_e = e;
        if (!mixed) lat_e = e;
        else if (wave < 2) a.row_exps[((int64_t)place * 2 + wave) * kUnit + lane] = wave ? rope_e : lat_e;
    }
    if (tid == 0) {
        a.exps[place] = mixed ? e + kMixed : e;
        a.bad[place] = worst;
        if (a.any_bad && worst < kUnit) *a.any_bad = 1;   // cleared by the plan; every writer writes the same
    }
    #pragma unroll
    for (int i = 0; i < kWaveRows; ++i) {
        v4u o = x[i];
        if constexpr (!Half<TL>::kF16) {
            const float f = two_to(-__builtin_amdgcn_readlane(lat_e, w0 + i));
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(x[i][k]);
                o[k] = Half<TL>::pack2(v[0] * f, v[1] * f);
            }
        }
        reinterpret_cast<v4u*>(lat + (w0 + i) * kR)[lane] = o;
    }
    v4u o = y;
    if constexpr (!Half<TL>::kF16) {
        const float f = two_to(-__shfl(rope_e, yr));
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
            const v2f_t v = halves<TL>(y[k]);
            o[k] = pack_f16x2(v[0] * f, v[1] * f);
        }
    }
    reinterpret_cast<v4u*>(rot + yr * kD)[tid & 7] = o;
}

// ---- attention ------------------------------------------------------------------------------
// A workgroup has 128 query rows of one head, a wave 32 of them, and walks the keys in steps of a
// unit: its keys (nope 16 KB, rope 8 KB) and values (16 KB) go global -> LDS with direct loads, two
// stages of them, and two workgroups share a CU.
// A wave's scores are S^T = K Q^T, 32 keys x 32 queries an accumulator: a lane has one query's
// scores (the other half-wave the other half of them), so that maxima, sums and rescaling are a
// lane's own business, and the exponentials, packed as they lie, are the B operand of O^T = V^T P^T:
// a lane's eight of a 16-key step are keys 4h + 0..3 and 8 + 4h + 0..3 (h: its half), and V's
// transposing reads take the rows in that order.
// The reference of a row's exponentials moves only when a score passes it by kRise powers of two (few
// do after the first step), and what is in the accumulators is scaled then.  They are fp16, as keys and
// values are (the gather's comment): they start at 2^kBias, so that small ones keep more bits above
// fp16's subnormals, and rise to 2^(kBias + kRise) < 65504; their sum is of what is packed.
// A unit's power of two is one number a step: its keys' goes into the factor of the scores, its values'
// into the exponentials, as d = e - E <= 0 with the largest e so far in E (what is in the accumulators
// is scaled when that grows); the sum takes it out again.  Where d is far below, or the unit is mixed, fp16
// exponentials would lose it: there they stay without it, and the values' product, for rows of like
// exponents at a time, is scaled in float32.  Where d is far above (2^kGrow, past which what is in the accumulators could
// leave float32), too: the power of two of a row then rises where the unit has something under a weight for it, and stays
// where the row does not see the keys that are so large.  Such steps are done outside the loop of the ordinary ones, which
// so keeps its registers (inside it they cost up to 28%).  bf16 queries are made fp16 under a power of two of their own.
// What bounds it: the matrix cores' power, and what does not fit beside them.  4,096 causal rows of 128 heads 711 us, 967
// TFLOP/s; 2,048 rows over 32,768 keys of 16 heads 640, 1,040 TFLOP/s (a large fp16 library product 1,318).  The second
// (666 in the run of these) takes 629 us without exponentials, 609 without reads of fragments, 559 without softmax and
// reads, that is with its matrix instructions, barriers and loads of stages alone, and 471 without any matrix
// instruction; the cores are busy 0.58 and 0.67 of the cycles and the VALU issues in 0.44, at the clock that they leave
// (no counter here shows it; with operands of zeros the second is a fifth faster).  Other structures, each on one card
// against this one: the next step's scores and the last one's values between the exponentials of a step (+6%), the same
// with 64 rows a wave in 512 registers (+60%) or eight waves a workgroup (+10%); eight waves of which four have matrix
// instructions between two barriers while four have exponentials (-3% where most keys are visible, +4 to +10% where tiles
// of 256 rows meet the diagonal or a chunk's end); loads between the score MFMAs (+12%), the MFMAs at a higher wave
// priority (+1%), windows of 3 and 4 fragments (+0.3%, +1.5%), left to the compiler's order (+5%).
struct HeadsArgs {
    const uint16_t* qn;      // [B, Sq, H, 128]
    const uint16_t* qr;      // [B, Sq, H, 64]
    const uint16_t* kv;      // [heads][rows_cap][256]
    const uint16_t* rot;     // [rows_cap][64]
    const int* unit;
    const int* bad;
    const int* exps;
    const int* row_exps;
    const int* any_bad;      // null: look for yourself
    const int* w_flag;       // as the gather's
    const int* w_exps;
    const int* seq_lens;
    const int* new_lens;
    const int* order;        // null: as they come
    uint16_t* out;           // [B, Sq, H, 128]
    float* part;             // SPLIT: [splits][B, Sq, heads][128] rows of a split, divided by its sums,
    float2* state;           // [splits][B, Sq, heads] {reference, sum}
    int B, Sq, Sk, H, h0, heads, units, tiles, causal, splits;
    int64_t head_stride;     // elements of kv a head
    float c;                 // log2(e) / scale
};

constexpr int kHRows = 128, kHThreads = 256;
constexpr int kLeast = 100 + kHead;          // the least unit's power of two is 2^-kLeast
constexpr int kGrow = 32;                    // powers of two that an ordinary step raises a wave's by
constexpr int kWinK = 2, kWinV = 3;          // fragments read ahead (keys by pairs)
constexpr int kKBytes = kUnit * 2 * kN, kRBytes = kUnit * 2 * kD;       // a stage's parts
constexpr int kKeyBytes = kKBytes + kRBytes;                            // keys: nope and rope columns
constexpr int kSlice = kUnit * 64;
constexpr int kStageBytes = kKeyBytes + kKBytes, kVAt = kKeyBytes;      // then values

// Two outputs in their type.  An average of fp16 values up to 65504 stays there, also where its weights
// are rounded up (a NaN is NaN).
template <typename TL>
__device__ __forceinline__ uint32_t to_half2(float x, float y) {
    if constexpr (Half<TL>::kF16) {
        x = fabsf(x) > 65504.f ? copysignf(65504.f, x) : x;
        y = fabsf(y) > 65504.f ? copysignf(65504.f, y) : y;
    }
    return Half<TL>::pack2(x, y);
}

// PAIR: chunks of up to 64 rows, which two waves have; the other two take the second half of each step's keys, and
// the halves are joined at the end (a call of 64 rows over 512 keys 49.2 -> 46.2 us, eight of 64 over 512 240 -> 233,
// 64 over 8,256 485 -> 478).
template <typename TL, bool SPLIT, bool PAIR>
__global__ void __launch_bounds__(kHThreads, 2) heads_kernel(HeadsArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStageBytes];
    constexpr float kRise = 6.f, kBias = 8.f;
    constexpr int KB = PAIR ? 1 : 2;              // 32 keys, of a step's 64, a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, q = lane & 31;
    const uint32_t lds0 = lds_addr(smem);

    // The longest sequences first; an XCD has heads of its own (one in eight; where that does not divide, a
    // contiguous run of all items), whose tiles follow one another and find each other's keys in its L2, those that
    // see most first.  Where a sequence's tiles differ (the chunk is an eighth of its keys or more) they are taken
    // from four heads in turn, so that no head's long ones are left for the end: the 4,096 rows 788 -> 757 us; of
    // chunks a tenth of their keys four heads' keys at a time would only fill the L2 (747 -> 759).
    const bool eighth = a.heads % kNumXCDs == 0;
    int item = eighth ? blockIdx.x / kNumXCDs : xcd_logical_block(blockIdx.x, gridDim.x);
    int sp = 0;
    if constexpr (SPLIT) { sp = item % a.splits; item /= a.splits; }
    const int some = eighth ? a.heads / kNumXCDs : a.heads, share_b = a.tiles * some;
    const int b = a.order ? load_uniform(a.order + item / share_b) : item / share_b;
    item %= share_b;
    const int len = a.seq_lens ? min(max(load_uniform(a.seq_lens + b), 0), a.Sk) : a.Sk;
    int turn = a.causal && len / 8 <= a.Sq ? 4 : 1;
    while (some % turn) --turn;
    const int run = item / (a.tiles * turn), in_run = item % (a.tiles * turn);
    const int t = a.tiles - 1 - in_run / turn;
    const int hs = run * turn + in_run % turn;
    const int hl = eighth ? hs * kNumXCDs + blockIdx.x % kNumXCDs : hs;
    const int h = a.h0 + hl;
    const int fresh = a.new_lens ? min(max(load_uniform(a.new_lens + b), 0), a.Sq) : a.Sq;
    const int pad = a.Sq - fresh;
    const int64_t row_stride = (int64_t)a.H * kN;
    uint16_t* const out = a.out + (int64_t)b * a.Sq * row_stride + (int64_t)h * kN;

    // rows in front of the new ones
    for (int r = kHRows * t + (tid >> 4); sp == 0 && r < min(pad, kHRows * (t + 1)); r += kHThreads / 16)
        reinterpret_cast<v4u*>(out + r * row_stride)[tid & 15] = v4u{0, 0, 0, 0};
    const int r0 = pad + kHRows * t;
    if (r0 >= a.Sq) return;

    // row i sees keys up to lim(i)
    auto lim_of = [&](int row) __attribute__((always_inline)) {
        return a.causal ? min(len - a.Sq + row, len - 1) : len - 1;
    };
    const int w0 = r0 + 32 * (PAIR ? wave & 1 : wave), kh = PAIR ? 32 * (wave >> 1) : 0;   // first row, and key of a step
    const int row = min(w0 + q, a.Sq - 1);
    const int lim = lim_of(row);
    const int wave_first = w0 < a.Sq ? lim_of(w0) : -1, wave_last = w0 < a.Sq ? lim_of(min(w0 + 31, a.Sq - 1)) : -1;
    int n_tiles = (lim_of(min(r0 + kHRows, a.Sq) - 1) + kUnit) / kUnit;   // lim -1: 0
    int first = 0;               // SPLIT: a share of them
    n_tiles = max(n_tiles, 0);
    if constexpr (SPLIT) {
        const int share = (n_tiles + a.splits - 1) / a.splits;
        first = sp * share;
        n_tiles = min(n_tiles, first + share);
    }

    v4u qf[12];
    {
        const uint16_t* p = a.qn + ((int64_t)b * a.Sq + row) * row_stride + (int64_t)h * kN + 8 * hi;
        #pragma unroll
        for (int i = 0; i < 8; ++i) qf[i] = *reinterpret_cast<const v4u*>(p + 16 * i);
        const uint16_t* r = a.qr + (((int64_t)b * a.Sq + row) * a.H + h) * kD + 8 * hi;
        #pragma unroll
        for (int i = 0; i < 4; ++i) qf[8 + i] = *reinterpret_cast<const v4u*>(r + 16 * i);
    }
    int qe = 0;                  // bf16: the row's power of two
    if (!Half<TL>::kF16 && (load_uniform(a.w_flag + 2 * h) & kScaled)) {
        // columns that W_uk's rows have left their powers of two to
        auto column = [&](int i, int k) __attribute__((always_inline)) {
            if (i >= 8) return 0;
            const int e = a.w_exps[2 * kN * h + 16 * i + 8 * hi + k];
            return e == kOddRow ? 0 : e;
        };
        int top = -1000;
        #pragma unroll
        for (int i = 0; i < 12; ++i)
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(qf[i][k]);
                #pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float x = fabsf(v[n]);
                    if (x > 0.f && x < INFINITY) top = max(top, exponent_of(x) + column(i, 2 * k + n));
                }
            }
        const auto x = __builtin_amdgcn_permlane32_swap((uint32_t)top, (uint32_t)top, false, false);
        qe = max((int)x[0], (int)x[1]);
        if (qe == -1000) qe = 0;
        #pragma unroll
        for (int i = 0; i < 12; ++i)
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(qf[i][k]);
                qf[i][k] = pack_f16x2(ldexpf(v[0], column(i, 2 * k) - qe), ldexpf(v[1], column(i, 2 * k + 1) - qe));
            }
    } else if constexpr (!Half<TL>::kF16) {
        float top = 0.f;
        #pragma unroll
        for (int i = 0; i < 12; ++i)
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(qf[i][k]);
                top = finite_max(finite_max(top, v[0]), v[1]);
            }
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        qe = min(exponent_of(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]))), 126);
        const float f = two_to(-qe);
        #pragma unroll
        for (int i = 0; i < 12; ++i)
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                const v2f_t v = halves<TL>(qf[i][k]);
                qf[i][k] = pack_f16x2(v[0] * f, v[1] * f);
            }
    }

    // ---- staging, in slices of 64 bytes a row: a load is 16 rows of one, lane l chunk l % 4 of row
    // l / 4.  Chunk c of a key or rope row r lies at c ^ ((r >> 2) & 3) (the 16 lanes of a ds_read_b128 cycle
    // touch 16 different places of 256 bytes), values as they come (four rows of a transposing read are
    // 256 bytes).  So a step's reads differ by constants, but for one bit in keys.
    const uint64_t kv = reinterpret_cast<uint64_t>(a.kv + hl * a.head_stride);
    const uint64_t rot = reinterpret_cast<uint64_t>(a.rot);
    const int* units = a.unit + (int64_t)b * a.units;
    const uint32_t r16 = 16 * wave + (lane >> 2), c_sw = 16 * ((lane & 3) ^ (lane >> 4));
    const uint32_t voff_k = r16 * 512 + c_sw, voff_r = r16 * 128 + c_sw;
    const uint32_t voff_v = r16 * 512 + 256 + 16 * (lane & 3);
    auto issue = [&](int place, uint32_t st) __attribute__((always_inline)) {
        const v4i rk = rsrc_span(kv + (uint64_t)place * (kUnit * 512), 0, kUnit * 512);
        const v4i rr = rsrc_span(rot + (uint64_t)place * (kUnit * 128), 0, kUnit * 128);
        const uint32_t base = __builtin_amdgcn_readfirstlane(lds0 + st + 1024 * wave);
        #pragma unroll
        for (int i = 0; i < 6; ++i) dma16(i < 4 ? rk : rr, base + kSlice * i, i < 4 ? voff_k + 64 * i : voff_r + 64 * (i - 4));
        #pragma unroll
        for (int i = 0; i < 4; ++i) dma16(rk, base + kVAt + kSlice * i, voff_v + 64 * i);
    };

    // ---- fragments
    const uint32_t k_rd = (uint32_t)(kh + q) * 64 + 16 * (hi ^ ((q >> 2) & 3));
    const int G4 = lane >> 4, q4 = (lane >> 2) & 3, i4 = lane & 3;
    const uint32_t v_rd = (uint32_t)(kh + 4 * (G4 >> 1) + q4) * 64 + 32 * (G4 & 1) + 8 * i4;
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    auto k_frag = [&](uint32_t st, int kb, int i) __attribute__((always_inline)) {   // i: 16 of 192 columns
        return *reinterpret_cast<const v4u*>(smem + st + kSlice * (i >> 1) + 2048 * kb + (k_rd ^ (32 * (i & 1))));
    };
    auto v_frag = [&](uint32_t st, int i) __attribute__((always_inline)) {   // i: 4 * (16 keys) + columns
        const uint8_t* at = smem + st + kVAt + kSlice * (i & 3) + 1024 * (i >> 2) + v_rd;
        const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
        const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 512));
        return __builtin_bit_cast(v4u, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    v16f o[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = v16f{};
    float m_ref = -INFINITY, l = 0.f;
    const h2_t ones = {(_Float16)1.f, (_Float16)1.f};

    int next = n_tiles > first ? load_uniform(units + first) : 0, here = next;
    int e_next = n_tiles > first ? load_uniform(a.exps + next) : 0;
    if (n_tiles > first) issue(next, 0);
    next = n_tiles > first + 1 ? load_uniform(units + first + 1) : 0;
    int E = -1000;               // below any unit's (-kLeast)

    // ---- steps
    int j = first, place = 0, ee = 0;
    uint32_t st = 0;
    auto begin = [&]() __attribute__((always_inline)) {     // step j's data are there, the next one's on their way
        st = ((j - first) & 1) * kStageBytes;
        wait_vm<0>();
        lds_barrier();      // step j has landed; every wave is done with step j - 1
        place = here, ee = e_next;
        here = next;
        if (j + 1 < n_tiles) {
            issue(next, kStageBytes - st);
            e_next = load_uniform(a.exps + next);
            next = j + 2 < n_tiles ? load_uniform(units + j + 2) : 0;
        }
    };
    auto hide = [&](v16f (&s)[KB]) __attribute__((always_inline)) {
        if (j * kUnit + kUnit - 1 <= wave_first) return;
        int past = lim - j * kUnit - kh - 4 * hi;                // (opaque: 32 differences are not to stay in registers)
        asm volatile("" : "+v"(past));
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb)
            #pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + acc_row(i, 0) <= past ? s[kb][i] : -INFINITY;
    };
    // (not 0, which under zero queries and keys it could round to: a hidden score times it has to stay -infinity)
    auto factor = [&](int e) __attribute__((always_inline)) {
        return fmaxf(Half<TL>::kF16 ? a.c : ldexpf(a.c, qe + e), 1.17549435e-38f);
    };
    auto scale_out = [&](float f) __attribute__((always_inline)) {
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            #pragma unroll
            for (int k = 0; k < 16; ++k) o[i][k] *= f;
    };
    auto grow = [&](int ev) __attribute__((always_inline)) {
        if (ev <= E) return;
        const float f = ev - E > 126 ? 0.f : two_to(E - ev);
        E = ev;
        scale_out(f);
    };
    bool huge = false, apart = false;   // apart: the rows of the wave have powers of two of their own,
    int Er = 0;                         // 2^Er, in place of 2^E
    // Moves the references of rows whose scores passed them (those only).  Past 2^24 a reference is off its own score by
    // more than a power of two, which a fused product would show, and so would another order of sums: `huge`.  An
    // ordinary step that finds it leaves everything as it is to the step that is done apart, which refers to scores
    // of its own making.
    auto refer = [&](const v16f (&s)[KB], float ct, bool ordinary) __attribute__((always_inline)) {
        float top = fmaxf(s[0][0], s[0][1]);
        #pragma unroll
        for (int i = 2; i < 16; i += 2) top = fmaxf(fmaxf(s[0][i], s[0][i + 1]), top);
        #pragma unroll
        for (int i = 16; i < 16 * KB; i += 2) top = fmaxf(fmaxf(s[i >> 4][i & 15], s[i >> 4][(i & 15) + 1]), top);
        if (__builtin_amdgcn_ballot_w64(top * ct > m_ref + kRise)) {
            const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * ct;
            const bool over = top > m_ref + kRise;
            const float m = over ? top : m_ref;
            huge = __builtin_amdgcn_ballot_w64(fabsf(m) > 16777216.f && fabsf(m) < INFINITY) != 0;
            if (ordinary && huge) return;
            const float f = over ? __builtin_amdgcn_exp2f(m_ref - m) : 1.f;
            m_ref = m;
            l *= f;
            scale_out(f);
        }
    };
    #pragma unroll 1
    while (j < n_tiles) {
        #pragma unroll 1
        for (; j < n_tiles; ++j) {
            begin();
            if (j * kUnit + kh > wave_last) continue;
            if (__builtin_expect(huge || apart || ee > kMixed / 2 || E - ee > 8 || (ee - E > kGrow && E >= -kLeast), 0)) break;
            // scores; a fragment's place is read again as soon as it is used
            v16f s[KB] = {};
            v4u kf[kWinK][KB];
            #pragma unroll
            for (int i = 0; i < kWinK; ++i)
                #pragma unroll
                for (int kb = 0; kb < KB; ++kb) kf[i][kb] = k_frag(st, kb, i);
            #pragma unroll
            for (int i = 0; i < 12; ++i) {
                #pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    s[kb] = Mma<f16_t>::sub(kf[i % kWinK][kb], qf[i], 0, s[kb]);
                    if (i + kWinK < 12) kf[i % kWinK][kb] = k_frag(st, kb, i + kWinK);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            hide(s);
            // weights
            const float ct = factor(ee);
            grow(ee);
            refer(s, ct, true);
            if (__builtin_expect(huge, 0)) break;
            const int d = ee - E;
            const float neg = (m_ref == -INFINITY ? 0.f : kBias - m_ref) + (float)d;
            float sum = 0.f;
            v4u p[2 * KB];
            #pragma unroll
            for (int i = 0; i < 8 * KB; ++i) {
                const int kb = i >> 3, k = 2 * (i & 7);
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][k], ct, neg));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][k + 1], ct, neg));
                const uint32_t w = pack_f16x2(x, y);
                p[i >> 2][i & 3] = w;
                sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, w), ones, sum, false);
            }
            l += sum * two_to(-d);
            // values
            v4u vf[kWinV];
            #pragma unroll
            for (int i = 0; i < kWinV; ++i) vf[i] = v_frag(st, i);
            #pragma unroll
            for (int i = 0; i < 8 * KB; ++i) {
                o[i & 3] = Mma<f16_t>::sub(vf[i % kWinV], p[i >> 2], 0, o[i & 3]);
                if (i + kWinV < 8 * KB) vf[i % kWinV] = v_frag(st, i + kWinV);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (j >= n_tiles) break;
        // A step that is not ordinary.  A mixed unit's scores have its nope and rope columns each under their row's power
        // of two.  They are made in their own units, 2^qe and a.c in them: nothing of a row's passes through another's.
        const bool mixed = ee > kMixed / 2;
        const int e = mixed ? ee - kMixed : ee;
        const int* const rows = a.row_exps + (int64_t)place * 2 * kUnit;
        auto row_exps = [&](int rope, int kb, int i) __attribute__((always_inline)) {   // 4 keys from 8 i + 4 h on
            return mixed ? *reinterpret_cast<const v4i*>(rows + kUnit * rope + kh + 32 * kb + 8 * i + 4 * hi) : v4i{e, e, e, e};
        };
        const int mine = mixed ? rows[lane] : e;           // row `lane`
        v16f s[KB];
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            v16f r = {};
            s[kb] = v16f{};
            #pragma unroll
            for (int i = 0; i < 8; ++i) s[kb] = Mma<f16_t>::sub(k_frag(st, kb, i), qf[i], 0, s[kb]);
            #pragma unroll
            for (int i = 8; i < 12; ++i) r = Mma<f16_t>::sub(k_frag(st, kb, i), qf[i], 0, r);
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v4i x = row_exps(0, kb, i), y = row_exps(1, kb, i);
                #pragma unroll
                for (int k = 0; k < 4; ++k)
                    s[kb][4 * i + k] = ldexpf(s[kb][4 * i + k] * a.c, x[k] + qe) + ldexpf(r[4 * i + k] * a.c, y[k] + qe);
            }
        }
        hide(s);
        refer(s, 1.f, false);
        // score and reference rounded alike; exponentials without a unit's power of two, in float32; then the values'
        // product in levels of rows whose exponents are within kSpread of the largest one left
        const float m = m_ref == -INFINITY ? 0.f : m_ref;
        float sum = 0.f;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb)
            #pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(s[kb][i] - m + kBias);
                sum += s[kb][i];
            }
        l += sum;
        if (!apart) Er = E;
        int level = mine;
        #pragma unroll
        for (int i = 1; i < 64; i *= 2) level = max(level, __shfl_xor(level, i));
        level = __builtin_amdgcn_readfirstlane(level);
        #pragma unroll 1
        while (true) {
            v4u p[2 * KB];
            #pragma unroll
            for (int i = 0; i < 4 * KB; ++i) {
                const v4i x = row_exps(0, i >> 2, i & 3);
                #pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    float v[2];
                    #pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int ex = x[k + n];
                        v[n] = ex <= level && ex >= level - kSpread ? s[i >> 2][4 * (i & 3) + k + n] * two_to(ex - level) : 0.f;
                    }
                    p[i >> 1][2 * (i & 1) + (k >> 1)] = pack_f16x2(v[0], v[1]);
                }
            }
            auto product = [&](int vb) __attribute__((always_inline)) {
                v16f t = {};
                #pragma unroll
                for (int i = 0; i < 2 * KB; ++i) t = Mma<f16_t>::sub(v_frag(st, 4 * i + vb), p[i], 0, t);
                return t;
            };
            // a row's power of two rises where the level gives it something, not for keys that it does not see
            float most = 0.f;
            #pragma unroll 1
            for (int vb = 0; vb < 4; ++vb) {
                const v16f t = product(vb);
                #pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(t[i]));
            }
            const int up = most > 0.f ? max(Er, level) : Er;
            if (__builtin_amdgcn_ballot_w64(up > Er)) scale_out(up - Er > 126 ? 0.f : two_to(Er - up));
            Er = up;
            const float f = level > Er || level - Er < -126 ? 0.f : two_to(level - Er);
            #pragma unroll
            for (int vb = 0; vb < 4; ++vb) {
                const v16f t = product(vb);
                #pragma unroll
                for (int i = 0; i < 16; ++i) o[vb][i] = __builtin_fmaf(t[i], f, o[vb][i]);
            }
            int below = mine < level - kSpread ? mine : -0x7fffffff;
            #pragma unroll
            for (int i = 1; i < 64; i *= 2) below = max(below, __shfl_xor(below, i));
            below = __builtin_amdgcn_readfirstlane(below);
            if (below == -0x7fffffff) break;
            level = below;
        }
        E = __builtin_amdgcn_readfirstlane(Er);
        apart = __builtin_amdgcn_ballot_w64(Er != E) != 0;
        ++j;
    }
    if (!apart) Er = E;

    {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    if constexpr (PAIR) {
        // 16 KB of outputs, references, sums and powers of two from each wave of the second halves
        float* const theirs = reinterpret_cast<float*>(smem) + (wave & 1) * (67 * 64) + lane;
        __syncthreads();
        if (kh) {
            #pragma unroll
            for (int i = 0; i < 64; ++i) theirs[64 * i] = o[i >> 4][i & 15];
            theirs[64 * 64] = m_ref;
            theirs[64 * 65] = l;
            theirs[64 * 66] = __int_as_float(Er);
        }
        __syncthreads();
        if (kh) return;
        const float m1 = theirs[64 * 64], l1 = theirs[64 * 65];
        const int E1 = __float_as_int(theirs[64 * 66]), top = max(Er, E1);
        const float m = fmaxf(m_ref, m1);
        float f0 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m_ref - m), f1 = l1 == 0.f ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
        l = l * f0 + l1 * f1;
        f0 = top - Er > 126 ? 0.f : f0 * two_to(Er - top);
        f1 = top - E1 > 126 ? 0.f : f1 * two_to(E1 - top);
        m_ref = m;
        Er = top;
        #pragma unroll
        for (int i = 0; i < 64; ++i) o[i >> 4][i & 15] = o[i >> 4][i & 15] * f0 + theirs[64 * i] * f1;
    }
    float f = l == 0.f || Er < -kLeast ? 0.f : two_to(Er) / l;      // (without any value that counts: zeros)
    if (!a.any_bad || load_uniform(a.any_bad)) {
        int worst = 0x7fffffff;
        for (int j = first + lane; j < n_tiles; j += 64) {
            const int r = a.bad[units[j]];
            if (r < kUnit) worst = min(worst, j * kUnit + r);
        }
        #pragma unroll
        for (int i = 1; i < 64; i *= 2) worst = min(worst, __shfl_xor(worst, i));
        if (worst <= lim) l = f = __uint_as_float(0x7fc00000u);
    }
    const int w_uk = load_uniform(a.w_flag + 2 * h), w_uv = load_uniform(a.w_flag + 2 * h + 1);
    if ((w_uk & kOdd) && l != 0.f) l = f = __uint_as_float(0x7fc00000u);
    if (w0 + q >= a.Sq) return;
    auto outputs = [&](int vb, int i) __attribute__((always_inline)) {     // four columns from 32 vb + 2 i + 4 hi on
        v4f x = {o[vb][i], o[vb][i + 1], o[vb][i + 2], o[vb][i + 3]};
        if (w_uv == 0) return x * f;
        // W_uv's rows' powers of two
        const v4i e = *reinterpret_cast<const v4i*>(a.w_exps + (2 * h + 1) * kN + 32 * vb + 2 * i + 4 * hi);
        const float g = f == 0.f ? 0.f : f != f ? f : 1.f / l;
        #pragma unroll
        for (int k = 0; k < 4; ++k)
            x[k] = e[k] != kOddRow ? ldexpf(x[k] * g, Er + e[k]) : l == 0.f ? 0.f : __uint_as_float(0x7fc00000u);
        return x;
    };
    if constexpr (SPLIT) {
        const int64_t at = ((int64_t)(sp * a.B + b) * a.Sq + row) * a.heads + hl;
        if (hi == 0) a.state[at] = make_float2(m_ref, l);
        float* const dst = a.part + at * kN + 4 * hi;
        #pragma unroll
        for (int vb = 0; vb < 4; ++vb)
            #pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<v4f*>(dst + 32 * vb + 2 * i) = outputs(vb, i);
    } else {
        uint16_t* const dst = out + row * row_stride + 4 * hi;
        #pragma unroll
        for (int vb = 0; vb < 4; ++vb)
            #pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const v4f x = outputs(vb, i);
                *reinterpret_cast<v2u_t*>(dst + 32 * vb + 2 * i) = v2u_t{to_half2<TL>(x[0], x[1]), to_half2<TL>(x[2], x[3])};
            }
    }
}

// Rows from their splits' (averages of values, each with the reference and sum of its weights): half a wave
// a row.
template <typename TL>
__global__ void __launch_bounds__(256) heads_merge_kernel(HeadsArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)a.B * a.Sq * a.heads;
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= rows) return;
    const int64_t bi = r / a.heads;
    const int hl = (int)(r - bi * a.heads), b = (int)(bi / a.Sq), i = (int)(bi - (int64_t)b * a.Sq);
    const int fresh = a.new_lens ? min(max(a.new_lens[b], 0), a.Sq) : a.Sq;
    if (i < a.Sq - fresh) return;        // padding has its zeros
    float M = -INFINITY;
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.state[s * rows + r].x);
    v4f o = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float2 x = a.state[s * rows + r];
        if (x.y == 0.f) continue;        // no key seen there
        const float w = x.y * __builtin_amdgcn_exp2f(x.x - M);
        total += w;
        o += *reinterpret_cast<const v4f*>(a.part + (s * rows + r) * kN + 4 * lane) * w;
    }
    const float f = total == 0.f ? 0.f : 1.f / total;
    uint16_t* const dst = a.out + (bi * a.H + a.h0 + hl) * kN;
    reinterpret_cast<v2u_t*>(dst)[lane] = v2u_t{to_half2<TL>(o[0] * f, o[1] * f), to_half2<TL>(o[2] * f, o[3] * f)};
}

template <typename TL, bool SPLIT>
void launch_heads(const HeadsArgs& a, dim3 grid, hipStream_t stream) {
    if (a.Sq <= 64) hipLaunchKernelGGL((heads_kernel<TL, SPLIT, true>), grid, dim3(kHThreads), 0, stream, a);
    else hipLaunchKernelGGL((heads_kernel<TL, SPLIT, false>), grid, dim3(kHThreads), 0, stream, a);
}

// ---- queries per head -----------------------------------------------------------------------
// The nope columns of q_raw (fp32 [rows, H (nope + rope)]) in 16 bits, [rows, H, nope].
template <typename TL>
__global__ void __launch_bounds__(256) q_nope_kernel(const float* __restrict__ raw, uint16_t* __restrict__ out,
                                                     int64_t chunks, int nope, int qk) {
    const int per = nope / 8;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < chunks; i += gridDim.x * 256ll) {
        const int64_t r = i / per;
        const float* p = raw + r * qk + 8 * (i - r * per);
        const v4f x = *reinterpret_cast<const v4f*>(p), y = *reinterpret_cast<const v4f*>(p + 4);
        reinterpret_cast<v4u*>(out)[i] = v4u{Half<TL>::pack2(x[0], x[1]), Half<TL>::pack2(x[2], x[3]),
                                             Half<TL>::pack2(y[0], y[1]), Half<TL>::pack2(y[2], y[3])};
    }
}

// Keys and values of this many bytes at a time at most, in groups of heads (one head at least) as alike as multiples
// of the XCDs make them: 128 heads of 512 rows over 33,280 keys 2,730 us in 64 + 64, 3,520 in 127 + 1.  In groups of
// 0.5 GiB they take 2,920 us, in one of 2.1 GiB 2,700.
constexpr int64_t kExpandBytes = (int64_t)2 << 30;
int expand_heads(int H, int64_t rows) {
    int64_t most = std::max<int64_t>(1, kExpandBytes / (rows * 512));
    if (most >= H) return H;
    const int64_t step = most >= kNumXCDs ? kNumXCDs : 1;
    most -= most % step;
    const int64_t groups = (H + most - 1) / most;
    return (int)(((H + groups - 1) / groups + step - 1) / step * step);
}

}  // namespace

// Key splits of the attention, where its workgroups are fewer than two a CU (which share the matrix cores' and
// the VALU's time): 256 of them over 512 units 1,023 us unsplit, 836 in 2, 871 in 3, 836 in 4.  A
// share is at least 8 units of the span (128 workgroups over 8 units 51.1 us unsplit, 52.0 in 2, 54.8 in 4); how much
// of it the sequences hold is not known here, and a tile that sees less has as many, smaller shares.
// MLA_EXPAND_SPLITS overrides the rule.
int expand_splits(int64_t items, int units) {
    if (const char* e = std::getenv("MLA_EXPAND_SPLITS")) {
        const int n = std::atoi(e);
        if (n >= 1) return std::min(n, 64);
    }
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(2 * kNumCUs / items, 16), units / 8));
}

ExpandPlan plan_expand(int B, int Sq, int Sk, int H, bool paged, bool f16) {
    ExpandPlan p;
    p.units = (Sk + kUnit - 1) / kUnit;
    const int64_t places = (int64_t)B * p.units;
    p.rows_cap = places * kUnit;
    p.heads = expand_heads(H, p.rows_cap);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        const size_t at = o;
        o = (o + bytes + 255) / 256 * 256;
        return at;
    };
    p.off_owner = take(paged ? places * 4 : 0);
    p.off_rank = take(paged ? places * 4 : 0);
    p.off_count = take(paged ? (size_t)B * 4 : 0);
    p.off_order = take(paged ? (size_t)B * 4 : 0);
    p.off_unit = take(places * 4);
    p.off_bad = take(places * 4);
    p.off_exps = take(places * 4);
    p.off_row_exps = take(places * 8 * kUnit);
    p.off_any = take(8);                      // any_bad, rows
    p.off_w_flag = take((size_t)H * 8);
    p.off_w_exps = take((size_t)H * 8 * kN);
    p.off_w_copy = take(f16 ? 0 : (size_t)H * 4 * kN * kR);
    p.off_lat = take((size_t)p.rows_cap * kR * 2);
    p.off_rot = take((size_t)p.rows_cap * kD * 2);
    p.off_kv = take((size_t)p.heads * p.rows_cap * 512);
    const int64_t tiles = (Sq + kHRows - 1) / kHRows;
    p.splits = expand_splits(tiles * B * p.heads, p.units);
    const size_t rows = p.splits > 1 ? (size_t)p.splits * B * Sq * p.heads : 0;
    p.off_part = take(rows * kN * 4);
    p.off_state = take(rows * 8);
    p.total = o;
    return p;
}

hipError_t launch_expand(const ExpandProblem& p, const ExpandPlan& plan, void* workspace, hipStream_t stream) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    auto ints = [&](size_t off) { return reinterpret_cast<int*>(ws + off); };
    auto half = [&](size_t off) { return reinterpret_cast<uint16_t*>(ws + off); };
    const int64_t tiles = (p.Sq + kHRows - 1) / kHRows;
    if (p.B > 65535 || plan.rows_cap > 0x7fffffff || tiles * p.B * plan.heads * plan.splits > 0xffffffffll / kHThreads)
        return hipErrorInvalidValue;
    int* any_bad = ints(plan.off_any);
    PlanArgs u;
    u.seq_lens = p.seq_lens; u.table = p.block_table;
    u.owner = ints(plan.off_owner); u.rank = ints(plan.off_rank); u.count = ints(plan.off_count);
    u.order = ints(plan.off_order); u.any_bad = any_bad;
    u.B = p.B; u.Sk = p.Sk; u.units = plan.units;
    u.max_pages = p.block_table ? p.Sk / p.page_size : 0;
    u.per_page = p.block_table ? p.page_size / kUnit : 1;
    // one sequence shares nothing; of up to 64 units a lane of the attention looks each up for itself
    const bool alone = p.B == 1 && plan.units <= kWave;
    if (!alone) hipLaunchKernelGGL(expand_plan_kernel, dim3(p.block_table ? p.B : 1), dim3(kPlanThreads), 0, stream, u);
    GatherArgs g;
    g.c_kv = p.c_kv; g.pe = p.pe; g.scales = static_cast<const uint8_t*>(p.scales);
    g.seq_lens = p.seq_lens; g.table = p.block_table;
    g.owner = u.owner; g.rank = u.rank; g.count = u.count;
    g.unit = ints(plan.off_unit); g.bad = ints(plan.off_bad); g.exps = ints(plan.off_exps);
    g.row_exps = ints(plan.off_row_exps); g.rows = any_bad + 1;
    g.any_bad = alone ? nullptr : any_bad; g.planned = p.block_table && p.B > 1;
    g.lat = half(plan.off_lat); g.rot = half(plan.off_rot);
    g.B = p.B; g.Sk = p.Sk; g.units = plan.units;
    g.page_size = p.page_size; g.max_pages = u.max_pages; g.num_pages = p.num_pages;
    g.block_shift = p.scale_block == 16 ? 4 : p.scale_block == 32 ? 5 : 6;
    g.W_uk = static_cast<const uint16_t*>(p.W_uk); g.W_uv = static_cast<const uint16_t*>(p.W_uv);
    g.w_flag = ints(plan.off_w_flag); g.w_exps = ints(plan.off_w_exps); g.w_copy = half(plan.off_w_copy);
    g.H = p.H; g.w_groups = (2 * p.H + p.B - 1) / p.B;
    const dim3 gather((unsigned)(plan.units + g.w_groups), (unsigned)p.B);
    if (p.scales) {
        if (p.f16) hipLaunchKernelGGL((expand_gather_kernel<f16_t, true>), gather, dim3(kGatherThreads), 0, stream, g);
        else hipLaunchKernelGGL((expand_gather_kernel<bf16_t, true>), gather, dim3(kGatherThreads), 0, stream, g);
    } else {
        if (p.f16) hipLaunchKernelGGL((expand_gather_kernel<f16_t, false>), gather, dim3(kGatherThreads), 0, stream, g);
        else hipLaunchKernelGGL((expand_gather_kernel<bf16_t, false>), gather, dim3(kGatherThreads), 0, stream, g);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;

    HeadsArgs a;
    a.qn = static_cast<const uint16_t*>(p.q_nope); a.qr = static_cast<const uint16_t*>(p.q_rope);
    a.kv = half(plan.off_kv); a.rot = g.rot;
    a.unit = g.unit; a.bad = g.bad; a.exps = g.exps; a.row_exps = g.row_exps; a.any_bad = g.any_bad;
    a.w_flag = g.w_flag; a.w_exps = g.w_exps;
    a.seq_lens = p.seq_lens; a.new_lens = p.new_lens;
    a.order = p.block_table && p.B > 1 ? u.order : nullptr;
    a.part = reinterpret_cast<float*>(ws + plan.off_part);
    a.state = reinterpret_cast<float2*>(ws + plan.off_state);
    a.splits = plan.splits;
    a.out = static_cast<uint16_t*>(p.out);
    a.B = p.B; a.Sq = p.Sq; a.Sk = p.Sk; a.H = p.H; a.units = plan.units;
    a.tiles = (int)tiles; a.causal = p.causal;
    a.head_stride = plan.rows_cap * 256;
    a.c = (float)(1.4426950408889634 / p.scale);
    for (int h0 = 0; h0 < p.H; h0 += plan.heads) {
        const int heads = std::min(plan.heads, p.H - h0);
        KvExpand k;
        k.f16 = p.f16;
        k.lat = g.lat; k.kv = half(plan.off_kv);
        k.W_uk = static_cast<const uint16_t*>(p.W_uk) + (int64_t)h0 * kN * kR;
        k.W_uv = static_cast<const uint16_t*>(p.W_uv) + (int64_t)h0 * kN * kR;
        k.w_flag = g.w_flag + 2 * h0;
        k.w_copy = p.f16 ? nullptr : g.w_copy + (int64_t)h0 * 2 * kN * kR;
        k.rows = g.rows; k.rows_cap = plan.rows_cap; k.heads = heads;
        e = launch_kv_expand(k, stream);
        if (e != hipSuccess) return e;
        a.h0 = h0; a.heads = heads;
        const dim3 grid((unsigned)(tiles * p.B * heads * plan.splits));
        if (plan.splits > 1) {
            if (p.f16) launch_heads<f16_t, true>(a, grid, stream);
            else launch_heads<bf16_t, true>(a, grid, stream);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
            const dim3 merge((unsigned)(((int64_t)p.B * p.Sq * heads + 7) / 8));
            if (p.f16) hipLaunchKernelGGL(heads_merge_kernel<f16_t>, merge, dim3(256), 0, stream, a);
            else hipLaunchKernelGGL(heads_merge_kernel<bf16_t>, merge, dim3(256), 0, stream, a);
        } else {
            if (p.f16) launch_heads<f16_t, false>(a, grid, stream);
            else launch_heads<bf16_t, false>(a, grid, stream);
        }
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_q_nope(const float* raw, void* out, bool f16, int64_t rows, int nope, int qk,
                         hipStream_t stream) {
    const int64_t chunks = rows * (nope / 8);
    const dim3 grid((unsigned)std::min<int64_t>((chunks + 255) / 256, 16 * kNumCUs));
    uint16_t* o = static_cast<uint16_t*>(out);
    if (f16) hipLaunchKernelGGL(q_nope_kernel<f16_t>, grid, dim3(256), 0, stream, raw, o, chunks, nope, qk);
    else hipLaunchKernelGGL(q_nope_kernel<bf16_t>, grid, dim3(256), 0, stream, raw, o, chunks, nope, qk);
    return hipGetLastError();
}

}  // namespace mla
