// Routing rows to experts: scores, choice of the best k and their weights (forward and backward), and the CSR structure
// of the chosen (row, expert) pairs.
//
// topk_route, one row per warp.  With l the row's logits and b the bias (fp32, choice only, no gradient):
//     s = softmax(l) or sigmoid(l)        c = s + b        c = -inf where l = -inf (a masked expert) or c is NaN
//     a group's score = sum of its group_top (1 or 2) largest c; the kept_groups best groups stay open
//     index = the k largest c of the open groups, descending, ties to the lowest index (groups likewise)
//     weight = scale * s[index] / (renormalize ? sum s[index] : 1), 0 where that sum is 0
// The choice must not hang on how exp rounds.  Without bias, and with groups ranked by one score, c orders as l does and the
// choice compares the logits themselves, exactly.  Otherwise it compares scores, in 64 bits where fp32 cannot tell.
//
// Backward (u = grad * scale, sums over the chosen i):
//     softmax, renormalized:  dl_i = w_i (u_i - sum u w)                     with w the softmax over the chosen logits
//     softmax:                dl_j = s_j ([j chosen] u_j - sum u s)          for every expert j
//     sigmoid, renormalized:  dl_i = w_i (1 - s_i) (u_i - sum u w)           with w = s / sum s
//     sigmoid:                dl_i = u_i s_i (1 - s_i)
// and 0 for every expert that has no term.  Under softmax a row with a NaN or +inf has weights of NaN, and so its whole gradient is.
//
// route_csr is a stable counting sort of the pairs by expert; see there.
#include <algorithm>

#include "common.cuh"

namespace opsgnn {
namespace route {

constexpr int kWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

struct RouteParams {
    int64_t rows;
    int32_t experts, k, groups, kept_groups, group_top;
    int32_t softmax, renormalize;
    float scale;
    uint8_t* undefined;  // may be null; forward writes, backward reads 1 for a row whose softmax has no value
};

// Order-preserving keys; 0 is below every number and marks what cannot be chosen any more.  NaN ranks with -inf.
__device__ __forceinline__ uint32_t KeyOf(float v)
{
    v = (v != v) ? -INFINITY : v + 0.0f;  // -0 and +0 are one value
    const uint32_t u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t KeyOf(double v)
{
    v = (v != v) ? -static_cast<double>(INFINITY) : v + 0.0;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ULL);
}

__device__ __forceinline__ uint64_t WarpMax(uint64_t v)
{
    const uint32_t hi = static_cast<uint32_t>(v >> 32);
    const uint32_t top = __reduce_max_sync(kFull, hi);
    const uint32_t lo = __reduce_max_sync(kFull, hi == top ? static_cast<uint32_t>(v) : 0u);
    return (static_cast<uint64_t>(top) << 32) | lo;
}
template <class T> __device__ __forceinline__ T WarpSum(T v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        v += __shfl_xor_sync(kFull, v, d);
    }
    return v;
}

// The same over teams of LANES neighbouring lanes.  The whole warp calls, never from a branch that one team's row takes and
// another's does not: a lane that stays out leaves the others waiting.
template <int LANES> __device__ __forceinline__ float TeamMax(float v)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        v = fmaxf(v, __shfl_xor_sync(kFull, v, d));
    }
    return v;
}
template <int LANES> __device__ __forceinline__ float TeamSum(float v)
{
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        v += __shfl_xor_sync(kFull, v, d);
    }
    return v;
}

// Lane l of a row's lanes holds experts l * VPL + j, j < VPL: a row of whole vectors is read with wide loads.
template <class T, int VPL> __device__ __forceinline__ void LoadRow(const T* row, int experts, bool wide, int lane, float (&out)[VPL])
{
    constexpr int VEC = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : VPL;
    if (wide) {
#pragma unroll
        for (int j = 0; j < VPL; j += VEC) {
            const int at = lane * VPL + j;
            if (at < experts) {
                const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(row + at);
                float f[VEC];
                Unpack<float, T, VEC>(p, f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    out[j + i] = f[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    out[j + i] = -INFINITY;
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int at = lane * VPL + j;
            out[j] = at < experts ? Widen<float, T>(LoadNc(row + at)) : -INFINITY;
        }
    }
}

// Value of a key that came from a number.
__device__ __forceinline__ float ValueOf(uint32_t key) { return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key); }
constexpr uint32_t kMasked = 0x007fffffu;  // KeyOf(-inf)

__device__ __forceinline__ float Sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// Sorts a lane's keys, largest first (odd-even merge; VPL a power of two).
template <int VPL> __device__ __forceinline__ void SortDown(uint32_t (&key)[VPL])
{
#pragma unroll
    for (int p = 1; p < VPL; p <<= 1) {
#pragma unroll
        for (int q = p; q >= 1; q >>= 1) {
#pragma unroll
            for (int j = q % p; j + q < VPL; j += 2 * q) {
#pragma unroll
                for (int i = 0; i < q; ++i) {
                    if (j + i + q < VPL && (j + i) / (2 * p) == (j + i + q) / (2 * p)) {
                        const uint32_t a = key[j + i], b = key[j + i + q];
                        key[j + i] = max(a, b);
                        key[j + i + q] = min(a, b);
                    }
                }
            }
        }
    }
}

// Ranks the groups of a row by the sum of the `top` largest keys' values (keys themselves for top 1) and tells whether the
// lane's experts are in an open one.  `gap`: how far the worst open group is above the best closed one, less the errors of their scores:
// `margin` and 2^-22 of the magnitude of what is added up.
// A group of whole lanes, a power of two of them, is ranked by shuffles; other sizes go through shared memory.
template <int VPL>
__device__ __forceinline__ void CloseGroups(const RouteParams& p, uint32_t (&key)[VPL], uint32_t* row_keys, int lane, float margin, float& gap)
{
    const int size = p.experts / p.groups;
    const int lanes = size / VPL;
    const bool whole = size % VPL == 0 && (lanes & (lanes - 1)) == 0;
    uint32_t first = 0, second = 0;
    if (whole) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            second = max(second, min(first, key[j]));
            first = max(first, key[j]);
        }
        for (int d = 1; d < lanes; d <<= 1) {
            const uint32_t a = __shfl_xor_sync(kFull, first, d), b = __shfl_xor_sync(kFull, second, d);
            second = max(max(second, b), min(first, a));
            first = max(first, a);
        }
    } else {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            if (lane * VPL + j < p.experts) {
                row_keys[lane * VPL + j] = key[j];
            }
        }
        __syncwarp();
        if (lane < p.groups) {
            for (int i = 0; i < size; ++i) {
                const uint32_t v = row_keys[lane * size + i];
                second = max(second, min(first, v));
                first = max(first, v);
            }
        }
    }
    // Group g is at lane g * lanes (whole) or g.
    const int step = whole ? lanes : 1;
    const int mine = whole ? lane / lanes : lane;
    const uint32_t score = mine < p.groups ? (p.group_top == 2 ? KeyOf(ValueOf(first) + ValueOf(second)) : first) : 0u;
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
        const uint32_t other = __shfl_sync(kFull, score, g * step);
        ahead += (other > score || (other == score && g < mine)) ? 1 : 0;
    }
    const bool open = mine < p.groups && ahead < p.kept_groups;
    const float value = ValueOf(score);
    const float error = margin + (fabsf(ValueOf(first)) + (p.group_top == 2 ? fabsf(ValueOf(second)) : 0.0f)) * 0x1p-22f;
    const uint32_t worst = ~__reduce_max_sync(kFull, open ? ~KeyOf(value - error) : 0u);
    const uint32_t best = __reduce_max_sync(kFull, open || mine >= p.groups ? 0u : KeyOf(value + error));
    gap = best == 0 ? INFINITY : ValueOf(worst) - ValueOf(best);
    if (whole) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            key[j] = open ? key[j] : 0u;
        }
    } else {
        const unsigned set = __ballot_sync(kFull, open);
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const int at = lane * VPL + j;
            if (at < p.experts && !((set >> (at / size)) & 1u)) {
                key[j] = 0;
            }
        }
    }
}

// What the choice goes by, in 64 bits; `inverse`: 1 / the softmax's sum.
template <bool BIASED> __device__ __forceinline__ double FineScore(const RouteParams& p, float l, float base, double inverse)
{
    const double x = static_cast<double>(l);
    if constexpr (!BIASED) {
        return base == base ? x : static_cast<double>(NAN);  // scores order as the logits do
    }
    return p.softmax ? exp(x - static_cast<double>(base)) * inverse : 1.0 / (1.0 + exp(-x));
}

// The choice in 64 bits, for rows whose packed keys are too close to tell.  Lane i < k gets the i-th choice.  The
// keys live in shared memory (experts keys per warp), so that nothing of this weighs on the registers of the common path.
template <class T, bool BIASED>
__device__ __noinline__ void ChooseFine(const RouteParams& p, const T* row, const float* bias, float base, uint64_t* keys, int& chosen)
{
    const int lane = threadIdx.x & 31;
    double inverse = 1.0;
    if (BIASED && p.softmax) {
        double part = 0.0;
#pragma unroll 4
        for (int at = lane; at < p.experts; at += 32) {
            const float l = Widen<float, T>(LoadNc(row + at));
            part += l != -INFINITY ? exp(static_cast<double>(l) - static_cast<double>(base)) : 0.0;
        }
        inverse = 1.0 / WarpSum(part);
    }
    __syncwarp();
#pragma unroll 4
    for (int at = lane; at < p.experts; at += 32) {
        const float l = Widen<float, T>(LoadNc(row + at));
        double v = FineScore<BIASED>(p, l, base, inverse);
        if (bias != nullptr) {
            v += static_cast<double>(__ldg(bias + at));
        }
        keys[at] = KeyOf(l == -INFINITY ? -static_cast<double>(INFINITY) : v);
    }
    __syncwarp();
    if (p.groups > 1) {
        const int size = p.experts / p.groups;
        uint64_t mine = 0;
        if (lane < p.groups) {
            uint64_t first = 0, second = 0;
#pragma unroll 4
            for (int i = 0; i < size; ++i) {
                const uint64_t v = keys[lane * size + i];
                second = v > first ? first : (v > second ? v : second);
                first = v > first ? v : first;
            }
            mine = first;
            if (p.group_top == 2) {
                // back from keys to values; both are numbers or -inf
                const uint64_t a = (first >> 63) ? (first & 0x7fffffffffffffffULL) : ~first;
                const uint64_t b = (second >> 63) ? (second & 0x7fffffffffffffffULL) : ~second;
                mine = KeyOf(__longlong_as_double(static_cast<long long>(a)) + __longlong_as_double(static_cast<long long>(b)));
            }
        }
        int ahead = 0;
        for (int g = 0; g < p.groups; ++g) {
            const uint64_t other = __shfl_sync(kFull, mine, g);
            ahead += (other > mine || (other == mine && g < lane)) ? 1 : 0;
        }
        const unsigned open = __ballot_sync(kFull, lane < p.groups && ahead < p.kept_groups);
        __syncwarp();
        for (int at = lane; at < p.experts; at += 32) {
            if (!((open >> (at / size)) & 1u)) {
                keys[at] = 0;
            }
        }
        __syncwarp();
    }
    for (int i = 0; i < p.k; ++i) {
        uint64_t best = 0;
        int where = 0;
#pragma unroll 4
        for (int at = lane; at < p.experts; at += 32) {
            const uint64_t v = keys[at];
            where = v > best ? at : where;
            best = v > best ? v : best;
        }
        const uint64_t winner = WarpMax(best);
        const int at = static_cast<int>(__reduce_min_sync(kFull, best == winner ? static_cast<uint32_t>(where) : 0xffffffffu));
        if ((at & 31) == lane) {
            keys[at] = 0;
        }
        chosen = lane == i ? at : chosen;
        __syncwarp();
    }
}

// BIASED: the choice needs the scores themselves (a bias, or groups ranked by a sum of two); otherwise it compares logits.
//
// Every expert gets one 32-bit key that differs from all others: where it stands in the order, then its number, the lower first.
// Each step of the choice is one warp maximum (redux) and a pop from the winning lane's sorted keys.  Logits of 16 bits fit
// the key as they are.  Others are measured on a scale of 22 bits that reaches from the largest down to the smallest of the
// lanes' largest values, below which no k <= 31 winners lie, and neighbours in the resulting order that are too close to tell
// send the row to ChooseFine: closer than the scale's steps or, BIASED, than twice the error of the scores, unless they are
// equal by their inputs.  (4099 x 256, bias, 8 groups: 17.4 us with 32-bit keys and a search for the winner's lane, 13.4 us;
// about one row in 300 goes to ChooseFine.)
//
// BIASED scores are formed in fp32 with the fast exponential and division.  A sigmoid is off by at most 2^-22: its slope times
// the exponential's 2 + 1.16 |x| steps, an addition, a division.  A softmax is off by 2^-21 of its largest score, and the sum's
// error is shared; the bias adds 2^-24 of the result.  Only the sizes of scores that are compared count: a bias of -1e9 for one
// expert in five sends no more rows to ChooseFine than none does (65536 x 256, k 8: 70 and 69 us, 209 us when all sizes counted;
// eight groups 93 and 93 us, 297).  Where it leaves all experts of a lane and there are no groups, the scale reaches down to it and
// tells nothing apart: 211 us.
constexpr float kScale = 4194000.0f;

template <class T, int VPL, bool BIASED>
__global__ void __launch_bounds__(kWarps * 32) TopkKernel(RouteParams p, const T* __restrict__ logits, const float* __restrict__ bias,
                                                          T* __restrict__ weight, int64_t* __restrict__ index, bool wide)
{
    extern __shared__ __align__(16) unsigned char shared[];
    constexpr bool PACKED = sizeof(T) == 2 && !BIASED;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // The keys of a warp's row, needed across lanes only where groups are not whole lanes, and by ChooseFine.
    unsigned char* row_keys = shared + static_cast<size_t>(warp) * p.experts * (PACKED ? 4 : 8);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + warp; r < p.rows; r += static_cast<int64_t>(gridDim.x) * kWarps) {
        const T* row = logits + r * p.experts;
        float l[VPL];
        LoadRow<T, VPL>(row, p.experts, wide, lane, l);
        // A softmax over NaN or +inf has no finite value: the whole row is NaN, as torch.softmax has it.
        float top = -INFINITY;
        bool bad = false;
        if (p.softmax) {
            bool odd = false;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                top = fmaxf(top, l[j]);
                odd |= !(l[j] < INFINITY);
            }
            bad = __any_sync(kFull, odd);
            if (BIASED || !p.renormalize) {
                top = ValueOf(__reduce_max_sync(kFull, KeyOf(top)));
            }
        }

        // What the choice goes by, as order-preserving keys.
        uint32_t key[VPL];
        float margin = 0.0f;
        if constexpr (BIASED) {
            float c[VPL];
            if (p.softmax) {
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    c[j] = l[j] == -INFINITY ? 0.0f : __expf(l[j] - top);
                    part += c[j];
                }
                const float inverse = 1.0f / WarpSum(part);
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    c[j] *= inverse;
                }
                margin = inverse * 0x1p-19f;
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    c[j] = __fdividef(1.0f, 1.0f + __expf(-l[j]));
                }
                margin = 0x1p-20f;
            }
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int at = lane * VPL + j;
                if (bias != nullptr && at < p.experts) {
                    c[j] += __ldg(bias + at);
                }
                c[j] = l[j] == -INFINITY ? -INFINITY : (bad ? NAN : c[j]);
                key[j] = at < p.experts ? KeyOf(c[j]) : 0u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int at = lane * VPL + j;
                key[j] = KeyOf(bad ? -INFINITY : l[j]);
                if constexpr (PACKED) {
                    // the 16 bits of the logit, ordered, then the lower expert first
                    uint32_t bits;
                    if constexpr (std::is_same<T, __half>::value) {
                        const float v = bad || l[j] != l[j] ? -INFINITY : l[j] + 0.0f;
                        bits = __half_as_ushort(__float2half_rn(v));
                        bits = (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
                    } else {
                        bits = key[j] >> 16;  // bf16 is the upper half of fp32, and so is its order
                    }
                    key[j] = (bits << 16) | (0xffffu - static_cast<uint32_t>(at));
                }
                key[j] = at < p.experts ? key[j] : 0u;
            }
        }

        bool sure = true;
        if (p.groups > 1) {
            // (Packed keys rank a group by its best logit, ties to the lower group: the expert's number orders the same way.)
            float gap;
            CloseGroups<VPL>(p, key, reinterpret_cast<uint32_t*>(row_keys), lane, margin, gap);
            sure = !BIASED || gap > 0.0f;
        }

        const int steps = PACKED ? p.k : min(p.k + 3, 32);  // a few beyond the choice, to see that it is clear of them
        float units = 0.0f;                                 // of the scale: what tells two neighbours apart
        if constexpr (!PACKED) {
            uint32_t mine = 0;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                mine = max(mine, key[j]);
            }
            const uint32_t high = __reduce_max_sync(kFull, mine);
            uint32_t low = mine > kMasked ? mine : 0xffffffffu;
            if (__popc(__ballot_sync(kFull, mine > kMasked)) <= steps) {  // too few lanes: the smallest value of all
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    low = min(low, key[j] > kMasked ? key[j] : 0xffffffffu);
                }
            }
            low = __reduce_min_sync(kFull, low);
            const float floor = ValueOf(low), range = ValueOf(high) - floor;
            const float scale = high > kMasked && range > 0.0f ? kScale / range : 0.0f;
            // (the error of a sum with the bias goes by its size; what lies below the scale is not compared with what is on it)
            units = (BIASED ? margin + fmaxf(fabsf(ValueOf(high)), fabsf(floor)) * 0x1p-22f : 0.0f) * scale + 4.0f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                const int at = lane * VPL + j;
                // 0 closed, 1 masked or below the scale
                // (a range too small or too large for its scale makes it infinite or 0, and then every pair is open)
                const uint32_t place = key[j] >= low ? 2u + static_cast<uint32_t>(fminf((ValueOf(key[j]) - floor) * scale, kScale)) : 1u;
                key[j] = key[j] == 0u ? 0u : (place << 10) | (1023u - static_cast<uint32_t>(at));
            }
        }

        if constexpr (VPL <= 8) {
            SortDown<VPL>(key);
        }
        uint32_t head = key[0];
        if constexpr (VPL > 8) {
#pragma unroll
            for (int j = 1; j < VPL; ++j) {
                head = max(head, key[j]);
            }
        }
        uint32_t mine = 0;
        for (int i = 0; i < steps; ++i) {
            const uint32_t winner = __reduce_max_sync(kFull, head);
            mine = lane == i ? winner : mine;
            if (head == winner) {
                if constexpr (VPL <= 8) {
#pragma unroll
                    for (int j = 0; j + 1 < VPL; ++j) {
                        key[j] = key[j + 1];
                    }
                    key[VPL - 1] = 0;
                    head = key[0];
                } else {
                    head = 0;
#pragma unroll
                    for (int j = 0; j < VPL; ++j) {
                        head = max(head, key[j] < winner ? key[j] : 0u);
                    }
                }
            }
        }
        int chosen = 0;
        float chosen_logit = -INFINITY;
        if constexpr (PACKED) {
            if (lane < p.k) {
                chosen = static_cast<int>(0xffffu - (mine & 0xffffu));
                uint32_t bits = mine >> 16;
                bits = (bits & 0x8000u) ? (bits & 0x7fffu) : (~bits & 0xffffu);
                if constexpr (std::is_same<T, __half>::value) {
                    chosen_logit = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
                } else {
                    chosen_logit = __uint_as_float(bits << 16);
                }
                if (chosen_logit == -INFINITY) {  // the key of a masked expert is that of a NaN, too
                    chosen_logit = Widen<float, T>(LoadNc(row + chosen));
                }
            }
        } else {
            const uint32_t extra = __reduce_max_sync(kFull, head);  // the one after the last step
            uint32_t next = __shfl_down_sync(kFull, mine, 1);
            next = lane == steps - 1 ? extra : next;
            chosen = lane < steps && mine != 0 ? static_cast<int>(1023u - (mine & 1023u)) : 0;
            chosen_logit = lane < steps ? Widen<float, T>(LoadNc(row + chosen)) : 0.0f;
            // A pair of neighbours is clear (far apart, or the second masked: those go by their numbers), a tie (equal by
            // their inputs, the lower number first in every precision) or open.
            const bool pair = lane < steps && mine != 0;
            const bool clear = pair && ((next >> 10) <= 1u || static_cast<float>((mine >> 10) - (next >> 10)) > units);
            bool open = pair && !clear;
            if (__any_sync(kFull, open)) {
                const int other = static_cast<int>(1023u - (next & 1023u));
                if (open) {
                    const bool same = chosen_logit == Widen<float, T>(LoadNc(row + other));
                    open = !(same && (!BIASED || bias == nullptr || __ldg(bias + chosen) == __ldg(bias + other)));
                }
            }
            // All pairs within the choice are clear or ties; from its last one on, a clear pair comes before an open one.
            const unsigned opens = __ballot_sync(kFull, open), clears = __ballot_sync(kFull, clear);
            const unsigned behind = ~0u << (p.k - 1);
            const unsigned first = (opens | clears) & behind;
            sure = sure && (opens & ~behind) == 0 && (first & (0u - first) & clears) != 0;
            if (!sure) {
                ChooseFine<T, BIASED>(p, row, bias, bad ? NAN : top, reinterpret_cast<uint64_t*>(row_keys), chosen);
                chosen_logit = lane < p.k ? Widen<float, T>(LoadNc(row + chosen)) : 0.0f;
            }
        }

        // Weights.  A softmax renormalized over the chosen experts is the softmax of their logits.
        const bool taken = lane < p.k;
        float s = 0.0f, total = 1.0f;
        if (p.softmax) {
            float base = top;
            if (p.renormalize) {
                base = ValueOf(__reduce_max_sync(kFull, taken ? KeyOf(chosen_logit) : 0u));
            }
            s = taken && chosen_logit != -INFINITY ? expf(chosen_logit - base) : 0.0f;
            if (p.renormalize) {
                total = WarpSum(s);
            } else {
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    part += l[j] == -INFINITY ? 0.0f : expf(l[j] - top);
                }
                total = WarpSum(part);
            }
        } else {
            s = taken ? Sigmoid(chosen_logit) : 0.0f;
            total = p.renormalize ? WarpSum(s) : 1.0f;
        }
        if (p.undefined != nullptr && lane == 0) {
            p.undefined[r] = bad ? 1 : 0;
        }
        if (taken) {
            const float w = bad ? NAN : (total == 0.0f ? 0.0f : s / total * p.scale);
            weight[r * p.k + lane] = Narrow<T, float>(w);
            index[r * p.k + lane] = chosen;
        }
    }
}

// 16-bit logits without bias and groups, k <= 8, at most 256 experts: four rows per warp, eight lanes each.  A lane sorts its
// VPL packed keys eight at a time and merges the lists (of two sorted lists of eight, the eight largest are the pairwise
// maxima of one with the other reversed, a bitonic list), three more merges with its neighbours leave the row's eight largest in
// every lane; lane i then owns the i-th choice.  Per row a quarter of the instructions of the one-row-per-warp form, which
// is bound by them: 131072 x 128, k 8: 56 -> 31 us.
constexpr int kList = 8;

__device__ __forceinline__ void Exchange(uint32_t& a, uint32_t& b)
{
    const uint32_t high = max(a, b), low = min(a, b);
    a = high;
    b = low;
}
// list <- the eight largest of list and other (both descending), descending.
__device__ __forceinline__ void Merge(uint32_t (&list)[kList], const uint32_t (&other)[kList])
{
#pragma unroll
    for (int i = 0; i < kList; ++i) {
        list[i] = max(list[i], other[kList - 1 - i]);
    }
#pragma unroll
    for (int d = kList / 2; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < kList; ++i) {
            if ((i & d) == 0) {
                Exchange(list[i], list[i + d]);
            }
        }
    }
}

template <class T, int VPL>
__global__ void __launch_bounds__(kWarps * 32) TopkTeamKernel(RouteParams p, const T* __restrict__ logits, T* __restrict__ weight,
                                                              int64_t* __restrict__ index, bool wide)
{
    const int lane = threadIdx.x & 31, member = lane & 7;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * 4; r0 < p.rows; r0 += warps * 4) {
        const bool real = r0 + (lane >> 3) < p.rows;
        const int64_t r = real ? r0 + (lane >> 3) : r0;
        float l[VPL];
        LoadRow<T, VPL>(logits + r * p.experts, p.experts, wide, member, l);
        float top = -INFINITY;
        uint32_t odd = 0;
        if (p.softmax) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                odd |= l[j] < INFINITY ? 0u : 1u;
            }
            // NaN or +inf in a row makes it NaN
#pragma unroll
            for (int d = 4; d > 0; d >>= 1) {
                odd |= __shfl_xor_sync(kFull, odd, d);
            }
        }
        const bool bad = odd != 0;
        uint32_t list[kList];
#pragma unroll
        for (int first = 0; first < VPL; first += kList) {
            uint32_t key[kList];
#pragma unroll
            for (int j = 0; j < kList; ++j) {
                const int at = member * VPL + first + j;
                uint32_t bits;
                if constexpr (std::is_same<T, __half>::value) {
                    const float v = bad || l[first + j] != l[first + j] ? -INFINITY : l[first + j] + 0.0f;
                    bits = __half_as_ushort(__float2half_rn(v));
                    bits = (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
                } else {
                    bits = KeyOf(bad ? -INFINITY : l[first + j]) >> 16;
                }
                key[j] = at < p.experts ? (bits << 16) | (0xffffu - static_cast<uint32_t>(at)) : 0u;
            }
            SortDown<kList>(key);
            if (first == 0) {
#pragma unroll
                for (int j = 0; j < kList; ++j) {
                    list[j] = key[j];
                }
            } else {
                Merge(list, key);
            }
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            uint32_t other[kList];
#pragma unroll
            for (int j = 0; j < kList; ++j) {
                other[j] = __shfl_xor_sync(kFull, list[j], d);
            }
            Merge(list, other);
        }
        uint32_t mine = list[0];
#pragma unroll
        for (int j = 1; j < kList; ++j) {
            mine = member == j ? list[j] : mine;
        }
        const bool taken = member < p.k;
        const int chosen = taken ? static_cast<int>(0xffffu - (mine & 0xffffu)) : 0;
        auto value_of = [](uint32_t key) {
            uint32_t bits = key >> 16;
            bits = (bits & 0x8000u) ? (bits & 0x7fffu) : (~bits & 0xffffu);
            if constexpr (std::is_same<T, __half>::value) {
                return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
            } else {
                return __uint_as_float(bits << 16);
            }
        };
        float x = value_of(mine);
        if (taken && x == -INFINITY) {  // the key of a masked expert is that of a NaN, too
            x = Widen<float, T>(LoadNc(logits + r * p.experts + chosen));
        }
        float s, total = 1.0f;
        if (p.softmax) {
            top = value_of(list[0]);  // the row's largest logit, the first choice
            s = taken && x != -INFINITY ? expf(x - top) : 0.0f;
            if (p.renormalize) {
                total = TeamSum<8>(s);
            } else {
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    part += l[j] == -INFINITY ? 0.0f : expf(l[j] - top);
                }
                total = TeamSum<8>(part);
            }
        } else {
            s = taken ? Sigmoid(x) : 0.0f;
            total = p.renormalize ? TeamSum<8>(s) : 1.0f;
        }
        if (p.undefined != nullptr && member == 0 && real) {
            p.undefined[r] = bad ? 1 : 0;
        }
        if (taken && real) {
            const float w = bad ? NAN : (total == 0.0f ? 0.0f : s / total * p.scale);
            weight[r * p.k + member] = Narrow<T, float>(w);
            index[r * p.k + member] = chosen;
        }
    }
}

// LANES lanes per row: 8 where k and the row fit (four rows per warp), else 32.
template <class T, int VPL, int LANES>
__global__ void __launch_bounds__(kWarps * 32) TopkBackwardKernel(RouteParams p, const T* __restrict__ logits,
                                                                  const int64_t* __restrict__ index, const T* __restrict__ grad,
                                                                  T* __restrict__ grad_logits, bool wide)
{
    constexpr int ROWS = 32 / LANES;
    constexpr int VEC = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : VPL;
    const int lane = threadIdx.x & 31, member = lane % LANES;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * kWarps;
    for (int64_t r0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * ROWS; r0 < p.rows; r0 += warps * ROWS) {
        const bool real = r0 + lane / LANES < p.rows;
        const int64_t r = real ? r0 + lane / LANES : r0;
        const T* row = logits + r * p.experts;
        T* out = grad_logits + r * p.experts;
        const bool undefined = p.undefined != nullptr && __ldg(p.undefined + r) != 0;
        int64_t at = -1;
        float u = 0.0f, x = -INFINITY;
        if (member < p.k) {
            at = index[r * p.k + member];
            if (at >= 0 && at < p.experts) {
                u = Widen<float, T>(grad[r * p.k + member]) * p.scale;
                x = Widen<float, T>(row[at]);
            } else {
                at = -1;
            }
        }
        float value = 0.0f;   // gradient of the lane's chosen expert
        float spread = 0.0f;  // every other expert j gets -s_j * spread (softmax without renormalisation)
        float top = 0.0f, total = 1.0f;
        float l[VPL];
        if (p.softmax) {
            if (p.renormalize) {
                top = TeamMax<LANES>(at >= 0 ? x : -INFINITY);
                const float e = at < 0 || (x == -INFINITY && top == -INFINITY) ? 0.0f : expf(x - top);
                const float sum = TeamSum<LANES>(e);
                const float w = sum == 0.0f ? 0.0f : e / sum;
                const float mean = TeamSum<LANES>(u * w);
                value = w * (u - mean);
            } else {
                LoadRow<T, VPL>(row, p.experts, wide, member, l);
                top = -INFINITY;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    top = fmaxf(top, l[j]);
                }
                top = TeamMax<LANES>(top);
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    l[j] = l[j] == -INFINITY ? 0.0f : expf(l[j] - top);
                    part += l[j];
                }
                total = TeamSum<LANES>(part);
                total = total == 0.0f ? 0.0f : 1.0f / total;
                const float s = at < 0 || x == -INFINITY ? 0.0f : expf(x - top) * total;
                spread = TeamSum<LANES>(u * s);
                value = s * (u - spread);
            }
        } else {
            const float s = at < 0 ? 0.0f : Sigmoid(x);
            value = u * s * (1.0f - s);
            if (p.renormalize) {
                // (s / sum first: dividing by the sum alone overflows where scores are near the smallest number)
                const float sum = TeamSum<LANES>(s);
                const float w = sum == 0.0f ? 0.0f : s / sum;
                const float mean = TeamSum<LANES>(u * w);  // by every lane, also where the row's sum is 0 and its neighbours' are not
                value = w * (1.0f - s) * (u - mean);
            }
        }
        // The whole row first, the chosen experts over it: same warp, ordered by the barrier.
        const bool dense = p.softmax && !p.renormalize;
        if (wide) {
#pragma unroll
            for (int j = 0; j < VPL; j += VEC) {
                if (real && member * VPL + j < p.experts) {
                    float f[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        f[i] = dense ? -l[j + i] * total * spread : 0.0f;
                    }
                    *reinterpret_cast<Pack<T, VEC>*>(out + member * VPL + j) = Repack<T, float, VEC>(f);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                if (real && member * VPL + j < p.experts) {
                    out[member * VPL + j] = Narrow<T, float>(dense ? -l[j] * total * spread : 0.0f);
                }
            }
        }
        __syncwarp();
        if (real && at >= 0) {
            out[at] = Narrow<T, float>(value);
        }
        // A row without a softmax: the chosen experts of renormalised weights do not show it.
        if (__any_sync(kFull, undefined)) {
            __syncwarp();
            for (int j = undefined && real ? member : p.experts; j < p.experts; j += LANES) {
                out[j] = Narrow<T, float>(NAN);
            }
        }
    }
}

// The same for a backward pass that was not told which rows these are: NaN for the gradient of every row with a NaN or +inf.
template <class T>
__global__ void __launch_bounds__(kWarps * 32) UndefinedRowsKernel(RouteParams p, const T* __restrict__ logits, T* __restrict__ grad_logits)
{
    const int lane = threadIdx.x & 31;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); r < p.rows; r += static_cast<int64_t>(gridDim.x) * kWarps) {
        bool odd = false;
        for (int j = lane; j < p.experts; j += 32) {
            odd |= !(Widen<float, T>(LoadNc(logits + r * p.experts + j)) < INFINITY);
        }
        if (__any_sync(kFull, odd)) {
            for (int j = lane; j < p.experts; j += 32) {
                grad_logits[r * p.experts + j] = Narrow<T, float>(NAN);
            }
        }
    }
}

// ---- route_csr -----------------------------------------------------------------------------------------------------------
// Pairs (in the order they come) sorted by expert, stable: a counting sort in tiles of consecutive pairs, one thread block per
// tile.  A label outside [0, experts) is a dropped pair and counts in one more bin behind the last expert.
//   CountKernel  per tile: how many pairs of each bin                                  -> counts[bin][tile]
//   ScanKernel   per bin: exclusive prefix of its counts over the tiles, and its total -> counts, totals[bin]
//   PlaceKernel  per tile: where every bin starts (prefix of the totals), then every pair's place: bin start + pairs of the
//                bin in earlier tiles, in earlier warps of the tile, in earlier rounds of the warp, in lower lanes
// One tile needs the last kernel only.  No atomics on global memory; shared counters are per warp and commute.
// Bound by latency: three launches, and in the last a chain of counts, prefix and ranks.  1048576 pairs, 256 experts: 512 tiles
// of eight warps 21.9 us, one tile per SM of 32 warps 17.9 us (24.5 with the scan inside the last kernel, where every block reads
// all counts; 19.6 with perm sorted in shared memory before it is written); 512 pairs, 128 experts in one tile: 3.0 us with 16
// warps, 3.7 with 32.
constexpr int kMaxBins = 4096;
constexpr int kSortWarps = 32;

// Warps of a block: a table of bins each, which takes its time to clear and add up; a block on its own is done sooner with half
// as many.  1048576 pairs, 1500 experts: 35 us with 32 warps, 26 us with 16; 4000 experts: 48 us with eight.
inline int SortWarps(int bins, int64_t tiles) { return bins > 2000 ? 8 : (bins > 1000 || tiles == 1 ? kSortWarps / 2 : kSortWarps); }

template <class I> __device__ __forceinline__ int BinOf(const I* index, int64_t at, int64_t end, int experts)
{
    if (at >= end) {
        return -1;
    }
    const int64_t v = static_cast<int64_t>(__ldg(index + at));
    return v >= 0 && v < experts ? static_cast<int>(v) : experts;
}

template <class I>
__global__ void __launch_bounds__(1024) CountKernel(const I* __restrict__ index, int64_t count, int experts, int64_t tile,
                                                    int32_t* __restrict__ counts)
{
    extern __shared__ int32_t bins[];
    for (int b = threadIdx.x; b <= experts; b += blockDim.x) {
        bins[b] = 0;
    }
    __syncthreads();
    const int64_t first = blockIdx.x * tile, end = first + tile < count ? first + tile : count;
#pragma unroll 4
    for (int64_t at = first + threadIdx.x; at < end; at += blockDim.x) {
        atomicAdd(&bins[BinOf(index, at, end, experts)], 1);
    }
    __syncthreads();
    for (int b = threadIdx.x; b <= experts; b += blockDim.x) {
        counts[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = bins[b];
    }
}

// A warp per bin: its counts over the tiles become the pairs of the bin in earlier tiles, and their total.
__global__ void __launch_bounds__(256) ScanKernel(int32_t* __restrict__ counts, int bins, int tiles, int32_t* __restrict__ totals)
{
    const int lane = threadIdx.x & 31, bin = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (bin >= bins) {
        return;
    }
    int32_t* mine = counts + static_cast<int64_t>(bin) * tiles;
    int before = 0;
    for (int t0 = 0; t0 < tiles; t0 += 256) {
        int v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = t0 + i * 32 + lane;
            v[i] = t < tiles ? mine[t] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int inclusive = v[i];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(kFull, inclusive, d);
                inclusive += lane >= d ? up : 0;
            }
            const int t = t0 + i * 32 + lane;
            if (t < tiles) {
                mine[t] = before + inclusive - v[i];
            }
            before += __shfl_sync(kFull, inclusive, 31);
        }
    }
    if (lane == 0) {
        totals[bin] = before;
    }
}

// Exclusive prefix of v over the block, and its total.
__device__ __forceinline__ int BlockExclusive(int v, int* scratch, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int inclusive = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(kFull, inclusive, d);
        inclusive += lane >= d ? up : 0;
    }
    if (lane == 31) {
        scratch[warp] = inclusive;
    }
    __syncthreads();
    int sums = lane < warps ? scratch[lane] : 0;
    const int own = sums;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(kFull, sums, d);
        sums += lane >= d ? up : 0;
    }
    total = __shfl_sync(kFull, sums, 31);
    const int before = __shfl_sync(kFull, sums - own, warp);
    __syncthreads();
    return before + inclusive - v;
}

// Lanes with the same bin: one ballot per bit (match_any runs through the distinct values one by one, up to 32 of them).
__device__ __forceinline__ unsigned Peers(int bin, int bits)
{
    unsigned peers = __ballot_sync(kFull, bin >= 0);
    peers = bin >= 0 ? peers : ~peers;
    for (int i = 0; i < bits; ++i) {
        const bool set = (bin >> i) & 1;
        const unsigned with = __ballot_sync(kFull, set);
        peers &= set ? with : ~with;
    }
    return peers;
}

// Counts and places fit 32 bits: fewer than 2^31 pairs (checked on the host).
template <class I>
__global__ void __launch_bounds__(1024)
    PlaceKernel(const I* __restrict__ index, int64_t count, int experts, int64_t tile, const int32_t* __restrict__ counts,
                const int32_t* __restrict__ totals, int64_t* __restrict__ indptr, int64_t* __restrict__ perm, int64_t* __restrict__ position)
{
    extern __shared__ int32_t place[];  // [warps][experts + 1]: where the warp's next pair of a bin goes
    __shared__ int scratch[kSortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int bins = experts + 1;
    int32_t* mine = place + warp * bins;
    for (int b = threadIdx.x; b < bins * warps; b += blockDim.x) {
        place[b] = 0;
    }
    __syncthreads();
    // A warp takes consecutive pairs of the tile, 32 a round.
    const int64_t first = blockIdx.x * tile, end = first + tile < count ? first + tile : count;
    const int64_t share = ((tile + warps - 1) / warps + 31) / 32 * 32;
    const int64_t from = first + warp * share, to = from + share < end ? from + share : end;
#pragma unroll 4
    for (int64_t at = from + lane; at < to; at += 32) {
        atomicAdd(&mine[BinOf(index, at, to, experts)], 1);
    }
    __syncthreads();
    int before = 0;
    for (int b0 = 0; b0 < bins; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        int sum = 0, earlier = 0;
        if (b < bins) {
            if (counts != nullptr) {
                sum = totals[b];
                earlier = counts[static_cast<int64_t>(b) * gridDim.x + blockIdx.x];
            } else {
#pragma unroll 8
                for (int w = 0; w < warps; ++w) {
                    sum += place[w * bins + b];
                }
            }
        }
        int total;
        const int start = before + BlockExclusive(sum, scratch, total);
        before += total;
        if (b < bins) {
            if (blockIdx.x == 0) {
                indptr[b] = start;  // bin `experts` starts where the last expert ends
            }
            int next = start + earlier;
#pragma unroll 8
            for (int w = 0; w < warps; ++w) {
                const int here = place[w * bins + b];
                place[w * bins + b] = next;
                next += here;
            }
        }
    }
    __syncthreads();
    const int bits = 32 - __clz(experts);  // of the largest bin
    int next = BinOf(index, from + lane, to, experts);
    for (int64_t round = from; round < to; round += 32) {
        const int bin = next;
        next = BinOf(index, round + 32 + lane, to, experts);
        const unsigned peers = Peers(bin, bits);
        int where = 0;
        if (bin >= 0) {
            where = mine[bin] + __popc(peers & ((1u << lane) - 1u));
        }
        __syncwarp();
        if (bin >= 0) {
            if ((peers >> lane) == 1u) {  // the highest lane of the bin
                mine[bin] = where + 1;
            }
            perm[where] = round + lane;
            position[round + lane] = where;
        }
        __syncwarp();
    }
}

// Tiles: at most one per SM, of 1024 to 32768 pairs; of more pairs, 8192 each.  Long tiles write perm in so many far streams
// that sectors leave the cache half written: 8388608 pairs, 256 experts: 171 us with one tile per SM, 124 us with 1024 tiles
// (33554432: 1091 and 460), but 4194304 pairs 45 us with one tile per SM, 53 us with 512.
inline int64_t SortTiles(int64_t count)
{
    if (count <= 4096) {
        return 1;
    }
    const int64_t sms = SmCount();
    return count > sms * 32768 ? CeilDiv(count, 8192) : std::min<int64_t>(sms, CeilDiv(count, 1024));
}

constexpr int kMaxExperts = 1024;
constexpr int kMaxChosen = 32;
constexpr int kMaxGroups = 32;

int CheckRoute(const OpsgnnRouteDesc* d)
{
    if (d == nullptr || d->rows < 0 || d->experts < 1 || d->k < 1 || d->groups < 1 || d->kept_groups < 1 ||
        d->kept_groups > d->groups || d->experts % d->groups != 0 || (d->group_top != 1 && d->group_top != 2) ||
        (d->score != OPSGNN_ROUTE_SOFTMAX && d->score != OPSGNN_ROUTE_SIGMOID)) {
        return OPSGNN_ERR_INVALID;
    }
    const int64_t size = d->experts / d->groups;
    if (d->k > size * d->kept_groups || (d->groups > 1 && d->group_top > size)) {
        return OPSGNN_ERR_INVALID;
    }
    if (d->experts > kMaxExperts || d->k > kMaxChosen || d->groups > kMaxGroups) {
        return OPSGNN_ERR_LIMIT;
    }
    if (d->dtype != OPSGNN_F32 && d->dtype != OPSGNN_F16 && d->dtype != OPSGNN_BF16) {
        return OPSGNN_ERR_UNSUPPORTED;
    }
    return OPSGNN_OK;
}

RouteParams ParamsOf(const OpsgnnRouteDesc& d, uint8_t* undefined)
{
    RouteParams p;
    p.undefined = undefined;
    p.rows = d.rows;
    p.experts = static_cast<int32_t>(d.experts);
    p.k = static_cast<int32_t>(d.k);
    p.groups = static_cast<int32_t>(d.groups);
    p.kept_groups = static_cast<int32_t>(d.kept_groups);
    p.group_top = d.group_top;
    p.softmax = d.score == OPSGNN_ROUTE_SOFTMAX;
    p.renormalize = d.renormalize;
    p.scale = d.scale;
    return p;
}

int Grid(int64_t rows, int per_warp)
{
    return static_cast<int>(std::min<int64_t>(CeilDiv(rows, kWarps * per_warp), static_cast<int64_t>(SmCount()) * 16));
}

// Whole vectors: a lane's VPL values start on a vector boundary in every row.
template <class T, int VPL> bool Wide(int64_t experts, const void* a, const void* b)
{
    constexpr int VEC = VPL * sizeof(T) >= 16 ? 16 / sizeof(T) : VPL;
    return experts % VEC == 0 && Aligned(a, VEC * sizeof(T)) && Aligned(b, VEC * sizeof(T));
}

template <class T, int VPL>
int RunTopk(const OpsgnnRouteDesc& d, const void* logits, const float* bias, void* weight, int64_t* index, uint8_t* undefined,
            cudaStream_t stream)
{
    const RouteParams p = ParamsOf(d, undefined);
    const bool biased = bias != nullptr || (d.groups > 1 && d.group_top == 2);
    const T* in = static_cast<const T*>(logits);
    T* out = static_cast<T*>(weight);
    if constexpr (sizeof(T) == 2 && VPL <= 8) {
        if (!biased && d.groups == 1 && d.k <= kList) {
            constexpr int TEAM = VPL >= 2 ? 4 * VPL : 8;  // eight lanes hold what 32 do
            TopkTeamKernel<T, TEAM><<<Grid(d.rows, 4), kWarps * 32, 0, stream>>>(p, in, out, index, Wide<T, TEAM>(d.experts, in, in));
            return LaunchStatus();
        }
    }
    const bool wide = Wide<T, VPL>(d.experts, logits, logits);
    const bool packed = sizeof(T) == 2 && !biased;
    const size_t shared = !packed || d.groups > 1 ? static_cast<size_t>(kWarps) * d.experts * (packed ? 4 : 8) : 0;
    if (biased) {
        TopkKernel<T, VPL, true><<<Grid(d.rows, 1), kWarps * 32, shared, stream>>>(p, in, bias, out, index, wide);
    } else {
        TopkKernel<T, VPL, false><<<Grid(d.rows, 1), kWarps * 32, shared, stream>>>(p, in, bias, out, index, wide);
    }
    return LaunchStatus();
}

template <class T, int VPL>
int RunTopkBackward(const OpsgnnRouteDesc& d, const void* logits, const int64_t* index, const uint8_t* undefined, const void* grad,
                    void* grad_logits, cudaStream_t stream)
{
    const RouteParams p = ParamsOf(d, const_cast<uint8_t*>(undefined));
    const T* in = static_cast<const T*>(logits);
    const T* g = static_cast<const T*>(grad);
    T* out = static_cast<T*>(grad_logits);
    auto launched = [&]() {
        if (p.softmax && p.renormalize && undefined == nullptr) {
            UndefinedRowsKernel<T><<<Grid(d.rows, 1), kWarps * 32, 0, stream>>>(p, in, out);
        }
        return LaunchStatus();
    };
    if constexpr (VPL <= 8) {
        if (d.k <= 8) {
            TopkBackwardKernel<T, 4 * VPL, 8><<<Grid(d.rows, 4), kWarps * 32, 0, stream>>>(p, in, index, g, out,
                                                                                           Wide<T, 4 * VPL>(d.experts, in, out));
            return launched();
        }
    }
    TopkBackwardKernel<T, VPL, 32><<<Grid(d.rows, 1), kWarps * 32, 0, stream>>>(p, in, index, g, out,
                                                                              Wide<T, VPL>(d.experts, in, out));
    return launched();
}

// f(type tag, integral constant VPL): experts a lane of a warp holds, a power of two.
template <class F> int Dispatch(const OpsgnnRouteDesc& d, F&& f)
{
    auto by_width = [&](auto tag) {
        using std::integral_constant;
        if (d.experts <= 32) {
            return f(tag, integral_constant<int, 1>());
        }
        if (d.experts <= 64) {
            return f(tag, integral_constant<int, 2>());
        }
        if (d.experts <= 128) {
            return f(tag, integral_constant<int, 4>());
        }
        if (d.experts <= 256) {
            return f(tag, integral_constant<int, 8>());
        }
        if (d.experts <= 512) {
            return f(tag, integral_constant<int, 16>());
        }
        return f(tag, integral_constant<int, 32>());
    };
    switch (d.dtype) {
        case OPSGNN_F32:
            return by_width(float());
        case OPSGNN_F16:
            return by_width(__half());
        default:
            return by_width(__nv_bfloat16());
    }
}

}  // namespace route
}  // namespace opsgnn

using namespace opsgnn;

extern "C" int opsgnn_topk_route_recorded(const OpsgnnRouteDesc* desc, const void* logits, const float* bias, void* weight,
                                          int64_t* index, uint8_t* undefined, void* stream)
{
    const int status = route::CheckRoute(desc);
    if (status != OPSGNN_OK || desc->rows == 0) {
        return status;
    }
    if (logits == nullptr || weight == nullptr || index == nullptr) {
        return OPSGNN_ERR_INVALID;
    }
    return route::Dispatch(*desc, [&](auto tag, auto vpl) {
        return route::RunTopk<decltype(tag), decltype(vpl)::value>(*desc, logits, bias, weight, index, undefined, AsStream(stream));
    });
}

extern "C" int opsgnn_topk_route(const OpsgnnRouteDesc* desc, const void* logits, const float* bias, void* weight, int64_t* index,
                                 void* stream)
{
    return opsgnn_topk_route_recorded(desc, logits, bias, weight, index, nullptr, stream);
}

extern "C" int opsgnn_topk_route_backward_recorded(const OpsgnnRouteDesc* desc, const void* logits, const int64_t* index,
                                                   const uint8_t* undefined, const void* grad_weight, void* grad_logits, void* stream)
{
    const int status = route::CheckRoute(desc);
    if (status != OPSGNN_OK || desc->rows == 0) {
        return status;
    }
    if (logits == nullptr || index == nullptr || grad_weight == nullptr || grad_logits == nullptr) {
        return OPSGNN_ERR_INVALID;
    }
    return route::Dispatch(*desc, [&](auto tag, auto vpl) {
        return route::RunTopkBackward<decltype(tag), decltype(vpl)::value>(*desc, logits, index, undefined, grad_weight, grad_logits,
                                                                           AsStream(stream));
    });
}

extern "C" int opsgnn_topk_route_backward(const OpsgnnRouteDesc* desc, const void* logits, const int64_t* index, const void* grad_weight,
                                          void* grad_logits, void* stream)
{
    return opsgnn_topk_route_backward_recorded(desc, logits, index, nullptr, grad_weight, grad_logits, stream);
}

extern "C" int opsgnn_route_csr_workspace_bytes(int64_t count, int64_t experts, int64_t* bytes)
{
    if (bytes == nullptr || count < 0 || experts < 1) {
        return OPSGNN_ERR_INVALID;
    }
    if (experts > route::kMaxBins || count >= (INT64_C(1) << 31)) {
        return OPSGNN_ERR_LIMIT;
    }
    const int64_t tiles = route::SortTiles(count);
    *bytes = tiles > 1 ? (experts + 1) * (tiles + 1) * 4 : 0;
    return OPSGNN_OK;
}

extern "C" int opsgnn_route_csr(const void* index, int index_type, int64_t count, int64_t experts, int64_t* indptr, int64_t* perm,
                                int64_t* position, void* workspace, int64_t workspace_bytes, void* stream)
{
    int64_t need = 0;
    const int status = opsgnn_route_csr_workspace_bytes(count, experts, &need);
    if (status != OPSGNN_OK) {
        return status;
    }
    if (indptr == nullptr || (count > 0 && (index == nullptr || perm == nullptr || position == nullptr)) ||
        (index_type != OPSGNN_I32 && index_type != OPSGNN_I64)) {
        return OPSGNN_ERR_INVALID;
    }
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !Aligned(workspace, 8))) {
        return OPSGNN_ERR_WORKSPACE;
    }
    const int bins = static_cast<int>(experts) + 1;
    const int64_t tiles = route::SortTiles(count), tile = std::max<int64_t>(1, CeilDiv(count, tiles));
    int32_t* counts = tiles > 1 ? static_cast<int32_t*>(workspace) : nullptr;
    int32_t* totals = tiles > 1 ? counts + bins * tiles : nullptr;
    const int warps = route::SortWarps(bins, tiles);
    const int shared = warps * bins * 4;
    auto run = [&](auto tag) {
        using I = decltype(tag);
        const I* in = static_cast<const I*>(index);
        static std::atomic<uint64_t> allowed{0};
        OPSGNN_CUDA_TRY(static_cast<cudaError_t>(AllowShared(route::PlaceKernel<I>, 8 * (route::kMaxBins + 1) * 4, allowed)));
        if (tiles > 1) {
            route::CountKernel<I><<<static_cast<unsigned>(tiles), 1024, bins * 4, AsStream(stream)>>>(in, count, static_cast<int>(experts),
                                                                                                    tile, counts);
            route::ScanKernel<<<static_cast<unsigned>(CeilDiv(bins, 8)), 256, 0, AsStream(stream)>>>(counts, bins, static_cast<int>(tiles),
                                                                                                    totals);
        }
        route::PlaceKernel<I><<<static_cast<unsigned>(tiles), warps * 32, shared, AsStream(stream)>>>(
            in, count, static_cast<int>(experts), tile, counts, totals, indptr, perm, position);
        return LaunchStatus();
    };
    return index_type == OPSGNN_I32 ? run(int32_t()) : run(int64_t());
}
