// moe_route.cu -- routing of tokens to experts and the row plan of the grouped
// products (gemm_fp8_sm100.cu) that follow, and the routing weights' gradient.
//
//   s = softmax(l) or sigmoid(l) over a token's logits l; c = s + bias
//   the `top_groups` groups of experts with the largest sum of their two
//   largest c stay; of their experts the `top_k` largest c are chosen, ties to
//   the lowest index; w = scale * s (over the chosen ones' sum if renormalised)
//
// A logit of -inf or NaN (or a c of -inf or NaN) masks an expert: it is never
// chosen, and a slot that finds no expert gets id -1 and weight 0. Without a bias
// the experts' order is the logits' order, exactly. With one, or between groups,
// c is computed in f32 and compared; where two values that decide something lie
// closer than f32 can tell apart, the token is computed again in f64, so the
// choice is that of the definition in 64 bits at f32's cost for nearly all
// tokens.
//
// One warp per token, expert i * 32 + lane in register i. The plan is a stable
// counting sort of the slots by expert (tokens in order, so nothing depends on
// timing): counts per block of tokens, then every block sums the counts of the
// blocks before it and ranks its own slots. Few slots take one block and one
// launch.
//
// Bound by instruction issue (about 1400 a token at 256 experts in 8 groups with a
// bias and top_k 8, 600 without groups and bias): 16384 tokens take 47 to 51 us, 35
// of them the choice. 48 tokens of 64 experts take 9 us: one block, three tokens a
// warp one after another (the choice alone 6.5 us), then the plan. The gradient of
// 16383 x 160 softmax logits takes 11 us.
//
// Meant for up to 256 experts. Above, a lane holds 16 or 32 logits and the choice
// spills (its f64 form most): 16384 tokens, top_k 8, take 45 us at 512
// experts and 57 at 1024, with groups and a bias 103 and 150; 48 tokens 24 and 34 us;
// the softmax gradient of 16384 tokens 24 and 55 us.
#include <atomic>
#include <type_traits>

#include "gs_float.cuh"
#include "gs_fp8.h"

namespace gs {
namespace route {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPlanThreads = 1024;
// Threads of the kernel that only chooses: 32 warps hide the reductions' latency, where their registers allow it.
constexpr int choose_threads(int vpl) { return vpl >= 16 ? 512 : 1024; }
constexpr uint32_t kFull = 0xffffffffu;

// Order-preserving keys. -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double x) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
    return b ^ (static_cast<uint64_t>(static_cast<int64_t>(b) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __longlong_as_double(static_cast<long long>(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kFull, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(kFull, static_cast<uint32_t>(k >> 32));
    const uint32_t lo = __reduce_max_sync(kFull, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
// The choice's exponential and reciprocal: fast in f32, whose errors `doubt` allows for.
__device__ __forceinline__ float exp_of(float x) { return __expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float inverse(float x) { return __fdividef(1.0f, x); }
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }
template <typename R>
__device__ __forceinline__ R warp_sum(R v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
    return v;
}

constexpr float kTop = 3.402823466e38f;  // +inf counts as the largest finite value

// A token's logits, NaN and experts past the end as -inf.
template <typename T, int VPL>
__device__ __forceinline__ void load_row(const T *row, int experts, int lane, float (&l)[VPL]) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const int e = i * 32 + lane;
        float v = e < experts ? to_f32(row[e]) : -INFINITY;
        if (!(v >= -INFINITY)) v = -INFINITY;
        l[i] = fminf(v, kTop);
    }
}

template <int VPL>
__device__ __forceinline__ float row_top(const float (&l)[VPL]) {
    float top = l[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) top = fmaxf(top, l[i]);
    return value_of(warp_max(key_of(top)));
}
// Scores of all experts (masked ones: 0). top: softmax's largest logit.
template <typename R, int VPL>
__device__ __forceinline__ void scores(const float (&l)[VPL], bool sigmoid, float top, R (&s)[VPL]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            // f32: below -80 a sigmoid is 0 to within the doubt, and the fast quotient's range ends
            const R x = std::is_same<R, float>::value ? R(fmaxf(l[i], -80.0f)) : R(l[i]);
            s[i] = l[i] == -INFINITY ? R(0) : inverse(R(1) + exp_of(-x));
        }
        return;
    }
    R sum = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        s[i] = l[i] == -INFINITY ? R(0) : exp_of(R(l[i]) - R(top));
        sum += s[i];
    }
    sum = warp_sum(sum);
    const R inv = sum > R(0) ? R(1) / sum : R(0);
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] *= inv;
}

// Two best keys of the warp, from each lane's two best.
template <typename Key>
__device__ __forceinline__ void warp_top2(Key a1, Key a2, int lane, Key &m1, Key &m2) {
    m1 = warp_max(a1);
    const int owner = __ffs(__ballot_sync(kFull, a1 == m1)) - 1;
    m2 = warp_max(lane == owner ? a2 : a1);
}

// How far an f32 value of c may be from its exact value. Sigmoid: the fast exponential's (2 + 1.2 |x|) steps of 2^-23
// times the slope s (1 - s), at most 7e-8; two steps for the quotient and one for 1 + e, 3.1e-7. Softmax: s <= 1 times
// the sum's relative error, (2 + 1.2 ln 1024) steps of its terms and up to 37 additions, 4.1e-6. Then the sum with the
// bias, half a step of c.
__device__ __forceinline__ float doubt(const RouteDesc &d, float c) { return (d.sigmoid ? 5e-7f : 5e-6f) + 1e-7f * fabsf(c); }

// The top_k largest of the f32 keys, in order, to lanes 0 .. top_k - 1. At least top_k keys reach the top_k-th largest of
// the lanes' maxima, and usually only a few more do. Those (and, with a bias, the ones that may belong to them) are
// packed into `buf` (32 entries) and ranked against each other. Where neighbours are too close to call, each lane
// computes its candidate's c again in f64 and they are ranked by that.
// False if there are more than 32 candidates (many equal keys): the caller takes them one by one.
// About 220 instructions a token at 256 experts and top_k 8; taking the maximum top_k times costs 540.
template <int VPL>
__device__ __forceinline__ bool choose_sorted(const RouteDesc &d, const uint32_t (&key)[VPL], const float (&l)[VPL], float top, int lane,
                                              uint2 *buf, int &id) {
    const uint32_t none = key_of(-INFINITY);
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = max(m, key[i]);
#pragma unroll
    for (int size = 2; size <= 32; size *= 2) {  // bitonic, largest in lane 0
#pragma unroll
        for (int s = size / 2; s > 0; s /= 2) {
            const uint32_t o = __shfl_xor_sync(kFull, m, s);
            const bool up = ((lane & size) == 0) == ((lane & s) == 0);  // this lane keeps the larger
            m = up ? max(m, o) : min(m, o);
        }
    }
    uint32_t least = __shfl_sync(kFull, m, d.top_k - 1);
    if (d.bias != nullptr && least > none && value_of(least) < INFINITY) {
        const float v = value_of(least);
        least = key_of(v - 2.0f * doubt(d, v));
    }
    least = max(least, none + 1);
    int count = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        const bool in = key[i] >= least;
        const uint32_t who = __ballot_sync(kFull, in);
        const int at = count + __popc(who & ((1u << lane) - 1u));
        if (in && at < 32) buf[at] = make_uint2(key[i], static_cast<uint32_t>(i * 32 + lane));
        count += __popc(who);
    }
    if (count > 32) return false;
    __syncwarp();
    const uint2 own = lane < count ? buf[lane] : make_uint2(0u, ~0u);
    int rank = 0;
    bool near = false;
    const float c = value_of(own.x), reach = 2.0f * doubt(d, c);
    for (int x = 0; x < count; ++x) {
        const uint2 other = buf[x];
        rank += other.x > own.x || (other.x == own.x && other.y < own.y) ? 1 : 0;
        near |= x != lane && fabsf(value_of(other.x) - c) <= reach;
    }
    near = near && lane < count && rank <= d.top_k;
    if (d.bias != nullptr && __any_sync(kFull, near)) {
        double total = 0.0;
        if (!d.sigmoid) {
#pragma unroll 1
            for (int q = 0; q < VPL; ++q) {  // one copy of the f64 exponential: the register is picked by comparison
                float v = -INFINITY;
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (i == q) v = l[i];
                total += v == -INFINITY ? 0.0 : exp(static_cast<double>(v) - static_cast<double>(top));
            }
            total = warp_sum(total);
        }
        float x_own = 0.0f;  // the candidate's logit, from the lane that holds it
#pragma unroll
        for (int q = 0; q < VPL; ++q) {
            const float v = __shfl_sync(kFull, l[q], own.y & 31u);
            if (q == static_cast<int>(own.y >> 5)) x_own = v;
        }
        double exact = 0.0;
        uint64_t k64 = 0;
        if (lane < count) {
            const int e = static_cast<int>(own.y);
            const double v = x_own;
            exact = (d.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - static_cast<double>(top)) / total) + static_cast<double>(d.bias[e]);
            k64 = key_of(exact);
        }
        rank = 0;
        for (int x = 0; x < count; ++x) {
            const uint64_t other = __shfl_sync(kFull, k64, x);
            const uint32_t e = __shfl_sync(kFull, own.y, x);
            rank += other > k64 || (other == k64 && e < own.y) ? 1 : 0;
        }
    }
    __syncwarp();
    if (lane < count) buf[rank] = own;
    __syncwarp();
    if (lane < d.top_k && lane < count) id = static_cast<int>(buf[lane].y);
    return true;
}

// Chooses a token's experts: lane j < top_k gets the j-th id, or -1. Returns false if f32 values that decide something
// are too close to call.
template <typename R, int VPL>
__device__ __forceinline__ bool choose(const RouteDesc &d, const float (&l)[VPL], float top, int lane, uint2 *buf, int &id) {
    using Key = decltype(key_of(R(0)));
    constexpr bool F32 = std::is_same<R, float>::value;
    const Key none = key_of(R(-INFINITY));
    const bool grouped = d.groups > 1 && d.top_groups < d.groups;
    Key key[VPL];
    bool close = false;
    auto far = [&](float x, float y) { return !(fabsf(x - y) <= 2.0f * doubt(d, x)); };
    if (d.bias != nullptr || grouped) {
        R s[VPL];
        scores<R, VPL>(l, d.sigmoid != 0, top, s);
        Key ck[VPL];  // by c, which is what groups compare
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = i * 32 + lane;
            R c = s[i];
            if (d.bias != nullptr) c += e < d.experts ? R(d.bias[e]) : R(0);
            ck[i] = l[i] == -INFINITY || !(c > R(-INFINITY)) ? none : key_of(c);
            key[i] = d.bias != nullptr ? ck[i] : key_of(R(l[i]));
        }
        if (grouped) {
            const int size = d.group_size;
            Key k1 = none, k2 = none;  // lane g: group g's two best
            auto record = [&](Key a1, Key a2, int g) {
                Key m1, m2;
                warp_top2(a1, a2, lane, m1, m2);
                if (lane == g) { k1 = m1; k2 = m2; }
            };
            if (size == 32) {  // a group is a register
#pragma unroll
                for (int i = 0; i < VPL; ++i) record(ck[i], none, i);
            } else {
                for (int g = 0; g < d.groups; ++g) {
                    Key a1 = none, a2 = none;
#pragma unroll
                    for (int i = 0; i < VPL; ++i) {
                        const Key k = static_cast<int>((static_cast<uint32_t>(i * 32 + lane) * d.group_magic) >> 20) == g ? ck[i] : none;
                        if (k > a1) { a2 = a1; a1 = k; }
                        else if (k > a2) a2 = k;
                    }
                    record(a1, a2, g);
                }
            }
            const R c1 = value_of(k1), c2 = k2 != none ? value_of(k2) : R(0);
            const Key mine = k1 == none ? none : key_of(c1 + c2);
            int better = 0;
            for (int g = 0; g < d.groups; ++g) {
                const Key other = __shfl_sync(kFull, mine, g);
                better += other > mine || (other == mine && g < lane) ? 1 : 0;
            }
            const bool kept = lane < d.groups && better < d.top_groups;
            if constexpr (F32) {
                // How far the sum may be off: by its two terms' scores, and by half a step (6e-8 of it) of each c, of the
                // sum and of its limit, none of them larger than |c1| + |c2|, however small the sum is. The least that a
                // kept group may have has to pass the most that another may. A sum beyond f32's range may be anything
                // (its limits are NaN, or infinite).
                const bool live = k1 != none;
                const float sum = c1 + c2, reach = 2.0f * doubt(d, 0.0f) + 2e-7f * (fabsf(c1) + fabsf(c2));
                const Key worst = ~warp_max(kept && live ? ~key_of(fmaxf(sum - reach, -INFINITY)) : Key(0));
                const Key best = warp_max(!kept && live ? key_of(fminf(sum + reach, INFINITY)) : Key(0));
                if (best >= worst) close = true;
            }
            const uint32_t keep = __ballot_sync(kFull, kept);
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const uint32_t g = size == 32 ? static_cast<uint32_t>(i) : (static_cast<uint32_t>(i * 32 + lane) * d.group_magic) >> 20;
                if (g >= 32 || !((keep >> g) & 1u) || ck[i] == none) key[i] = none;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) key[i] = key_of(R(l[i]));
    }
    id = -1;
    if constexpr (F32) {
        if (!close && choose_sorted<VPL>(d, key, l, top, lane, buf, id)) return true;
    }
    Key last = none;
    Key best = none;  // this lane's best and its register
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
        if (key[i] > best) { best = key[i]; at = i; }
    for (int j = 0; j <= d.top_k; ++j) {  // one more than chosen, for the distance to the first that is not
        if (j == d.top_k && !(F32 && d.bias != nullptr)) break;
        const Key m = warp_max(best);
        if (m == none) break;
        if constexpr (F32) {
            if (d.bias != nullptr && j > 0 && !far(value_of(last), value_of(m))) close = true;
        }
        if (j == d.top_k) break;
        last = m;
        const uint32_t holders = __ballot_sync(kFull, best == m);
        uint32_t e;
        if ((holders & (holders - 1)) == 0) {
            const int owner = __ffs(holders) - 1;
            e = static_cast<uint32_t>(__shfl_sync(kFull, at, owner) * 32 + owner);
        } else {  // a tie: the lowest expert
            e = __reduce_min_sync(kFull, best == m ? static_cast<uint32_t>(at * 32 + lane) : ~0u);
        }
        if (lane == j) id = static_cast<int>(e);
        if (lane == static_cast<int>(e & 31u)) {
            best = none;
            const int gone = at;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                if (i == gone) key[i] = none;
                if (key[i] > best) { best = key[i]; at = i; }
            }
        }
    }
    return !close;
}

template <int VPL>
__device__ __noinline__ int choose_exactly(const RouteDesc &d, const float (&l)[VPL], float top, int lane) {
    int id;
    choose<double, VPL>(d, l, top, lane, nullptr, id);
    return id;
}

// Chooses and writes one token's ids and weights; returns lane j's id.
template <typename T, int VPL>
__device__ __forceinline__ int route_token(const RouteDesc &d, int t, int live, int lane, uint2 *buf) {
    int id = -1;
    float w = 0.0f;
    if (t < live) {
        const T *row = static_cast<const T *>(d.logits) + static_cast<long long>(t) * d.ld;
        float l[VPL];
        load_row<T, VPL>(row, d.experts, lane, l);
        const float top = d.sigmoid ? 0.0f : row_top(l);
        if (!choose<float, VPL>(d, l, top, lane, buf, id)) {
            float again[VPL];  // a copy of its own: l stays in registers
#pragma unroll
            for (int i = 0; i < VPL; ++i) again[i] = l[i];
            id = choose_exactly<VPL>(d, again, top, lane);
        }
        // The chosen ones' scores, one a lane.
        const float x = id >= 0 ? fminf(to_f32(row[id]), kTop) : -INFINITY;
        if (d.sigmoid) {
            w = 1.0f / (1.0f + expf(-x));
        } else {
            w = id >= 0 ? expf(x - top) : 0.0f;
            if (!d.renorm) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) sum += l[i] == -INFINITY ? 0.0f : expf(l[i] - top);
                sum = warp_sum(sum);
                w = sum > 0.0f ? w / sum : 0.0f;
            }
        }
        if (d.renorm) {
            const float sum = warp_sum(w);
            if (sum >= 1e-30f) {
                w = w / sum;
            } else {  // all far below f32's range, or none: as the definition in 64 bits
                double v = 0.0;
                if (id >= 0) v = d.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - static_cast<double>(top));
                const double all = warp_sum(v);
                w = all > 0.0 ? static_cast<float>(v / all) : 0.0f;
            }
        }
        w *= d.scale;
    }
    if (lane < d.top_k) {
        const long long at = static_cast<long long>(t) * d.top_k + lane;
        d.ids[at] = id;
        d.weights[at] = id < 0 ? 0.0f : w;
    }
    return id;
}

// Exclusive sums over the experts of their aligned counts: base[e] = first row of expert e, base[experts] = all rows.
// Called by the whole block; `count` and `base` in shared memory.
template <int THREADS>
__device__ void expert_bases(const int *count, int *base, int experts, int align) {
    for (int e = threadIdx.x; e < experts; e += THREADS) base[e] = align == 1 ? count[e] : (count[e] + align - 1) / align * align;
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, per = (experts + 31) / 32;
        const int lo = min(lane * per, experts), hi = min(lo + per, experts);
        int sum = 0;
        for (int e = lo; e < hi; ++e) sum += base[e];
        int incl = sum;
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += v;
        }
        int at = incl - sum;
        for (int e = lo; e < hi; ++e) {
            const int n = base[e];
            base[e] = at;
            at += n;
        }
        if (lane == 31) base[experts] = incl;
    }
    __syncthreads();
}

// Slots [lo, hi) of a block, a run of whole 32s to a warp: this warp's run.
template <int THREADS>
__device__ __forceinline__ void warp_run(long long lo, long long hi, long long &a, long long &b) {
    const long long per = ((hi - lo + THREADS / 32 - 1) / (THREADS / 32) + 31) / 32 * 32;
    a = min(lo + (threadIdx.x >> 5) * per, hi);
    b = min(a + per, hi);
}

// Rows of slots [lo, hi) of this block: next[w * ld + e] first counts warp w's slots of expert e, then becomes the row of
// its next one. `first` gives each expert's first row for this block; `ahead` is this thread's id of its warp's first 32.
template <int THREADS>
__device__ void rank_slots(const RouteDesc &d, const int *ids, long long lo, long long hi, int *next, const int *first, int experts, int ahead) {
    constexpr int WARPS = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ld = experts | 1;  // odd: an expert's counters lie in different banks
    long long a, b;
    warp_run<THREADS>(lo, hi, a, b);
    for (int i = threadIdx.x; i < WARPS * ld; i += THREADS) next[i] = 0;
    __syncthreads();
    for (long long i = a; i < b; i += 32) {
        const int e = i == a ? ahead : i + lane < b ? ids[i + lane - lo] : -1;
        const uint32_t same = __match_any_sync(kFull, e);
        if (e >= 0 && lane == __ffs(same) - 1) next[warp * ld + e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int e = warp; e < experts; e += WARPS) {  // a warp sums an expert's counters, one a lane
        const int n = lane < WARPS ? next[lane * ld + e] : 0;
        int incl = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += v;
        }
        if (lane < WARPS) next[lane * ld + e] = first[e] + incl - n;
    }
    __syncthreads();
    for (long long i = a; i < b; i += 32) {
        const int e = i == a ? ahead : i + lane < b ? ids[i + lane - lo] : -1;
        const uint32_t same = __match_any_sync(kFull, e);
        int row = -1;
        if (e >= 0) row = next[warp * ld + e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && lane == __ffs(same) - 1) next[warp * ld + e] += __popc(same);
        __syncwarp();
        if (i + lane < b) {
            d.slot_row[i + lane] = row;
            if (row >= 0 && row < d.rows) d.row_slot[row] = static_cast<int32_t>(i + lane);
        }
    }
}

// Rows that hold no slot: the padding behind an expert's rows, and the rows behind the last expert.
template <int THREADS>
__device__ void fill_padding(const RouteDesc &d, const int *count, const int *base, int block, int blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (d.align > 1)
        for (int e = block * (THREADS / 32) + warp; e < d.experts; e += blocks * (THREADS / 32))
            for (int r = base[e] + count[e] + lane; r < min(base[e + 1], d.rows); r += 32) d.row_slot[r] = -1;
    for (long long r = base[d.experts] + static_cast<long long>(block) * THREADS + threadIdx.x; r < d.rows;
         r += static_cast<long long>(blocks) * THREADS)
        d.row_slot[r] = -1;
}

constexpr int kSmallSlots = 1024;

// All in one block: few slots.
template <typename T, int VPL>
__global__ void __launch_bounds__(kThreads) k_route_small(const __grid_constant__ RouteDesc d) {
    extern __shared__ int sm[];
    __shared__ int ids[kSmallSlots];
    __shared__ uint2 buf[kWarps * 32];
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int live = d.token_count != nullptr ? *d.token_count : d.tokens;
    for (int t = warp; t < d.tokens; t += kWarps) {
        const int id = route_token<T, VPL>(d, t, live, lane, buf + warp * 32);
        if (lane < d.top_k) ids[t * d.top_k + lane] = id;
    }
    if (d.offsets == nullptr) return;
    int *count = sm, *base = sm + d.experts, *next = base + d.experts + 1;
    for (int e = threadIdx.x; e < d.experts; e += kThreads) count[e] = 0;
    __syncthreads();
    const int slots = d.tokens * d.top_k;
    for (int i = threadIdx.x; i < slots; i += kThreads)
        if (ids[i] >= 0) atomicAdd(&count[ids[i]], 1);  // whole numbers: any order gives the same sum
    __syncthreads();
    expert_bases<kThreads>(count, base, d.experts, d.align);
    for (int e = threadIdx.x; e <= d.experts; e += kThreads) d.offsets[e] = base[e];
    long long a, b;
    warp_run<kThreads>(0, slots, a, b);
    rank_slots<kThreads>(d, ids, 0, slots, next, base, d.experts, a + lane < b ? ids[a + lane] : -1);
    fill_padding<kThreads>(d, count, base, 0, 1);
}

// Many slots, first kernel: the choice, and the block's count of every expert.
template <typename T, int VPL>
__global__ void __launch_bounds__(choose_threads(VPL)) k_route_choose(const __grid_constant__ RouteDesc d, int per_block) {
    constexpr int THREADS = choose_threads(VPL);
    extern __shared__ int sm[];
    __shared__ uint2 buf[THREADS];
    grid_dep_wait();
    grid_dep_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int live = d.token_count != nullptr ? *d.token_count : d.tokens;
    const bool plan = d.offsets != nullptr;
    if (plan) {
        for (int e = threadIdx.x; e < d.experts; e += THREADS) sm[e] = 0;
        __syncthreads();
    }
    const long long lo = static_cast<long long>(blockIdx.x) * per_block;
    const int hi = static_cast<int>(min(lo + per_block, static_cast<long long>(d.tokens)));
    for (int t = static_cast<int>(min(lo, static_cast<long long>(hi))) + warp; t < hi; t += THREADS / 32) {
        const int id = route_token<T, VPL>(d, t, live, lane, buf + warp * 32);
        if (plan && id >= 0) atomicAdd(&sm[id], 1);
    }
    if (plan) {
        __syncthreads();
        for (int e = threadIdx.x; e < d.experts; e += THREADS) d.hist[static_cast<long long>(blockIdx.x) * d.experts + e] = sm[e];
    }
}

// Second kernel: every block sums the counts (all, and of the blocks before it), then ranks its slots.
__global__ void __launch_bounds__(kPlanThreads) k_route_plan(const __grid_constant__ RouteDesc d, int per_block) {
    extern __shared__ int sm[];
    grid_dep_wait();
    grid_dep_launch();
    const int experts = d.experts;
    int *count = sm, *before = count + experts, *base = before + experts, *next = base + experts + 1;
    const long long slots = static_cast<long long>(d.tokens) * d.top_k;
    const long long lo = min(static_cast<long long>(blockIdx.x) * per_block * d.top_k, slots);
    const long long hi = min(lo + static_cast<long long>(per_block) * d.top_k, slots);
    long long a, b;
    warp_run<kPlanThreads>(lo, hi, a, b);
    const int ahead = a + static_cast<int>(threadIdx.x & 31) < b ? d.ids[a + (threadIdx.x & 31)] : -1;  // while the counts come in
    for (int i = threadIdx.x; i < 2 * experts; i += kPlanThreads) sm[i] = 0;
    __syncthreads();
    // Each block begins at its own row, so that they do not all read the same lines at once.
    const int blocks = gridDim.x, self = static_cast<int>(blockIdx.x);
    if (experts % 4 == 0 && reinterpret_cast<uintptr_t>(d.hist) % 16 == 0) {  // four experts to a thread
        const int quads = experts / 4, parts = kPlanThreads / quads;  // experts <= 1024
        const int e = threadIdx.x % quads, part = threadIdx.x / quads;
        if (part < parts) {
            int4 all = make_int4(0, 0, 0, 0), mine = make_int4(0, 0, 0, 0);
            const int4 *hist = reinterpret_cast<const int4 *>(d.hist) + e;
#pragma unroll 8
            for (int x = part; x < blocks; x += parts) {
                const int b = x + self < blocks ? x + self : x + self - blocks;
                const int4 n = hist[b * quads];  // at most 148 x 256
                all.x += n.x; all.y += n.y; all.z += n.z; all.w += n.w;
                if (b < self) { mine.x += n.x; mine.y += n.y; mine.z += n.z; mine.w += n.w; }
            }
            atomicAdd(&count[4 * e], all.x); atomicAdd(&count[4 * e + 1], all.y);
            atomicAdd(&count[4 * e + 2], all.z); atomicAdd(&count[4 * e + 3], all.w);
            atomicAdd(&before[4 * e], mine.x); atomicAdd(&before[4 * e + 1], mine.y);
            atomicAdd(&before[4 * e + 2], mine.z); atomicAdd(&before[4 * e + 3], mine.w);
        }
    } else {
        const int parts = max(1, kPlanThreads / experts);
        for (int i = threadIdx.x; i < experts * parts; i += kPlanThreads) {
            const int e = i % experts, part = i / experts;
            int all = 0, mine = 0;
#pragma unroll 8
            for (int x = part; x < blocks; x += parts) {
                const int b = x + self < blocks ? x + self : x + self - blocks;
                const int n = d.hist[b * experts + e];
                all += n;
                if (b < self) mine += n;
            }
            atomicAdd(&count[e], all);
            atomicAdd(&before[e], mine);
        }
    }
    __syncthreads();
    expert_bases<kPlanThreads>(count, base, experts, d.align);
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e <= experts; e += kPlanThreads) d.offsets[e] = base[e];
    for (int e = threadIdx.x; e < experts; e += kPlanThreads) before[e] += base[e];
    __syncthreads();
    rank_slots<kPlanThreads>(d, d.ids + lo, lo, hi, next, before, experts, ahead);
    fill_padding<kPlanThreads>(d, count, base, blockIdx.x, blocks);
}

// Dynamic shared memory of the kernels that make a plan: count, bases and every warp's counters; the plan kernel's own
// counts besides.
constexpr size_t plan_bytes(bool small, int experts) {
    return (static_cast<size_t>(experts | 1) * (small ? kWarps : kPlanThreads / 32) + static_cast<size_t>(experts) * (small ? 2 : 3) + 1) * sizeof(int);
}

// Opts `kern` in to the most shared memory that any of its calls needs, once per device: the limit is the kernel's for
// all threads, so one that followed each call's size would change between another thread's setting and its launch.
// `done` is the kernel's own.
template <typename K>
static cudaError_t allow_shared(Context &ctx, K kern, size_t most, std::atomic<bool> (&done)[64]) {
    const bool known = ctx.device >= 0 && ctx.device < 64;
    if (most <= 32 * 1024 || (known && done[ctx.device].load(std::memory_order_relaxed))) return cudaSuccess;  // with the static arrays within the 48 KiB that need no opt-in
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
    if (e == cudaSuccess && known) done[ctx.device].store(true, std::memory_order_relaxed);
    return e;
}

template <typename T, int VPL>
static cudaError_t launch(Context &ctx, const RouteDesc &d) {
    static std::atomic<bool> small_set[64], plan_set[64];
    const int blocks = route_blocks(d.tokens, d.top_k);
    const size_t smem = d.offsets != nullptr ? plan_bytes(blocks == 0, d.experts) : 0;
    if (blocks == 0) {
        cudaError_t e = allow_shared(ctx, k_route_small<T, VPL>, plan_bytes(true, VPL * 32), small_set);
        if (e != cudaSuccess) return e;
        e = launch_pdl(k_route_small<T, VPL>, dim3(1), dim3(kThreads), smem, ctx.stream, 1, d);
        ctx.launches++;
        return e;
    }
    const int per = (d.tokens + blocks - 1) / blocks;
    cudaError_t e = launch_pdl(k_route_choose<T, VPL>, dim3(static_cast<unsigned>(blocks)), dim3(choose_threads(VPL)),
                               static_cast<size_t>(d.experts) * sizeof(int), ctx.stream, 1, d, per);
    ctx.launches++;
    if (e != cudaSuccess || d.offsets == nullptr) return e;
    e = allow_shared(ctx, k_route_plan, plan_bytes(false, GS_ROUTE_MAX_EXPERTS), plan_set);
    if (e != cudaSuccess) return e;
    e = launch_pdl(k_route_plan, dim3(static_cast<unsigned>(blocks)), dim3(kPlanThreads), smem, ctx.stream, 1, d, per);
    ctx.launches++;
    return e;
}

// Gradient of the weights with respect to the logits; the choice is constant.
//   renormalised: dl_j = w_j (g_j - sum g w), times 1 - s_j for sigmoid; experts that were not chosen get 0
//   otherwise dl = J^T g: g_j s_j (1 - s_j), or s_e ([e chosen] g_e - sum g s)
// Bound by writing dlogits (and, for softmax that is not renormalised, reading the logits).
template <typename T, typename TD, int VPL>
__global__ void __launch_bounds__(256) k_route_backward(const __grid_constant__ RouteBwdDesc d) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    for (long long t = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); t < d.tokens; t += static_cast<long long>(gridDim.x) * 8) {
        const T *logits = static_cast<const T *>(d.logits) + t * d.ld;
        const bool every = !d.renorm && !d.sigmoid;  // softmax that is not renormalised: every logit has a gradient
        float l[VPL];
        if (every) load_row<T, VPL>(logits, d.experts, lane, l);  // on its way while the ids come in
        int id = -1;
        float g = 0.0f, x = -INFINITY;  // lane j: the j-th chosen expert, its weight's gradient and its logit
        if (lane < d.top_k) {
            id = d.ids[t * d.top_k + lane];
            if (id < 0 || id >= d.experts) {
                id = -1;
            } else {
                g = d.dweights[t * d.top_k + lane] * d.scale;
                x = to_f32(logits[id]);
                x = x >= -INFINITY ? fminf(x, kTop) : -INFINITY;
            }
        }
        // slope: what chosen expert j's own logit gets; common: what every logit gets, times its score (softmax that is
        // not renormalised: the one case that needs the other experts' logits)
        float s[VPL], slope, common = 0.0f;
        if (d.renorm) {
            // Weights from the logits' differences, or from the sigmoids unless all of them are below f32's range (where a
            // sigmoid is an exponential).
            float v = d.sigmoid ? 1.0f / (1.0f + expf(-x)) : 0.0f;
            float sum = warp_sum(v);
            if (!(sum >= 1e-30f)) {
                const float most = value_of(warp_max(key_of(x)));
                v = id >= 0 && x > -INFINITY ? expf(x - most) : 0.0f;
                sum = warp_sum(v);
            }
            const float w = sum > 0.0f ? v / sum : 0.0f;
            slope = w * (g - warp_sum(g * w));
            if (d.sigmoid) slope *= 1.0f / (1.0f + expf(x));
        } else if (d.sigmoid) {
            slope = g / (1.0f + expf(-x)) * (1.0f / (1.0f + expf(x)));
        } else {
            const float top = row_top(l);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                s[i] = l[i] == -INFINITY ? 0.0f : expf(l[i] - top);
                sum += s[i];
            }
            sum = warp_sum(sum);
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) s[i] *= inv;
            slope = id >= 0 && x > -INFINITY ? g * (expf(x - top) * inv) : 0.0f;
            common = warp_sum(slope);
        }
        if (id < 0) slope = 0.0f;
        float out[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) out[i] = every ? -common * s[i] : 0.0f;
        for (int j = 0; j < d.top_k; ++j) {
            const int e = __shfl_sync(kFull, id, j);
            const float v = __shfl_sync(kFull, slope, j);
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (e >= 0 && e == i * 32 + lane) out[i] += v;
        }
        TD *row = static_cast<TD *>(d.dlogits) + t * d.ldd;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (i * 32 + lane < d.experts) row[i * 32 + lane] = from_f32<TD>(out[i]);
    }
}

// Registers per lane for a number of experts (at most 1024).
template <typename F>
static cudaError_t with_vpl(int experts, F f) {
    if (experts <= 32) return f(std::integral_constant<int, 1>{});
    if (experts <= 64) return f(std::integral_constant<int, 2>{});
    if (experts <= 128) return f(std::integral_constant<int, 4>{});
    if (experts <= 256) return f(std::integral_constant<int, 8>{});
    if (experts <= 512) return f(std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 32>{});
}

}  // namespace route

int route_blocks(int tokens, int top_k) {
    // One block chooses 16 tokens at a time; past 64 the second launch costs less than the wait.
    if (tokens <= 64 && static_cast<long long>(tokens) * top_k <= route::kSmallSlots) return 0;
    const int by_tokens = (tokens + route::kWarps - 1) / route::kWarps;
    return by_tokens < 148 ? by_tokens : 148;
}

cudaError_t launch_route(Context &ctx, const RouteDesc &d) {
    ctx.last_kernels |= GS_KERNEL_ROUTE;
    return with_float_type(d.type, [&](auto z) {
        return route::with_vpl(d.experts, [&](auto v) { return route::launch<decltype(z), decltype(v)::value>(ctx, d); });
    });
}

cudaError_t launch_route_backward(Context &ctx, const RouteBwdDesc &d) {
    ctx.last_kernels |= GS_KERNEL_ROUTE;
    const long long want = (static_cast<long long>(d.tokens) + 7) / 8, most = 32LL * ctx.sm_count;
    const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
    return with_float_type(d.type, [&](auto z) {
        return route::with_vpl(d.experts, [&](auto v) {
            using T = decltype(z);
            // the gradient has the logits' type, or f32
            auto kern = d.dtype == GS_R_32F ? route::k_route_backward<T, float, decltype(v)::value>
                                            : route::k_route_backward<T, T, decltype(v)::value>;
            const cudaError_t e = launch_pdl(kern, dim3(blocks), dim3(256), 0, ctx.stream, 1, d);
            ctx.launches++;
            return e;
        });
    });
}

}  // namespace gs
