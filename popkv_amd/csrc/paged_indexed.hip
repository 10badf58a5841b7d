// Decode attention over selected tokens of the paged 4-bit K/V cache, the
// current token among them or not.
#include "paged_attention.h"

namespace popkv {
namespace {

// Eight lanes a token, sixteen dims each (one scale group at G = 16, 32, 64).
struct Row4 {
    uint2 k, v;
    uint32_t ks, vs;
};

// An octet's state for one query head, its lane's sixteen dims.
struct FoldState {
    float m, l, acc[16];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[d] = 0.0f;
    }
    // the maximum of four more logits; the state follows it
    __device__ __forceinline__ bool raise(const float (&s)[4], float& by) {
        const float mn = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), m);
        if (__ballot(mn != m) == 0) return false;
        by = mn == -INFINITY ? 1.0f : exp2_fast(m - mn);
        l *= by;
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[d] *= by;
        m = mn;
        return true;
    }
    // the eight octets' states of a wave become one, in every octet
    __device__ __forceinline__ void join() {
        float mx = m;
        mx = fmaxf(mx, lane_xor<8>(mx));
        mx = fmaxf(mx, lane_xor<16>(mx));
        mx = fmaxf(mx, lane_xor<32>(mx));
        const float f = state_weight(m, l, mx);
        auto sum = [](float v) {
            v += lane_xor<8>(v);
            v += lane_xor<16>(v);
            return v + lane_xor<32>(v);
        };
        l = sum(l * f);
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[d] = sum(acc[d] * f);
        m = mx;
    }
};

// An octet's fold of four tokens for 16-bit and, below, fp32 queries; dead
// tokens have zero scales (their values count with weight 0).  16-bit: codes as
// fp16 c - 8, dot products in packed pairs (v_dot2, fp32 sums),
//   s = delta sum(q (c - 8)) + mid sum(q),  mid = low + 8 delta
//   acc += (p delta) (c - 8),  the p mid apart
// 76 instructions a token against 115 for values dequantised to fp32; taking
// the middle of the codes keeps the two sums from cancelling.
template <typename T>
struct PickFold {
    FoldState st;
    CodeBits bits;
    uint32_t qh[8];
    float qsum, factor, mid;
    __device__ __forceinline__ void start(const T* src) {
        st.clear();
        mid = 0.0f;
        float q[16], top = 0.0f;
        load8<T>(src, q);
        load8<T>(src + 8, q + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(q[i]));
        top = fmaxf(top, dpp_mov<0xB1>(top));
        top = fmaxf(top, dpp_mov<0x4E>(top));
        top = fmaxf(top, dpp_mov<0x141>(top));
        // fp16 to the queries' precision: the head's largest magnitude in [2^8, 2^9)
        const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xffu) - 127;
        factor = ldexpf(kScaleHigh, e - 8);
        qsum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            q[i] = ldexpf(q[i], 8 - e);
            qsum += q[i];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int j = 0; j < 4; ++j) qh[4 * w + j] = pack_half2(q[8 * w + j], q[8 * w + j + 4]);
    }
    __device__ __forceinline__ void fold(const Row4 (&r)[4], const bool (&live)[4]) {
        float s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float dot = 0.0f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                half2_t c[4];
                centred_pairs(bits, w ? r[t].k.y : r[t].k.x, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) dot = __builtin_amdgcn_fdot2(as_half2(qh[4 * w + j]), c[j], dot, false);
            }
            const float low = f16_lo(r[t].ks), delta = f16_hi(r[t].ks);
            const float x = row_sum<8>(fmaf(delta, dot, fmaf(8.0f, delta, low) * qsum)) * factor;
            s[t] = live[t] ? x : -INFINITY;
        }
        float by;
        if (st.raise(s, by)) mid *= by;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float p = s[t] == -INFINITY ? 0.0f : exp2_fast(s[t] - st.m);
            const float low = f16_lo(r[t].vs), delta = f16_hi(r[t].vs);
            st.l += p;
            mid = fmaf(p, fmaf(8.0f, delta, low), mid);
            const float pd = p * delta;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                half2_t c[4];
                centred_pairs(bits, w ? r[t].v.y : r[t].v.x, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    st.acc[8 * w + j] = fmaf(static_cast<float>(c[j][0]), pd, st.acc[8 * w + j]);
                    st.acc[8 * w + j + 4] = fmaf(static_cast<float>(c[j][1]), pd, st.acc[8 * w + j + 4]);
                }
            }
        }
    }
    __device__ __forceinline__ void join() {
#pragma unroll
        for (int d = 0; d < 16; ++d) st.acc[d] += mid;
        st.join();
    }
};
// fp32: values low + c * delta, rounded once to fp32.  (Sums of codes with the
// scales applied after save an fma a value, but delta sum(q c) and low sum(q)
// cancel: results were twice as far off.)
template <>
struct PickFold<float> {
    FoldState st;
    float q[16];
    __device__ __forceinline__ void start(const float* src) {
        st.clear();
        load8<float>(src, q);
        load8<float>(src + 8, q + 8);
    }
    static __device__ __forceinline__ void values16(uint2 w, uint32_t scale, float (&x)[16]) {
        codes8(w.x, x);
        codes8(w.y, x + 8);
        const float low = f16_lo(scale), delta = f16_hi(scale);
#pragma unroll
        for (int d = 0; d < 16; ++d) x[d] = fmaf(x[d], delta, low);
    }
    __device__ __forceinline__ void fold(const Row4 (&r)[4], const bool (&live)[4]) {
        float s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float k[16], dot = 0.0f;
            values16(r[t].k, r[t].ks, k);
#pragma unroll
            for (int d = 0; d < 16; ++d) dot = fmaf(q[d], k[d], dot);
            const float x = scaled_logit(row_sum<8>(dot));
            s[t] = live[t] ? x : -INFINITY;
        }
        float by;
        st.raise(s, by);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float v[16];
            values16(r[t].v, r[t].vs, v);
            const float p = s[t] == -INFINITY ? 0.0f : exp2_fast(s[t] - st.m);
            st.l += p;
#pragma unroll
            for (int d = 0; d < 16; ++d) st.acc[d] = fmaf(p, v[d], st.acc[d]);
        }
    }
    __device__ __forceinline__ void join() { st.join(); }
};

constexpr int kPickRows = 8;                            // tokens an octet loads at once
constexpr int kPickTile = kPickRows * kWave / 8;        // tokens of a wave's pass
constexpr int kPickBlocks = 256;                        // workgroups in all, one a CU
static_assert(int64_t{kPickBlocks} / 2 * 4 <= kPagedTicketBytes);  // (more rows than half of them have one split each)
constexpr int kPickState = kState + 1;                  // (m, l, acc[128], hits of the current token)

// A row's query and its current token, for output dim threadIdx.x of waves 0
// and 1.
template <typename T>
struct CurrentDim {
    float q0, q1, k0, k1, v;
    __device__ __forceinline__ void load(const T* q, const T* ck, const T* cv) {
        const int lane = threadIdx.x & (kWave - 1);
        q0 = Elem<T>::load(q, lane);
        q1 = Elem<T>::load(q, lane + 64);
        k0 = Elem<T>::load(ck, lane);
        k1 = Elem<T>::load(ck, lane + 64);
        v = Elem<T>::load(cv, threadIdx.x & 127);
    }
    // the output from the row's state and `hits` times the current token;
    // nothing at all gives zero
    __device__ __forceinline__ void finish(float m, float l, float x, float hits, T* out) const {
        if (hits > 0.0f) {
            const float s = scaled_logit(wave_sum(fmaf(q0, k0, q1 * k1))), mx = fmaxf(m, s);
            const float f = state_weight(m, l, mx);
            const float w = s == -INFINITY && mx != -INFINITY ? 0.0f : hits * exp2_fast(s - mx);
            l = fmaf(l, f, w);
            x = fmaf(x, f, w * v);
        }
        Elem<T>::store(out, threadIdx.x, l == 0.0f ? 0.0f : x / l);
    }
};

// Merges a row's `n` states by the whole workgroup: the weights of 32 states at
// a time by every wave alike, the sums by threads (dim, part of the states).
template <typename T, int W>
__device__ __forceinline__ void pick_merge(const float* ps, int n, const CurrentDim<T>& cur, T* out) {
    constexpr int PARTS = W * kWave / 128, BURST = 32, NF = BURST / PARTS;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int d = threadIdx.x & 127, part = threadIdx.x >> 7;
    float m = -INFINITY, l = 0.0f, hits = 0.0f, a = 0.0f;
    for (int s0 = 0; s0 < n; s0 += BURST) {
        const int k = min(BURST, n - s0);
        const float* p = ps + static_cast<int64_t>(s0) * kPickState;
        float x[NF], ms = -INFINITY, ls = 0.0f, hs = 0.0f;
        if (lane < k) {
            ms = ld_f32<true>(p + lane * kPickState);
            ls = ld_f32<true>(p + lane * kPickState + 1);
            hs = ld_f32<true>(p + lane * kPickState + kState);
        }
#pragma unroll
        for (int j0 = 0; j0 < NF; j0 += 4) {
            if (PARTS * j0 >= k) break;
#pragma unroll
            for (int j = j0; j < j0 + 4; ++j)
                x[j] = ld_f32<true>(p + min(PARTS * j + part, k - 1) * kPickState + 2 + d);
        }
        const float mx = fmaxf(m, wave_max(ms));
        const float f = state_weight(m, l, mx), w = state_weight(ms, ls, mx);
        l = fmaf(l, f, wave_sum(ls * w));
        hits += wave_sum(hs);
        a *= f;
#pragma unroll
        for (int j = 0; j < NF; ++j)
            if (PARTS * j + part < k) a = fmaf(__shfl(w, PARTS * j + part), x[j], a);
        m = mx;
    }
    __shared__ float s_sum[PARTS][128];
    s_sum[part][d] = a;
    __syncthreads();
    if (wave < 2) {
        float x = a;
#pragma unroll
        for (int i = 1; i < PARTS; ++i) x += s_sum[i][d];
        cur.finish(m, l, x, hits, out);
    }
}

// One workgroup a (split of the selection, query head, sequence): every query
// head gathers its own tokens, a line of codes and one of scales each, eight of
// them on their way in an octet (four: 19.1 us against 13.5, with fp32 products),
// the next eight indices behind them.  The current token is counted, not read:
// the merge folds it in as often as it was selected.  Bound by its chain of
// reads (index, page table entry, token) and the hand-off of the splits: 4096 of
// 32767 tokens for each of 32 heads, bf16, 64-dim groups, 20 MB: 11.9 us (1.7
// TB/s); 256 of them, without a hand-off, 6.4.
template <typename T, int G, typename I, int W>
__global__ __launch_bounds__(W * kWave) void paged_indexed_kernel(PagedAttend a, PagedIndexed ix, PagedView c,
                                                                     int splits, int per) {
    constexpr int R = 128 / G;
    const int s = blockIdx.x, qh = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int oct = lane / 8, d0 = (lane % 8) * 16;
    const int64_t row = static_cast<int64_t>(b) * a.q_heads + qh;
    const int64_t kvh = ix.head_to_kv[qh];
    const int h = static_cast<int>(kvh < 0 ? 0 : kvh >= c.kv_heads ? c.kv_heads - 1 : kvh);
    const int64_t count = clamp_count(c.counts[b], c.width << c.page_log2);
    PickFold<T> f;
    f.start(static_cast<const T*>(a.q) + row * 128 + d0);
    const I* idx = static_cast<const I*>(ix.indices) + row * ix.selected;
    const uint8_t* valid = ix.valid ? ix.valid + row * ix.selected : nullptr;
    const int32_t* table = c.table + b * c.width;
    const int64_t e0 = static_cast<int64_t>(s) * per, e1 = min<int64_t>(e0 + per, ix.selected);
    int hits = 0;
    I tok[kPickRows];
    auto pick = [&](int64_t e) {
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            const int64_t at = e + oct + 8 * i;
            const bool in = at < e1 && (!valid || valid[at] != 0);
            tok[i] = in ? idx[at] : I{-1};
        }
    };
    pick(e0 + wave * kPickTile);
    for (int64_t e = e0 + wave * kPickTile; e < e1; e += W * kPickTile) {
        Row4 r[2][4];
        bool live[2][4];
        int32_t page[kPickRows];
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            hits += tok[i] == count ? 1 : 0;
            page[i] = tok[i] >= 0 && tok[i] < count ? table[tok[i] >> c.page_log2] : -1;
        }
#pragma unroll
        for (int i = 0; i < kPickRows; ++i) {
            Row4& x = r[i / 4][i % 4];
            const bool there = static_cast<uint32_t>(page[i]) < static_cast<uint32_t>(c.pages);
            live[i / 4][i % 4] = there;
            x.k = x.v = make_uint2(0u, 0u);
            x.ks = x.vs = 0u;
            if (there) {
                const int64_t at_row = ((static_cast<int64_t>(page[i]) * c.kv_heads + h) << c.page_log2) +
                                       (tok[i] & ((1 << c.page_log2) - 1));
                const char* code = c.codes + at_row * kCodeRow + d0 / 2;
                const uint32_t* sc = c.scales + at_row * (2 * R) + d0 / G;
                x.k = *reinterpret_cast<const uint2*>(code);
                x.v = *reinterpret_cast<const uint2*>(code + 64);
                x.ks = sc[0];
                x.vs = sc[R];
            }
        }
        pick(e + W * kPickTile);  // the next pass's, on their way while this one's rows are
        f.fold(r[0], live[0]);
        f.fold(r[1], live[1]);
    }
    const int64_t kv = (static_cast<int64_t>(b) * c.kv_heads + h) * 128;
    CurrentDim<T> cur;  // on its way while the wave's octets join
    cur.load(static_cast<const T*>(a.q) + row * 128, static_cast<const T*>(a.cur_k) + kv,
             static_cast<const T*>(a.cur_v) + kv);
    f.join();
    const float wave_hits = wave_sum(static_cast<float>(hits)) * 0.125f;  // the eight lanes of an octet count alike
    __shared__ float s_m[W], s_l[W], s_hits[W], s_acc[W][128];
    if (lane < 8) {
#pragma unroll
        for (int d = 0; d < 16; ++d) s_acc[wave][d0 + d] = f.st.acc[d];
        if (lane == 0) {
            s_m[wave] = f.st.m;
            s_l[wave] = f.st.l;
            s_hits[wave] = wave_hits;
        }
    }
    __syncthreads();
    float* mine = a.partials + (row * splits + s) * kPickState;
    T* out = static_cast<T*>(a.out) + row * 128;
    if (wave < 2) {
        float mx = -INFINITY, l = 0.0f, x = 0.0f, n = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float g = state_weight(s_m[w], s_l[w], mx);
            x = fmaf(g, s_acc[w][threadIdx.x], x);
            l = fmaf(g, s_l[w], l);
            n += s_hits[w];
        }
        if (splits == 1) {
            cur.finish(mx, l, x, n, out);
        } else {
            st_f32<true>(mine + 2 + threadIdx.x, x);
            if (threadIdx.x == 0) {
                st_f32<true>(mine, mx);
                st_f32<true>(mine + 1, l);
                st_f32<true>(mine + kState, n);
            }
        }
    }
    if (splits == 1) return;
    __shared__ uint32_t s_last;
    if (!last_of(a.tickets + row, splits, &s_last)) return;
    pick_merge<T, W>(a.partials + row * splits * kPickState, splits, cur, out);
}

// Waves a workgroup, and the splits of a row's selection into `per` tokens each.
// Four waves where that leaves no more than a pass to each of one workgroup a CU
// (more CUs share the gathers: 1024 of 32767 tokens for 32 heads 8.7 us, by eight
// 10.2; 1001 for 48 rows fp32 9.2 and 11.4) and where there are more rows than
// CUs (several workgroups on each: 512 rows of 1000 24.4 and 27.4); else eight, a
// workgroup a CU and half as many states (4096 for 32 heads 11.9, by four 13.1;
// 256 rows of 1024 14.9 and 17.2, of 500 9.0 and 11.4; four sequences of 2048 for
// 32 heads 16.9 and 17.1).
struct PickPlan {
    int waves, splits, per;
};
PickPlan pick_plan(int64_t rows, int64_t selected) {
    const int64_t passes = rows * ((selected + 4 * kPickTile - 1) / (4 * kPickTile));
    const int waves = rows <= kPickBlocks && passes > kPickBlocks ? 8 : 4;
    const int64_t least = waves * kPickTile, most = (selected + least - 1) / least;
    int64_t want = kPickBlocks / rows;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = ((selected + want - 1) / want + least - 1) / least * least;
    return {waves, static_cast<int>((selected + per - 1) / per), static_cast<int>(per)};
}

template <typename T, int G>
hipError_t launch_indexed_t(const PagedAttend& a, const PagedIndexed& ix, const PagedView& c, hipStream_t stream) {
    const PickPlan p = pick_plan(static_cast<int64_t>(c.batch) * a.q_heads, ix.selected);
    const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.q_heads), static_cast<unsigned>(c.batch));
#define POPKV_PICK(I, W) \
    hipLaunchKernelGGL((paged_indexed_kernel<T, G, I, W>), grid, dim3(W * kWave), 0, stream, a, ix, c, p.splits, p.per)
    if (ix.index_dtype == POPKV_INDEX_I32) {
        if (p.waves == 8) POPKV_PICK(int32_t, 8);
        else POPKV_PICK(int32_t, 4);
    } else {
        if (p.waves == 8) POPKV_PICK(int64_t, 8);
        else POPKV_PICK(int64_t, 4);
    }
#undef POPKV_PICK
    return hipGetLastError();
}

}  // namespace

int64_t paged_indexed_splits(int64_t rows, int64_t selected) { return pick_plan(rows, selected).splits; }

hipError_t launch_paged_indexed(const PagedAttend& a, const PagedIndexed& ix, const PagedView& c, int dtype,
                                int dim_group, hipStream_t stream) {
#define POPKV_CALL(T, G) launch_indexed_t<T, G>(a, ix, c, stream)
    POPKV_PAGED_T(POPKV_CALL)
#undef POPKV_CALL
}

}  // namespace popkv
