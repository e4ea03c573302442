// gsd_attention_fwd.hip — cross attention, forward:
//   s = scale q.k,  p = softmax over the valid keys,  o = sum p v.
//
// One pass over the keys with a running maximum and sum per row.  A wave holds
// 32 rows as columns: s^T = K Q^T leaves a row's 32 scores of half a tile in
// the registers of two lanes, so maximum and sum need one exchange; o^T = V^T
// p^T takes p from those registers.  Keys and values pass through LDS in tiles
// of 64, two buffers, the next tile's loads in flight during the products.
//
// Matrix products and the vector instructions around the exponentials bound it.  A
// wave does one or the other, so two waves on a SIMD (heads of 128, whose sums and q
// take their registers) or four (64) share it.  Counters give, of a SIMD's cycles, 0.59
// with a matrix instruction, 0.49 with a vector one and 0.21 with both at once for heads
// of 128, at the 1.8 GHz that the card then runs at; for heads of 64, where an exponential
// goes with half the products, 0.43, 0.65 and 0.24.  4096 x 32400, 16 heads of 128: 0.96
// to 1.01 ms by card, 1.08 to 1.14 PFLOP/s (a large library product reaches 1.34); 4096 x
// 16200, 16 heads of 64: 0.31 ms, 0.87 PFLOP/s.
//
// Where the rows make too few work-groups, the keys are split into parts whose
// normalised sums and log-sums a second kernel joins.
#include "gsd_attention.h"

namespace gsd {

namespace {

constexpr int kRowsPerGroup = 128;

template <typename T, int DT, int DC, bool kList>
__global__ __launch_bounds__(kThreads, 2) void attention_kernel(AttnArgs a) {
    constexpr int kBytes = kTile * DT * 2;
    // one array per buffer: reads of one then wait for no load into another
    __shared__ __attribute__((aligned(256))) char s_k0[kBytes], s_v0[kBytes];
    __shared__ __attribute__((aligned(256))) char s_k1[kBytes], s_v1[kBytes];
    typedef typename T::vec8 vec8;

    const uint32_t id = work_of(blockIdx.x, a.blocks * a.parts * a.kv_heads);
    const uint32_t block = id % a.blocks;
    const uint32_t part = id / a.blocks % a.parts;
    const int bh = (int)(id / a.blocks / a.parts);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int lane = lane_id(), wave = wave_id(), half = lane >> 5;

    KeyDma<kList, DT> keys;
    keys.init(a, b, kvh);
    KeyWalk<kList> walk;
    walk.start(a, b, part);
    if (walk.more()) {
        walk.look_ahead();
        keys.fetch(walk, s_k0, s_v0);
    }

    const int row = (int)block * kRowsPerGroup + wave * 32 + (lane & 31);
    const bool live = row < a.rows;
    // a wave without a row only loads and waits
    const bool busy = (int)block * kRowsPerGroup + wave * 32 < a.rows;
    const int64_t l = live ? (uint32_t)row / (uint32_t)a.group : 0;
    const int head = kvh * a.group + (live ? row - (int)l * a.group : 0);
    vec8 q[DC / 16];
    {
        const char* from = a.q + b * a.qb + l * a.ql + head * a.qh;
#pragma unroll
        for (int ks = 0; ks < DC / 16; ++ks) {
            const int d = 16 * ks + 8 * half;
            u32x4 in{0, 0, 0, 0};
            if (live && d < a.dim) in = load_any<u32x4>(from + 2 * d);
            q[ks] = __builtin_bit_cast(vec8, in);
        }
    }
    f32x16 o[DC / 32];
#pragma unroll
    for (int db = 0; db < DC / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    // p = 2^(s c + off) with off = shift - m c; m is a maximum of some tile and
    // all before it, at most kSlack / c below the running one
    float m = -__builtin_inff(), off = T::kShift, sum = 0.0f;

    // one tile from its buffers, the next one's loads into the others; false
    // after the last.  few: the only tile, where p's rounding is made up for
    auto step = [&](auto few, const char* tile_k, const char* tile_v, char* next_k,
                    char* next_v) GSD_INLINE -> bool {
        constexpr bool kFew = decltype(few)::value;
        const int left = walk.left();
        walk.next();
        const bool more = !kFew && walk.more();
        if (more) {
            walk.look_ahead();
            keys.fetch(walk, next_k, next_v);
        }
        if (busy) {
            f32x16 s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[h][i] = 0.0f;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int ks = 0; ks < DC / 16; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    s[h] = T::mma(read_rows<T, DT>(tile_k, 32 * h, ks), q[ks], s[h]);
            pace<DC / 16, 2, 2, 2>();
            __builtin_amdgcn_s_setprio(0);
            if (left < kTile) {
                const int me = opaque(lane);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (past(h, i, me, left)) s[h][i] = -__builtin_inff();
            }
            float top = s[0][0];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
            top = fmaxf(top, other_half(top));
            if (ballot(top > m + a.slack)) {
                const float to = fmaxf(m, top);
                // no finite score so far: m stays -infinity and 2^(s c) is 0
                const bool none = to == -__builtin_inff();
                const float shrink = none ? 1.0f : __builtin_amdgcn_exp2f((m - to) * a.scale_log2);
                m = to;
                off = none ? T::kShift : T::kShift - to * a.scale_log2;
                sum *= shrink;
#pragma unroll
                for (int db = 0; db < DC / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[db][i] *= shrink;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i], a.scale_log2, off));
                    sum += s[h][i];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    // rounded to the type: a relative 2^-9 (2^-12) of each
                    // term, in the mean below the rounding of o itself
                    const vec8 p = pack<T>(s[h], k);
#pragma unroll
                    for (int db = 0; db < DC / 32; ++db) {
                        const vec8 vt = read_columns<T, DT>(tile_v, 32 * h + 16 * k, db);
                        o[db] = T::mma(vt, p, o[db]);
                        if constexpr (kFew)
                            o[db] = T::mma(vt, pack_low<T>(s[h], k), o[db]);
                    }
                }
            }
        }
        if (more) {
            dma_wait();
            __syncthreads();
        }
        return more;
    };
    if (walk.more()) {
        dma_wait();
        __syncthreads();
        if (walk.n <= kFewTerms)
            step(std::true_type{}, s_k0, s_v0, s_k1, s_v1);
        else
            while (step(std::false_type{}, s_k0, s_v0, s_k1, s_v1) &&
                   step(std::false_type{}, s_k1, s_v1, s_k0, s_v0)) {
            }
    }
    sum += other_half(sum);
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const float lse = sum == 0.0f ? -__builtin_inff()
                                  : __builtin_log2f(sum) - off;
    if (!live) return;
    if (a.parts == 1) {
        if (a.lse && half == 0) a.lse[(int64_t)bh * a.rows + row] = lse;
        const int64_t to = (((int64_t)b * (a.rows / a.group) + l) * a.heads + head) * a.dim;
#pragma unroll
        for (int db = 0; db < DC / 32; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = 32 * db + 8 * k + 4 * half;
                const float v[4] = {o[db][4 * k], o[db][4 * k + 1], o[db][4 * k + 2], o[db][4 * k + 3]};
                if (d < a.dim) put_rounded<T>(a.o, a.o_low, to + d, v, inv);
            }
    } else {
        const int64_t at = ((int64_t)part * a.batch * a.kv_heads + bh) * a.rows + row;
        if (half == 0) a.partial_lse[at] = lse;
        float* to = a.partial_o + at * a.dim;
#pragma unroll
        for (int db = 0; db < DC / 32; ++db)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = 32 * db + 8 * k + 4 * half;
                f32x4 out;
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = o[db][4 * k + i] * inv;
                if (d < a.dim) store_any(to + d, out);
            }
    }
}

// The same for at most 32 rows (single tokens): what counts is how fast the keys
// arrive.  The four waves share the rows and split the keys, each
// walking its own run of them in tiles of 32 that it loads for itself, so no wave
// waits for another before the end, where the four sums are joined through LDS.
// 8 x up to 8160 keys (100 MB of k and v in all), 4 heads of 128, each read for 4
// rows: 22 us, 4.8 TB/s.
constexpr int kFewTile = 32;

template <typename T, int DT, bool kList, bool kStream>
__global__ __launch_bounds__(kThreads) void attention_few_kernel(AttnArgs a) {
    constexpr int kBytes = kFewTile * DT * 2;  // of one tile of k or v
    constexpr int kChunks = kBytes / 1024;     // loads of a wave per tile
    constexpr int kPitch = DT + 4;             // floats per row of the joined sums
    __shared__ __attribute__((aligned(256))) char s_tile[kWaves][2][2][kBytes];
    __shared__ float s_top[kWaves][32], s_sum[kWaves][32];
    static_assert(kWaves * 32 * kPitch * 4 <= (int)sizeof(s_tile), "the sums reuse the tiles");
    typedef typename T::vec8 vec8;

    const uint32_t part = blockIdx.x % a.parts;
    const int bh = (int)(blockIdx.x / a.parts);
    const int b = bh / a.kv_heads, kvh = bh % a.kv_heads;
    const int lane = lane_id(), wave = wave_id(), half = lane >> 5;

    // this wave's share of the batch's tiles
    const int n = kList ? a.counts[b] : admitted_keys(a, b);
    const uint32_t tiles = ((uint32_t)n + kFewTile - 1) / kFewTile;
    const uint32_t shares = a.parts * kWaves, share = part * kWaves + wave;
    const int t0 = (int)((uint64_t)tiles * share / shares);
    const int t1 = (int)((uint64_t)tiles * (share + 1) / shares);

    const char* kbase = a.k + b * a.kb + kvh * a.kh;
    const char* vbase = a.v + b * a.vb + kvh * a.vh;
    // (list) the key of row lane % 32 of the tile that is fetched next
    const int32_t* list = kList ? a.list + (int64_t)b * a.keys : nullptr;
    auto ask = [&](int t) {
        const int j = t * kFewTile + (lane & 31);
        return kList && t < t1 && j < n ? list[j] : 0;
    };
    int named = ask(t0);
    auto fetch = [&](int t) {
        char* to = s_tile[wave][(t - t0) & 1][0];
        const int left = n - t * kFewTile;
        uint32_t ok[kChunks], ov[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int at = i * kWave + lane, r = at / (DT / 8);
            const int c = at % (DT / 8) ^ swizzle<DT>(r);
            const uint32_t from = kList ? (uint32_t)__shfl(named, r) : (uint32_t)r;
            const bool in = r < left && 8 * c < a.dim;
            ok[i] = in ? from * (uint32_t)a.ks + 16 * c : kOutside;
            ov[i] = in ? from * (uint32_t)a.vs + 16 * c : kOutside;
        }
        const u32x4 bk = buffer_at(kList ? kbase : kbase + (int64_t)t * kFewTile * a.ks);
        const u32x4 bv = buffer_at(kList ? vbase : vbase + (int64_t)t * kFewTile * a.vs);
        const uint32_t lds = lds_address(to);
        named = ask(t + 1);
#pragma unroll
        for (int i = 0; i < kChunks; i += 4) {
            const uint32_t x[4] = {ok[i], ok[i + 1], ok[i + 2], ok[i + 3]};
            dma16<kStream>(bk, x, lds + 1024 * i);
        }
#pragma unroll
        for (int i = 0; i < kChunks; i += 4) {
            const uint32_t x[4] = {ov[i], ov[i + 1], ov[i + 2], ov[i + 3]};
            dma16<kStream>(bv, x, lds + kBytes + 1024 * i);
        }
    };
    if (t0 < t1) fetch(t0);

    const int row = lane & 31;
    const bool live = row < a.rows;
    const int64_t l = live ? (uint32_t)row / (uint32_t)a.group : 0;
    const int head = kvh * a.group + (live ? row - (int)l * a.group : 0);
    vec8 q[DT / 16];
    {
        const char* from = a.q + b * a.qb + l * a.ql + head * a.qh;
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) {
            const int d = 16 * ks + 8 * half;
            u32x4 in{0, 0, 0, 0};
            if (live && d < a.dim) in = load_any<u32x4>(from + 2 * d);
            q[ks] = __builtin_bit_cast(vec8, in);
        }
    }
    f32x16 o[DT / 32];
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    float m = -__builtin_inff(), sum = 0.0f;
    for (int t = t0; t < t1; ++t) {
        // the reads of the tile before last are done before its place is loaded
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (t + 1 < t1) {
            fetch(t + 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kChunks) : "memory");
        } else {
            dma_wait();
        }
        const char* tile_k = s_tile[wave][(t - t0) & 1][0];
        const char* tile_v = s_tile[wave][(t - t0) & 1][1];
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) s = T::mma(read_rows<T, DT>(tile_k, 0, ks), q[ks], s);
        const int left = n - t * kFewTile;
        if (left < kFewTile) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (past(0, i, lane, left)) s[i] = -__builtin_inff();
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
        top = fmaxf(top, other_half(top));
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float shrink = __builtin_amdgcn_exp2f((m - base) * a.scale_log2);
        const float off = T::kShift - base * a.scale_log2;
        m = top;
        sum *= shrink;
#pragma unroll
        for (int db = 0; db < DT / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= shrink;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, off));
            sum += s[i];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const vec8 p = pack<T>(s, k);
#pragma unroll
            for (int db = 0; db < DT / 32; ++db)
                o[db] = T::mma(read_columns<T, DT>(tile_v, 16 * k, db), p, o[db]);
        }
        if (n <= kFewTerms)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const vec8 p = pack_low<T>(s, k);
#pragma unroll
                for (int db = 0; db < DT / 32; ++db)
                    o[db] = T::mma(read_columns<T, DT>(tile_v, 16 * k, db), p, o[db]);
            }
    }
    sum += other_half(sum);

    // the four waves' sums, in log2 units of the largest maximum
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(&s_tile[0][0][0][0]);
    if (half == 0) {
        s_top[wave][row] = m;
        s_sum[wave][row] = sum;
    }
#pragma unroll
    for (int db = 0; db < DT / 32; ++db)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f32x4 out;
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = o[db][4 * k + i];
            *reinterpret_cast<f32x4*>(s_o + (wave * 32 + row) * kPitch + 32 * db + 8 * k + 4 * half) = out;
        }
    __syncthreads();
    const int units = a.dim / 8;
    for (int at = threadIdx.x; at < a.rows * units; at += kThreads) {
        const int r = at / units, c = at - r * units;
        float top = s_top[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_top[w][r]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f((s_top[w][r] - base) * a.scale_log2);
            total = __builtin_fmaf(f, s_sum[w][r], total);
            const float* from = s_o + (w * 32 + r) * kPitch + 8 * c;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(f, from[i], acc[i]);
        }
        const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
        const float lse = total == 0.0f ? -__builtin_inff()
                                        : base * a.scale_log2 + __builtin_log2f(total) - T::kShift;
        if (a.parts == 1) {
            if (a.lse && c == 0) a.lse[(int64_t)bh * a.rows + r] = lse;
            const int lr = r / a.group;
            const int64_t hr = kvh * a.group + (r - lr * a.group);
            put_rounded<T>(a.o, a.o_low,
                           (((int64_t)b * (a.rows / a.group) + lr) * a.heads + hr) * a.dim + 8 * c, acc,
                           inv);
        } else {
            const int64_t to = ((int64_t)part * a.batch * a.kv_heads + bh) * a.rows + r;
            if (c == 0) a.partial_lse[to] = lse;
            f32x4 u, v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = acc[i] * inv;
                v[i] = acc[4 + i] * inv;
            }
            store_any(a.partial_o + to * a.dim + 8 * c, u);
            store_any(a.partial_o + to * a.dim + 8 * c + 4, v);
        }
    }
}

// o = sum over parts of o_part 2^(lse_part - lse), a thread per eight values of a
// row (at all, part p's at p all more).
struct Joined {
    float top = -__builtin_inff(), sum = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    __device__ __forceinline__ void add(float lse, float w0, const float* v) {
        const float to = fmaxf(top, lse);
        const float base = to == -__builtin_inff() ? 0.0f : to;
        const float keep = __builtin_amdgcn_exp2f(top - base);
        const float w = __builtin_amdgcn_exp2f(lse - base);
        top = to;
        sum = __builtin_fmaf(sum, keep, w * w0);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w, v[i], acc[i] * keep);
    }
    __device__ __forceinline__ void add_part(const AttnArgs& a, int64_t all, int64_t at, int c,
                                             uint32_t p) {
        const float* from = a.partial_o + (p * all + at) * a.dim + 8 * c;
        const f32x4 u = load_any<f32x4>(from), w = load_any<f32x4>(from + 4);
        const float v[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
        add(a.partial_lse[p * all + at], 1.0f, v);
    }
    template <typename T>
    __device__ __forceinline__ void write(const AttnArgs& a, int64_t at, int c) const {
        const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        const int64_t bh = at / a.rows;
        const int row = (int)(at - bh * a.rows), l = row / a.group;
        const int64_t b = bh / a.kv_heads;
        const int64_t head = (bh - b * a.kv_heads) * a.group + (row - l * a.group);
        put_rounded<T>(a.o, a.o_low, ((b * (a.rows / a.group) + l) * a.heads + head) * a.dim + 8 * c,
                       acc, inv);
        if (a.lse && c == 0)
            a.lse[at] = sum == 0.0f ? -__builtin_inff()
                                    : (top == -__builtin_inff() ? 0.0f : top) + __builtin_log2f(sum);
    }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(AttnArgs a) {
    const int units = a.dim / 8;
    const int64_t all = (int64_t)a.batch * a.kv_heads * a.rows;
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (id >= all * units) return;
    const int64_t at = id / units;
    const int c = (int)(id - at * units);
    Joined j;
    for (uint32_t p = 0; p < a.parts; ++p) j.add_part(a, all, at, c, p);
    j.write<T>(a, at, c);
}

// The same where that is few threads and many parts: a work-group has one row, lane
// p of 16 takes parts p, p + 16, ..., and the lanes' sums are joined through LDS in
// their order.  32 rows of 8 parts: 4.0 us, 12 with one thread for all parts.
constexpr int kJoinLanes = 16;

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_join_few_kernel(AttnArgs a) {
    __shared__ float s_top[kJoinLanes], s_sum[kJoinLanes], s_acc[kJoinLanes][128];
    const int64_t all = (int64_t)a.batch * a.kv_heads * a.rows, at = blockIdx.x;
    const int lane = threadIdx.x / 16, c = threadIdx.x % 16;
    const bool in = 8 * c < a.dim;
    Joined j;
    if (in)
        for (uint32_t p = lane; p < a.parts; p += kJoinLanes) j.add_part(a, all, at, c, p);
    if (c == 0) {
        s_top[lane] = j.top;
        s_sum[lane] = j.sum;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_acc[lane][8 * c + i] = j.acc[i];
    __syncthreads();
    if (!in || lane != 0) return;
    for (int k = 1; k < kJoinLanes; ++k) j.add(s_top[k], s_sum[k], &s_acc[k][8 * c]);
    j.write<T>(a, at, c);
}

// A mask as the list of its valid keys, in order, so that only those are loaded and
// multiplied: 3600 keys of which seven in ten are valid take 0.7 of all, and no
// score is masked but in the last tile.  A work-group per batch; a wave takes up to
// 4096 neighbouring keys at a time, whose words of validity its lanes hold.  3600
// keys: 5 us.
constexpr int kListWaves = 16;

__global__ __launch_bounds__(kListWaves* kWave) void key_list_kernel(AttnArgs a) {
    __shared__ int s_total[2][kListWaves];
    const int b = blockIdx.x, lane = lane_id(), wave = threadIdx.x / kWave;
    const int n = admitted_keys(a, b);
    const uint8_t* mask = a.mask + b * a.mb;
    int32_t* list = a.list + (int64_t)b * a.keys;
    int done = 0, side = 0;
    for (int64_t base = 0; base < n; side ^= 1) {
        // words per wave: those left, shared out, a lane's worth at most
        const int64_t left = (n - base + kListWaves * kWave - 1) / (kListWaves * kWave);
        const int words = left < kWave ? (int)left : kWave;
        const int64_t first = base + (int64_t)wave * words * kWave;
        base += (int64_t)kListWaves * words * kWave;
        uint64_t mine = 0;
        for (int i = 0; i < words; i += 8) {
            uint8_t byte[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int64_t j = first + (i + u) * kWave + lane;
                byte[u] = i + u < words && j < n ? mask[j * a.ms] : 0;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint64_t word = ballot(byte[u] != 0);
                if (lane == i + u) mine = word;
            }
        }
        const int own = __popcll(mine);
        int upto = own;  // of this lane's words and those before
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int other = __shfl_up(upto, d);
            if (lane >= d) upto += other;
        }
        if (lane == kWave - 1) s_total[side][wave] = upto;
        __syncthreads();
        int before = done, all = 0;
        for (int w = 0; w < kListWaves; ++w) {
            before += w < wave ? s_total[side][w] : 0;
            all += s_total[side][w];
        }
        const int start = before + upto - own;
        for (int i = 0; i < words && first + i * kWave < n; ++i) {
            const uint64_t word = __shfl(mine, i);
            const int at = __shfl(start, i);
            if ((word >> lane) & 1)
                list[at + __popcll(word & ((1ull << lane) - 1))] = (int)(first + i * kWave + lane);
        }
        done += all;
    }
    if (threadIdx.x == 0) a.counts[b] = done;
}

}  // namespace

hipError_t launch_key_list(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(key_list_kernel, dim3((unsigned)a.batch), dim3(kListWaves * kWave), 0, st, a);
    return hipGetLastError();
}

AttnArgs attention_args(const gsd_attention& g, int32_t* list) {
    AttnArgs a{};
    // without keys there is nothing to list: the lengths alone say so
    if (g.key_mask && g.keys > 0) {
        a.list = list;
        a.counts = list + g.batch * g.keys;
    }
    a.q = static_cast<const char*>(g.q);
    a.k = static_cast<const char*>(g.k);
    a.v = static_cast<const char*>(g.v);
    a.qb = 2 * g.q_stride_b;
    a.ql = 2 * g.q_stride_l;
    a.qh = 2 * g.q_stride_h;
    a.kb = 2 * g.k_stride_b;
    a.ks = 2 * g.k_stride_l;
    a.kh = 2 * g.k_stride_h;
    a.vb = 2 * g.v_stride_b;
    a.vs = 2 * g.v_stride_l;
    a.vh = 2 * g.v_stride_h;
    a.lengths = g.key_lengths;
    a.mask = g.key_mask;
    a.mb = g.mask_stride_b;
    a.ms = g.mask_stride_s;
    a.o = static_cast<char*>(g.o);
    a.o_low = static_cast<char*>(g.o_low);
    a.lse = g.lse;
    a.batch = (int32_t)g.batch;
    a.heads = (int32_t)g.heads;
    a.kv_heads = (int32_t)g.kv_heads;
    a.group = (int32_t)(g.heads / g.kv_heads);
    a.dim = (int32_t)g.dim;
    a.rows = (int32_t)(g.queries * a.group);
    a.keys = g.keys;
    a.scale = g.scale;
    a.slack = (float)(kSlack / ((double)g.scale * 1.4426950408889634073599246810019));
    a.scale_log2 = (float)((double)g.scale * 1.4426950408889634073599246810019);
    return a;
}

// Parts of the walked axis, so that blocks x parts work-groups are `per_unit` for
// each compute unit at most, each with at least `least` tiles.  The forward of heads
// of 64 has room for four on a unit: 2 x 1237 x 4134, 8 heads in groups of 4, takes 44
// us with the join, 46 with three.  dq has room for three and takes 74 us in four, 80
// in three (2 x 1237 x 8260, 8 heads); dk and dv have room for three: 112 us so, 130
// in two.
int64_t split_parts(int64_t blocks, int64_t tiles, int64_t least, int64_t per_unit) {
    if (blocks <= 0 || tiles <= 0) return 1;
    int64_t parts = per_unit * kComputeUnits / blocks;
    const int64_t most = tiles / least;
    parts = parts < most ? parts : most;
    if (parts <= 1) return 1;
    const int64_t per = (tiles + parts - 1) / parts;  // no part without a tile
    return (tiles + per - 1) / per;
}

// At most 32 rows per batch and key head.
bool few_rows(const gsd_attention& g) { return g.queries * (g.heads / g.kv_heads) <= 32; }

AttentionSplit attention_split_rows(const gsd_attention& g) {
    AttentionSplit s;
    if (few_rows(g)) {
        s.blocks = 1;
        s.tiles = (g.keys + kFewTile - 1) / kFewTile;
        // one work-group per compute unit (its tiles fill LDS), each wave with four
        // tiles at least: 8 x 8160 keys, 4 heads of 128 took 22.8 us, 23.8 with two
        // work-groups for each unit, 28.5 with four
        const int64_t problems = g.batch > 0 ? g.batch * g.kv_heads : 1;
        const int64_t parts = (kComputeUnits + problems - 1) / problems;
        const int64_t most = (s.tiles + 4 * kWaves - 1) / (4 * kWaves);
        s.parts = parts < most ? parts : most;
        s.parts = s.parts < 1 ? 1 : s.parts;
        return s;
    }
    s.blocks = (g.queries * (g.heads / g.kv_heads) + kRowsPerGroup - 1) / kRowsPerGroup;
    s.tiles = (g.keys + kTile - 1) / kTile;
    s.parts = split_parts(s.blocks * g.batch * g.kv_heads, s.tiles, 2, g.dim > 64 ? 2 : 4);
    return s;
}

namespace {

// Whether k and v, which the kernel for few rows reads once, are more than the last
// cache holds (what strides of 0 repeat counts once): 8 x 32400 keys, 4 heads of 128, 531
// MB, take 84 us (6.3 TB/s) past the caches and 98 through them; 104 MB, 23.8 and 22.7.
bool few_stream(const AttnArgs& a) {
    auto bytes = [&](int64_t b, int64_t s, int64_t h) {
        return (b ? a.batch : 1) * (s ? a.keys : 1) * (h ? a.kv_heads : 1) * 2 * a.dim;
    };
    return bytes(a.kb, a.ks, a.kh) + bytes(a.vb, a.vs, a.vh) > kLastCacheBytes;
}

template <typename T, int DT, int DC>
void launch_heads(const AttnArgs& a, bool few, hipStream_t st) {
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.total), dim3(kThreads), 0, st, a); };
    if (few && few_stream(a))
        a.list ? go(attention_few_kernel<T, DT, true, true>)
               : go(attention_few_kernel<T, DT, false, true>);
    else if (few)
        a.list ? go(attention_few_kernel<T, DT, true, false>)
               : go(attention_few_kernel<T, DT, false, false>);
    else
        a.list ? go(attention_kernel<T, DT, DC, true>) : go(attention_kernel<T, DT, DC, false>);
}

template <typename T>
hipError_t launch_typed(const AttnArgs& a, bool few, hipStream_t st) {
    const dim3 block(kThreads);
    if (a.dim <= 64)
        launch_heads<T, 64, 64>(a, few, st);
    else if (a.dim <= kMiddle)
        launch_heads<T, 128, kMiddle>(a, few, st);
    else
        launch_heads<T, 128, 128>(a, few, st);
    if (a.parts > 1) {
        // a wave on half of the SIMDs is enough to have a thread take all parts
        const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
        const int64_t threads = rows * (a.dim / 8);
        if (threads >= kComputeUnits * 2 * kWave || a.parts < 4)
            hipLaunchKernelGGL(attention_join_kernel<T>,
                               dim3((unsigned)((threads + kThreads - 1) / kThreads)), block, 0, st, a);
        else
            hipLaunchKernelGGL(attention_join_few_kernel<T>, dim3((unsigned)rows), block, 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(const gsd_attention& g, const AttentionSplit& sp, float* partial_o,
                            float* partial_lse, int32_t* list, hipStream_t st) {
    AttnArgs a = attention_args(g, list);
    if (list && g.keys > 0) {
        const hipError_t e = launch_key_list(a, st);
        if (e != hipSuccess) return e;
    }
    a.blocks = (uint32_t)sp.blocks;
    a.parts = (uint32_t)sp.parts;
    a.total = (uint32_t)(sp.blocks * sp.parts * g.batch * g.kv_heads);
    a.tiles = (int32_t)sp.tiles;
    a.tiles_per_part = (int32_t)((sp.tiles + sp.parts - 1) / sp.parts);
    a.partial_o = partial_o;
    a.partial_lse = partial_lse;
    return g.dtype == GSD_BF16 ? launch_typed<Bf16>(a, few_rows(g), st)
                               : launch_typed<F16>(a, few_rows(g), st);
}

}  // namespace gsd
