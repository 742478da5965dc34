// Attention of trees of drafted tokens over the paged cache.
//
// Request s has L = lengths[s] tokens of text in the cache and n = cu_nodes[s + 1] - cu_nodes[s] rows in the step, whose keys and
// values stand in the cache behind the text (row i at place L + i).  Row i sees all of the text and the rows j whose bit is set in
// its words of `ancestors`:
//     o_i = sum over visible x of softmax_x(scale * q_i . k_x) v_x,        zeros where nothing is visible.
// The places from L + n on hold other requests' or old data: they are never read (their part of a tile is zeros).
//
// What bounds it: a key and a value row are read once for all n * (heads per key/value head) query rows that use them, so few
// rows are bound by the cache's bytes and many by the products (32-bit: by the CUDA cores' fused multiply-adds).
//
// The maximum is kept as a score, and a weight is 2^((s - max) * scale * log2 e): the difference first, so that scores of any size
// give weights up to 1 (a fused s * c - rounded(max * c) leaves a rounding of the maximum's size, which overflows from 2^31 on).
//
// Layout.  The query rows of one key/value head (row r = node r / G, head r % G of its group of G) are packed into tiles of
// RW rows a warp and WR warps.  A block walks one span of the keys of one (request, key/value head): WK groups of WR warps take its
// tiles of BK keys in turn, each with stages of its own in shared memory (cp.async, ST deep, the block-table entries one tile
// further ahead: a lane looks one key's page up and hands it round) and its own running maximum, sum and output rows in registers;
// the groups meet in order at the end.  Spans of one request meet in tree_attention_join_kernel, in order of position.
//   bfloat16: S = Q K^T and O += P V on mma.sync.m16n8k16, p as two bfloat16 terms (its rounding and what that left out), so the
//             weights keep about 16 bits; sums in 32 bits.
//   float32:  fused multiply-adds on the CUDA cores; a lane owns one key of a tile for S and DP / 32 columns for O.
// Values in places that some rows see and others do not (the tree's own) may be infinite or NaN: a weight of zero would turn them
// into NaN, so such elements are taken out of the tile and added to the rows that see them only.
#include "common.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned int NO_ROW = 0xffffffffu;

struct TreeArgs {
    const void* q; long long ldq;
    const void* k_pages; const void* v_pages;
    const int* block_table; int bt_stride, width;
    const int* lengths; const int* cu_nodes; const int* ancestors; int words;
    void* out; long long ldo;
    float* part_o; float* part_ml;          // [splits, T, H, dh] and [splits, T, H, 2]
    int T, H, Hkv, dh, page_size, page_shift, splits, row_tiles, q_vec, out_vec;
    float scale_log2;
};

__device__ __forceinline__ uint32_t s_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;                     // 0 source bytes: the 16 bytes are filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s_u32(dst)), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s_u32(p)) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s_u32(p)) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// The warps of one group; one warp needs no barrier of the block.
template <int WR> __device__ __forceinline__ void group_sync(int group) {
    if (WR == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WR * 32) : "memory");
}
template <int WR> __device__ __forceinline__ bool group_any(int group, bool x) {
    if (WR == 1) return __any_sync(0xffffffffu, x);
    int r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((int)x), "r"(group + 1), "n"(WR * 32) : "memory");
    return r != 0;
}

// Whether any of the 16 bytes' elements is infinite or NaN (the exponent's bits all set).
template <typename T> __device__ __forceinline__ bool odd_element(uint32_t w);
template <> __device__ __forceinline__ bool odd_element<float>(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; }
template <> __device__ __forceinline__ bool odd_element<__nv_bfloat16>(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
template <typename T> __device__ __forceinline__ uint32_t without_odd(uint32_t w);
template <> __device__ __forceinline__ uint32_t without_odd<float>(uint32_t w) { return odd_element<float>(w) ? 0u : w; }
template <> __device__ __forceinline__ uint32_t without_odd<__nv_bfloat16>(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}

// How the keys of a request are cut into spans: as evenly as whole units of `unit` keys allow.
__device__ __forceinline__ int span_of(int keys, int splits, int unit) {
    return ((keys + splits - 1) / splits + unit - 1) / unit * unit;
}
constexpr int SPAN_UNIT = 64;

// Keys of a request that its block table holds, and the text's share of them.
__device__ __forceinline__ int keys_of(const TreeArgs& a, int len, int n) {
    return (int)min((long long)len + n, (long long)a.width * a.page_size);
}

// Which of the 64 keys from `key0` on a node sees: bit b for key key0 + b.
__device__ __forceinline__ unsigned long long tile_mask(const int* words, int n_words, int len, int keys, int key0, bool node) {
    const int j0 = key0 - len;                              // place of the first key in the tree
    auto word = [&](int w) -> unsigned long long { return w >= 0 && w < n_words && node ? (unsigned int)words[w] : 0u; };
    auto from = [&](int j) -> unsigned long long {          // bits j .. j + 63 of the node's words, j >= 0
        const int w = j >> 5, sh = j & 31;
        unsigned long long lo = word(w) | word(w + 1) << 32;
        if (sh) lo = lo >> sh | word(w + 2) << (64 - sh);
        return lo;
    };
    unsigned long long m = j0 >= 0 ? from(j0) : j0 <= -64 ? ~0ull : ((1ull << -j0) - 1ull) | from(0) << -j0;
    const int left = keys - key0;                           // keys of the request from key0 on
    if (left <= 0) return 0;
    return left >= 64 ? m : m & ((1ull << left) - 1ull);
}

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST>
struct Shape {
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int ROW = DP + VEC;                    // padded rows: neighbours start on other banks
    static constexpr int ROWS = RW * WR;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr size_t q_bytes = (size_t)ROWS * ROW * sizeof(T);
    static constexpr size_t kv_bytes = (size_t)WK * ST * 2 * BK * ROW * sizeof(T);
    static constexpr size_t p_bytes = F32 ? (size_t)WK * WR * RW * BK * 4 : 0;
    static constexpr int STATE = F32 ? RW * (DP / 32) + 2 * RW : DP / 2 + 4;     // 32-bit words a thread hands over
    static constexpr size_t xch_bytes = (size_t)(WK - 1) * WR * 32 * STATE * 4;
    static constexpr size_t bytes = q_bytes + (kv_bytes + p_bytes > xch_bytes ? kv_bytes + p_bytes : xch_bytes);
};

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST>
__global__ void __launch_bounds__(WR * WK * 32)
tree_attention_kernel(const TreeArgs a) {
    using S = Shape<T, DP, RW, WR, WK, BK, ST>;
    constexpr int VEC = S::VEC, ROW = S::ROW, CH = DP / VEC, NT = WR * 32;
    constexpr bool F32 = S::F32;
    extern __shared__ __align__(16) uint8_t smem[];
    T* sQ = reinterpret_cast<T*>(smem);
    uint8_t* shared_rest = smem + S::q_bytes;
    const int group = threadIdx.x / NT, gtid = threadIdx.x % NT, warp = gtid >> 5, lane = gtid & 31;
    T* sKV = reinterpret_cast<T*>(shared_rest) + (size_t)group * ST * 2 * BK * ROW;     // [ST][K, V][BK][ROW]
    float* sP = reinterpret_cast<float*>(shared_rest + S::kv_bytes) + (size_t)(group * WR + warp) * RW * BK;

    pdl_wait();
    pdl_launch();
    const int s = blockIdx.z, hk = blockIdx.y % a.Hkv, G = a.H / a.Hkv;
    const int first = a.cu_nodes[s], n = a.cu_nodes[s + 1] - first, len = a.lengths[s];
    if (n <= 0) return;
    const int keys = keys_of(a, len, n), span = span_of(keys, a.splits, SPAN_UNIT);
    const int k0 = (int)blockIdx.x * span, k1 = min(keys, k0 + span);
    if (k0 >= k1) return;
    const bool alone = span >= keys;                        // the request's keys are one span: no join follows
    const int rows = n * G;
    const T* k_pages = static_cast<const T*>(a.k_pages);
    const T* v_pages = static_cast<const T*>(a.v_pages);
    const int* bt = a.block_table + (size_t)s * a.bt_stride;
    const int t_first = k0 / BK, t_last = (k1 - 1) / BK;    // spans start at multiples of 64, tiles never straddle them
    const int dh_ch = a.dh / VEC;                           // 16-byte pieces of a row; the rest of DP is zeros

    for (int rt = (int)blockIdx.y / a.Hkv; rt * S::ROWS < rows; rt += a.row_tiles) {
        // the queries of this tile of rows
        const int r0 = rt * S::ROWS;
        const T* q = static_cast<const T*>(a.q);
        for (int i = threadIdx.x; i < S::ROWS * CH; i += WR * WK * 32) {
            const int r = i / CH, c = i % CH;
            const int node = (r0 + r) / G, h = hk * G + (r0 + r) % G;
            const bool ok = r0 + r < rows && c < dh_ch;
            const T* src = q + (size_t)(first + (ok ? node : 0)) * a.ldq + (size_t)h * a.dh + c * VEC;
            if (a.q_vec) {
                cp_async16(sQ + r * ROW + c * VEC, ok ? src : q, ok);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) sQ[r * ROW + c * VEC + e] = ok ? src[e] : from_f32<T>(0.f);
            }
        }
        cp_commit();

        // A lane looks up the rows of the tile's keys lane, lane + 32, ...; every thread of the group has its warp's copy.
        unsigned int row_id[BK / 32];
        auto look_up = [&](int t) {
#pragma unroll
            for (int u = 0; u < BK / 32; ++u) {
                const int kp = t * BK + u * 32 + lane;
                row_id[u] = NO_ROW;
                if (t <= t_last && kp < k1) {
                    const int p = a.page_shift >= 0 ? kp >> a.page_shift : kp / a.page_size;
                    row_id[u] = ((unsigned int)bt[p] * a.Hkv + hk) * a.page_size + (kp - p * a.page_size);
                }
            }
        };
        auto load = [&](int stage) {                          // with the rows that look_up() brought
            T* dK = sKV + (size_t)stage * 2 * BK * ROW;
            T* dV = dK + BK * ROW;
#pragma unroll
            for (int it = 0; it < (BK * CH + NT - 1) / NT; ++it) {
                const int i = gtid + it * NT;
                const int r = i / CH, c = i % CH;
                unsigned int id = __shfl_sync(0xffffffffu, row_id[0], r & 31);
#pragma unroll
                for (int u = 1; u < BK / 32; ++u) {
                    const unsigned int other = __shfl_sync(0xffffffffu, row_id[u], r & 31);
                    id = r >> 5 == u ? other : id;
                }
                if (BK * CH % NT == 0 || i < BK * CH) {
                    const bool ok = id != NO_ROW && c < dh_ch;
                    const size_t off = ok ? (size_t)id * a.dh + c * VEC : 0;
                    cp_async16(dK + r * ROW + c * VEC, k_pages + off, ok);
                    cp_async16(dV + r * ROW + c * VEC, v_pages + off, ok);
                }
            }
        };
        int t = t_first + group;
#pragma unroll
        for (int st = 0; st < ST - 1; ++st) {
            look_up(t + st * WK);
            if (t + st * WK <= t_last) load(st);
            cp_commit();
        }
        look_up(t + (ST - 1) * WK);
        cp_wait<ST - 1>();                                    // the queries are in
        __syncthreads();

        // ---- running state
        constexpr int VD = DP / 32;                           // float32: columns a lane owns
        constexpr int ON = F32 ? RW * VD : DP / 2;
        float o[ON];
#pragma unroll
        for (int i = 0; i < ON; ++i) o[i] = 0.f;
        constexpr int MN = F32 ? RW : 2;                      // rows whose maximum and sum a thread keeps
        float m_run[MN], l_run[MN];
#pragma unroll
        for (int i = 0; i < MN; ++i) { m_run[i] = -INFINITY; l_run[i] = 0.f; }
        const int g = lane >> 2, tq = lane & 3;               // bfloat16: fragment row and column
        uint32_t qa[F32 ? 1 : DP / 16][4];
        if (!F32) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) ldsm_x4(qa[ks], sQ + (warp * 16 + (lane & 15)) * ROW + ks * 16 + (lane >> 4) * 8);
        }
        auto row_of = [&](int i) { return r0 + warp * RW + (F32 ? i : g + 8 * i); };      // the query row of a thread's i-th state
        auto words_of = [&](int r) { return a.ancestors + (size_t)(first + (r < rows ? r / G : 0)) * a.words; };

        int stage = 0;
        for (; t <= t_last; t += WK) {
            {
                const int ahead = stage == 0 ? ST - 1 : stage - 1;     // the stage whose tile was used last
                if (t + (ST - 1) * WK <= t_last) load(ahead);
                cp_commit();
                look_up(t + ST * WK);
            }
            cp_wait<ST - 1>();
            T* tK = sKV + (size_t)stage * 2 * BK * ROW;
            T* tV = tK + BK * ROW;
            const int key0 = t * BK;
            const bool tail = key0 + BK > min(len, keys);     // the tile reaches into the tree or past the keys
            bool odd = false;
            if (tail) {
                // infinite and NaN values: looked for by the threads that copied them, before the group reads the tile
                for (int i = gtid; i < BK * CH; i += NT) {
                    const uint4 w = *reinterpret_cast<const uint4*>(tV + (i / CH) * ROW + (i % CH) * VEC);
                    odd |= key0 + i / CH >= len && (odd_element<T>(w.x) || odd_element<T>(w.y) || odd_element<T>(w.z) || odd_element<T>(w.w));
                }
                odd = group_any<WR>(group, odd);
                if (odd) {
                    for (int i = gtid; i < BK * CH; i += NT) {
                        if (key0 + i / CH < len) continue;
                        uint4* w = reinterpret_cast<uint4*>(tV + (i / CH) * ROW + (i % CH) * VEC);
                        *w = make_uint4(without_odd<T>(w->x), without_odd<T>(w->y), without_odd<T>(w->z), without_odd<T>(w->w));
                    }
                }
                group_sync<WR>(group);
            } else {
                group_sync<WR>(group);
            }
            unsigned long long seen[MN];
            if (tail) {
#pragma unroll
                for (int i = 0; i < MN; ++i)
                    seen[i] = tile_mask(words_of(row_of(i)), a.words, len, keys, key0, row_of(i) < rows);
            }

            if constexpr (!F32) {
                // ---- S = Q K^T: 16 rows x BK keys
                float sc[BK / 8][4];
#pragma unroll
                for (int nt = 0; nt < BK / 8; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) sc[nt][k] = 0.f;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
                    for (int np = 0; np < BK / 16; ++np) {
                        uint32_t b[4];
                        ldsm_x4(b, tK + (np * 16 + (lane & 7) + ((lane >> 4) << 3)) * ROW + ks * 16 + ((lane >> 3) & 1) * 8);
                        mma16816(sc[2 * np], qa[ks], b[0], b[1]);
                        mma16816(sc[2 * np + 1], qa[ks], b[2], b[3]);
                    }
                }
                if (tail) {
#pragma unroll
                    for (int nt = 0; nt < BK / 8; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!(seen[k >> 1] >> (nt * 8 + 2 * tq + (k & 1)) & 1)) sc[nt][k] = -INFINITY;
                }
                float alpha[2], mneg[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int nt = 0; nt < BK / 8; ++nt) mx = fmaxf(mx, fmaxf(sc[nt][2 * r], sc[nt][2 * r + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float m_new = fmaxf(m_run[r], mx);
                    const float m_use = m_new == -INFINITY ? 0.f : m_new;
                    alpha[r] = fast_exp2((m_run[r] - m_use) * a.scale_log2);
                    m_run[r] = m_new;
                    mneg[r] = -m_use;
                }
                float rs[2] = {0.f, 0.f};
                uint32_t pa[BK / 16][4], pb[BK / 16][4];
#pragma unroll
                for (int nt = 0; nt < BK / 8; ++nt) {
                    const float p0 = fast_exp2((sc[nt][0] + mneg[0]) * a.scale_log2), p1 = fast_exp2((sc[nt][1] + mneg[0]) * a.scale_log2);
                    const float p2 = fast_exp2((sc[nt][2] + mneg[1]) * a.scale_log2), p3 = fast_exp2((sc[nt][3] + mneg[1]) * a.scale_log2);
                    rs[0] += p0 + p1;
                    rs[1] += p2 + p3;
                    const uint32_t h01 = pack_bf16(p0, p1), h23 = pack_bf16(p2, p3);
                    pa[nt >> 1][(nt & 1) * 2] = h01;
                    pa[nt >> 1][(nt & 1) * 2 + 1] = h23;
                    pb[nt >> 1][(nt & 1) * 2] = pack_bf16(p0 - __uint_as_float(h01 << 16), p1 - __uint_as_float(h01 & 0xffff0000u));
                    pb[nt >> 1][(nt & 1) * 2 + 1] = pack_bf16(p2 - __uint_as_float(h23 << 16), p3 - __uint_as_float(h23 & 0xffff0000u));
                }
                // a thread's share of the sums; the four lanes of a row meet at the end
                l_run[0] = l_run[0] * alpha[0] + rs[0];
                l_run[1] = l_run[1] * alpha[1] + rs[1];
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) {
                        o[4 * i] *= alpha[0]; o[4 * i + 1] *= alpha[0];
                        o[4 * i + 2] *= alpha[1]; o[4 * i + 3] *= alpha[1];
                    }
                }
                // ---- O += P V
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) {
#pragma unroll
                    for (int dp = 0; dp < DP / 16; ++dp) {
                        uint32_t b[4];
                        ldsm_x4_trans(b, tV + (kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * ROW + dp * 16 + (lane >> 4) * 8);
                        float (&c0)[4] = *reinterpret_cast<float (*)[4]>(&o[8 * dp]);
                        float (&c1)[4] = *reinterpret_cast<float (*)[4]>(&o[8 * dp + 4]);
                        mma16816(c0, pa[kk], b[0], b[1]);
                        mma16816(c1, pa[kk], b[2], b[3]);
                        mma16816(c0, pb[kk], b[0], b[1]);
                        mma16816(c1, pb[kk], b[2], b[3]);
                    }
                }
            } else {
                // ---- S: lane = key
                static_assert(!F32 || BK == 32, "a lane owns one key of a tile");
                float sc[RW];
#pragma unroll
                for (int r = 0; r < RW; ++r) sc[r] = 0.f;
                const float* kr = reinterpret_cast<const float*>(tK) + lane * ROW;
                const float* qr = reinterpret_cast<const float*>(sQ) + warp * RW * ROW;
#pragma unroll 4
                for (int d = 0; d < DP; d += 4) {
                    const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
                    for (int r = 0; r < RW; ++r) {
                        const float4 qv = *reinterpret_cast<const float4*>(qr + r * ROW + d);
                        sc[r] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, sc[r]))));
                    }
                }
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    if (tail && !(seen[r] >> lane & 1)) sc[r] = -INFINITY;
                    const float m_new = fmaxf(m_run[r], warp_max(sc[r]));
                    const float m_use = m_new == -INFINITY ? 0.f : m_new;
                    const float alpha = exp2f((m_run[r] - m_use) * a.scale_log2);
                    m_run[r] = m_new;
                    const float p = exp2f((sc[r] - m_use) * a.scale_log2);
                    l_run[r] = l_run[r] * alpha + p;                     // this lane's keys; the lanes meet at the end
#pragma unroll
                    for (int v = 0; v < VD; ++v) o[r * VD + v] *= alpha;
                    sP[r * BK + lane] = p;
                }
                __syncwarp();
                // ---- O: a lane owns VD columns
                const float* vr = reinterpret_cast<const float*>(tV) + lane * VD;
#pragma unroll 2
                for (int k = 0; k < BK; k += 4) {
                    float v[4][VD];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int x = 0; x < VD; ++x) v[e][x] = vr[(k + e) * ROW + x];
#pragma unroll
                    for (int r = 0; r < RW; ++r) {
                        const float4 p = *reinterpret_cast<const float4*>(sP + r * BK + k);
#pragma unroll
                        for (int x = 0; x < VD; ++x)
                            o[r * VD + x] = fmaf(p.w, v[3][x], fmaf(p.z, v[2][x], fmaf(p.y, v[1][x], fmaf(p.x, v[0][x], o[r * VD + x]))));
                    }
                }
                __syncwarp();
            }
            if (tail && odd) {
                // infinite and NaN elements, from memory, to the rows that see them
                for (int b = max(0, len - key0); b < min(BK, k1 - key0); ++b) {
                    const int kp = key0 + b, p = kp / a.page_size;
                    const T* vrow = v_pages + (((size_t)bt[p] * a.Hkv + hk) * a.page_size + kp % a.page_size) * a.dh;
#pragma unroll
                    for (int i = 0; i < MN; ++i) {
                        if (!(seen[i] >> b & 1)) continue;
                        constexpr int PER = F32 ? VD : DP / 4;
#pragma unroll
                        for (int e = 0; e < PER; ++e) {
                            const int d = F32 ? lane * VD + e : (e >> 1) * 8 + 2 * tq + (e & 1);
                            if (d >= a.dh) continue;
                            const float v = to_f32(vrow[d]);
                            if (!(fabsf(v) < INFINITY)) o[F32 ? i * VD + e : (e >> 1) * 4 + 2 * i + (e & 1)] += v;
                        }
                    }
                }
            }
            group_sync<WR>(group);                            // the stage may be overwritten by the next load
            stage = stage + 1 == ST ? 0 : stage + 1;
        }
        cp_wait<0>();
        // the lanes' shares of the sums
#pragma unroll
        for (int i = 0; i < MN; ++i) {
            if (F32) {
                l_run[i] = warp_sum(l_run[i]);
            } else {
                l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
                l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
            }
        }
        // ---- the groups meet, in order, in the first one's registers
        if (WK > 1) {
            __syncthreads();
            float* xch = reinterpret_cast<float*>(shared_rest);
            constexpr int N = S::STATE;
            if (group > 0) {
                float* mine = xch + (size_t)(group - 1) * N * NT + gtid;
#pragma unroll
                for (int i = 0; i < MN; ++i) { mine[(2 * i) * NT] = m_run[i]; mine[(2 * i + 1) * NT] = l_run[i]; }
#pragma unroll
                for (int i = 0; i < ON; ++i) mine[(2 * MN + i) * NT] = o[i];
            }
            __syncthreads();
            if (group == 0) {
                for (int other = 0; other < WK - 1; ++other) {
                    const float* his = xch + (size_t)other * N * NT + gtid;
#pragma unroll
                    for (int i = 0; i < MN; ++i) {
                        const float m1 = his[(2 * i) * NT], l1 = his[(2 * i + 1) * NT];
                        const float mm = fmaxf(m_run[i], m1), use = mm == -INFINITY ? 0.f : mm;
                        const float w0 = exp2f((m_run[i] - use) * a.scale_log2), w1 = exp2f((m1 - use) * a.scale_log2);
                        m_run[i] = mm;
                        l_run[i] = l_run[i] * w0 + l1 * w1;
                        if (F32) {
#pragma unroll
                            for (int x = 0; x < VD; ++x) o[i * VD + x] = o[i * VD + x] * w0 + his[(2 * MN + i * VD + x) * NT] * w1;
                        } else {
#pragma unroll
                            for (int e = 0; e < DP / 8; ++e)
#pragma unroll
                                for (int b = 0; b < 2; ++b)
                                    o[e * 4 + 2 * i + b] = o[e * 4 + 2 * i + b] * w0 + his[(2 * MN + e * 4 + 2 * i + b) * NT] * w1;
                        }
                    }
                }
            }
        }
        // ---- out
        if (group == 0) {
#pragma unroll
            for (int i = 0; i < MN; ++i) {
                const int r = row_of(i);
                if (r >= rows) continue;
                const int token = first + r / G, h = hk * G + r % G;
                const float inv = l_run[i] > 0.f || l_run[i] != l_run[i] ? 1.f / l_run[i] : 0.f;
                const size_t pr = ((size_t)blockIdx.x * a.T + token) * a.H + h;
                if (!alone && (F32 ? lane == 0 : tq == 0)) {
                    a.part_ml[2 * pr] = m_run[i];
                    a.part_ml[2 * pr + 1] = l_run[i];
                }
                T* orow = static_cast<T*>(a.out) + (size_t)token * a.ldo + (size_t)h * a.dh;
                float* prow = a.part_o + pr * a.dh;
                if (F32) {
#pragma unroll
                    for (int x = 0; x < VD; ++x) {
                        const int d = lane * VD + x;
                        if (d >= a.dh) continue;
                        if (alone) orow[d] = from_f32<T>(o[i * VD + x] * inv);
                        else prow[d] = o[i * VD + x];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < DP / 8; ++e) {
                        const int d = e * 8 + 2 * tq;
                        if (d >= a.dh) continue;
                        const float x0 = o[e * 4 + 2 * i], x1 = o[e * 4 + 2 * i + 1];
                        if (!alone) *reinterpret_cast<float2*>(prow + d) = make_float2(x0, x1);
                        else if (a.out_vec) *reinterpret_cast<uint32_t*>(orow + d) = pack_bf16(x0 * inv, x1 * inv);
                        else { orow[d] = from_f32<T>(x0 * inv); orow[d + 1] = from_f32<T>(x1 * inv); }
                    }
                }
            }
        }
        __syncthreads();                                      // shared memory is free for the next tile of rows
    }
}

// The spans of a request's keys meet: a warp per (row, head), spans in order of position.
template <typename T>
__global__ void __launch_bounds__(128)
tree_attention_join_kernel(const TreeArgs a) {
    pdl_wait();
    pdl_launch();
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const int first = a.cu_nodes[s], n = a.cu_nodes[s + 1] - first, len = a.lengths[s];
    if (n <= 0) return;
    const int keys = keys_of(a, len, n), span = span_of(keys, a.splits, SPAN_UNIT);
    if (keys <= 0 || span >= keys) return;
    const int spans = (keys + span - 1) / span;
    const size_t step = (size_t)a.T * a.H;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 5); r < n * a.H; r += gridDim.x * 4) {
        const size_t at = (size_t)first * a.H + r;
        float m = -INFINITY;
        for (int k = lane; k < spans; k += 32) m = fmaxf(m, a.part_ml[2 * (k * step + at)]);
        m = warp_max(m);
        const float use = m == -INFINITY ? 0.f : m;
        float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < spans; ++k) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (k * step + at));
            if (ml.x == -INFINITY) continue;                  // nothing visible in this span
            const float w = exp2f((ml.x - use) * a.scale_log2);
            l += ml.y * w;
            const float* po = a.part_o + (k * step + at) * a.dh;
#pragma unroll
            for (int x = 0; x < 8; ++x)
                if (x * 32 + lane < a.dh) o[x] = fmaf(po[x * 32 + lane], w, o[x]);
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        T* orow = static_cast<T*>(a.out) + (size_t)(at / a.H) * a.ldo + (at % a.H) * a.dh;
#pragma unroll
        for (int x = 0; x < 8; ++x)
            if (x * 32 + lane < a.dh) orow[x * 32 + lane] = from_f32<T>(o[x] * inv);
    }
}

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST>
int launch(const TreeArgs& a, int S, cudaStream_t stream) {
    using Sh = Shape<T, DP, RW, WR, WK, BK, ST>;
    static_assert(Sh::bytes <= 232448, "shared memory of a block");
    auto kern = tree_attention_kernel<T, DP, RW, WR, WK, BK, ST>;
    static bool set = false;
    if (!set && Sh::bytes > 48 * 1024) {
        MLLM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::bytes));
        set = true;
    }
    MLLM_CUDA(mllm_launch(kern, dim3(a.splits, a.Hkv * a.row_tiles, S), dim3(WR * WK * 32), Sh::bytes, stream, true, a));
    if (a.splits > 1) {
        const int blocks = (a.T * a.H + 4 * S - 1) / (4 * S);           // as many warps as rows, were the trees alike
        MLLM_CUDA(mllm_launch(tree_attention_join_kernel<T>, dim3(blocks < 1 ? 1 : blocks, S), dim3(128), 0, stream, true, a));
    }
    return 0;
}

template <int DP>
int by_rows(const TreeArgs& a, int dtype, int tile_rows, int S, cudaStream_t stream) {
    using bf = __nv_bfloat16;
    if (dtype == MLLM_BF16) {
        if (tile_rows == 16) return launch<bf, DP, 16, 1, DP == 256 ? 2 : 4, 32, DP >= 128 ? 2 : 3>(a, S, stream);
        if (tile_rows == 32) return launch<bf, DP, 16, 2, 2, DP >= 128 ? 32 : 64, 2>(a, S, stream);
        return launch<bf, DP, 16, 4, DP == 256 ? 1 : 2, DP >= 128 ? 32 : 64, 2>(a, S, stream);
    }
    if (tile_rows == 4) return launch<float, DP, 4, 1, DP == 256 ? 1 : DP == 128 ? 3 : 4, 32, 2>(a, S, stream);
    if (tile_rows == 8) return launch<float, DP, 8, 1, DP == 256 ? 1 : DP == 128 ? 3 : 4, 32, 2>(a, S, stream);
    if (tile_rows == 16) return launch<float, DP, 16, 1, DP == 256 ? 1 : DP == 128 ? 2 : 4, 32, 2>(a, S, stream);
    return launch<float, DP, 16, 4, 1, 32, 2>(a, S, stream);
}

}  // namespace

// tile_rows: 16, 32 or 64 (bfloat16), 4, 8, 16 or 64 (float32) query rows of a key/value head per block; row_tiles: blocks that
// share them.  splits: spans of a request's keys at most; more than one needs part_o [splits, T, H, dh] and part_ml
// [splits, T, H, 2].  The head size is a multiple of 16 up to 256.
MLLM_EXPORT int mllm_tree_attention(const void* q, long long ldq, const void* k_pages, const void* v_pages, long long pages,
                                    const int* block_table, int bt_stride, int width, const int* lengths, const int* cu_nodes,
                                    const int* ancestors, int words, void* out, long long ldo, float* part_o, float* part_ml, int T,
                                    int S, int H, int Hkv, int dh, int page_size, float scale, int tile_rows, int row_tiles,
                                    int splits, int dtype, cudaStream_t stream) {
    if (T <= 0 || S <= 0) return 0;
    if (Hkv <= 0 || H % Hkv != 0) return mllm_fail(1, "tree_attention: %d heads over %d key/value heads", H, Hkv);
    if (dh < 16 || dh > 256 || dh % 16) return mllm_fail(1, "tree_attention: head size %d is not a multiple of 16 in 16..256", dh);
    if (!(scale > 0.f)) return mllm_fail(1, "tree_attention: the score scale must be positive, got %g", (double)scale);
    if (dtype != MLLM_F32 && dtype != MLLM_BF16) return mllm_fail(1, "tree_attention: unknown dtype code %d", dtype);
    if (page_size <= 0 || width <= 0 || words <= 0 || splits <= 0 || row_tiles <= 0)
        return mllm_fail(1, "tree_attention: pages of %d, a table of %d columns, %d words, %d spans, %d row tiles", page_size, width,
                         words, splits, row_tiles);
    if (pages * Hkv * page_size >= (long long)NO_ROW)
        return mllm_fail(1, "tree_attention: a pool of %lld rows of keys is more than 32-bit row numbers hold", pages * Hkv * page_size);
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) % 16) return mllm_fail(1, "tree_attention: pages must be 16-byte aligned");
    if ((long long)Hkv * row_tiles > 65535 || S > 65535)
        return mllm_fail(1, "tree_attention: %d requests of %d row tiles are more than one launch takes", S, Hkv * row_tiles);
    if (splits > 1 && (!part_o || !part_ml)) return mllm_fail(1, "tree_attention: %d spans need scratch to meet in", splits);
    const int es = dtype == MLLM_F32 ? 4 : 2;
    int shift = -1;
    for (int b = 0; b < 31; ++b)
        if (page_size == 1 << b) shift = b;
    const TreeArgs a{q, ldq, k_pages, v_pages, block_table, bt_stride, width, lengths, cu_nodes, ancestors, words, out, ldo, part_o,
                     part_ml, T, H, Hkv, dh, page_size, shift, splits, row_tiles,
                     (uintptr_t)q % 16 == 0 && ldq * es % 16 == 0, (uintptr_t)out % 4 == 0 && ldo * es % 4 == 0, scale * LOG2E};
    if (dh <= 32) return by_rows<32>(a, dtype, tile_rows, S, stream);
    if (dh <= 64) return by_rows<64>(a, dtype, tile_rows, S, stream);
    if (dh <= 128) return by_rows<128>(a, dtype, tile_rows, S, stream);
    return by_rows<256>(a, dtype, tile_rows, S, stream);
}
