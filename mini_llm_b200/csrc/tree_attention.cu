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
// The maximum is kept as a score, and a weight is 2^((s - max) * scale * log2 e): the difference first, so that scores of any size
// give weights up to 1 (a fused s * c - rounded(max * c) leaves a rounding of the maximum's size, which overflows from 2^31 on).
//
// Layout.  The query rows of one key/value head (row r = node r / G, head r % G of its group of G) are packed into tiles of
// RW rows a warp and WR warps.  tree_attention.cuh says how the keys are cut into segments of blocks.  In a block WK groups of WR
// warps take a segment's tiles of BK keys in turn, each with its own running maximum, sum and output rows in registers and ST
// buffers of keys and of values in shared memory: a buffer's next tile is asked for (cp.async) as soon as the product that read it
// is done, the block-table entries one tile further ahead (a lane looks one key's page up and hands it round).  The groups meet in
// order at the end.
//   bfloat16: S = Q K^T and O += P V on mma.sync.m16n8k16, p as two bfloat16 terms (its rounding and what that left out), so the
//             weights keep about 16 bits; sums in 32 bits.
//   float32:  fused multiply-adds of packed pairs on the CUDA cores.  A lane owns RW / 4 rows x 4 keys of S and RW / 4 rows x DP / 8
//             columns of O: every 16 bytes from shared memory feed 8 to 16 of them.
// Values in places that some rows see and others do not (the tree's own) may be infinite or NaN: a weight of zero would turn them
// into NaN, so such elements are taken out of the tile and added to the rows that see them only.
#include "tree_attention.cuh"
#include <type_traits>

namespace {

using namespace tree;

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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// Two fused multiply-adds of neighbouring 32-bit floats in one instruction.
__device__ __forceinline__ void fma2(unsigned long long& c, unsigned long long a, unsigned long long b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}
__device__ __forceinline__ unsigned long long pair_of(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 halves(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
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

constexpr int P_ROW = 36;                                   // float32: a row of weights, padded so that 4 rows start on other banks

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST>
struct Shape {
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int ROW = DP + VEC;                    // padded rows: neighbours start on other banks
    static constexpr int ROWS = RW * WR;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr size_t q_bytes = (size_t)ROWS * ROW * sizeof(T);
    static constexpr size_t kv_bytes = (size_t)WK * ST * 2 * BK * ROW * sizeof(T);
    static constexpr size_t p_bytes = F32 ? (size_t)WK * WR * RW * P_ROW * 4 : 0;
    static constexpr int MN = F32 ? RW / 4 : 2;             // rows whose maximum and sum a thread keeps
    static constexpr int ON = F32 ? RW / 4 * (DP / 8) : DP / 2;
    static constexpr int X_ROW = DP + 8;                    // the groups' results meet as rows of 32-bit floats
    static constexpr size_t xch_bytes = WK > 1 ? (size_t)WK * ROWS * (X_ROW + 2) * 4 : 0;
    static constexpr size_t bytes = q_bytes + (kv_bytes + p_bytes > xch_bytes ? kv_bytes + p_bytes : xch_bytes);
};

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST, int PER_SM>
__global__ void __launch_bounds__(WR * WK * 32, PER_SM)
tree_attention_kernel(const Args a) {
    using S = Shape<T, DP, RW, WR, WK, BK, ST>;
    constexpr int VEC = S::VEC, ROW = S::ROW, CH = DP / VEC, NT = WR * 32, MN = S::MN, ON = S::ON;
    constexpr bool F32 = S::F32;
    using mask_t = typename std::conditional<BK == 32, uint32_t, unsigned long long>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    T* sQ = reinterpret_cast<T*>(smem);
    uint8_t* shared_rest = smem + S::q_bytes;
    const int group = threadIdx.x / NT, gtid = threadIdx.x % NT, warp = gtid >> 5, lane = gtid & 31;
    T* sK = reinterpret_cast<T*>(shared_rest) + (size_t)group * ST * 2 * BK * ROW;      // [ST][BK][ROW]
    T* sV = sK + ST * BK * ROW;
    float* sP = reinterpret_cast<float*>(shared_rest + S::kv_bytes) + (size_t)(group * WR + warp) * RW * P_ROW;

    pdl_wait();
    pdl_launch();
    const int G = a.G;
    const T* k_pages = static_cast<const T*>(a.k_pages);
    const T* v_pages = static_cast<const T*>(a.v_pages);
    const int dh_ch = a.dh / VEC;                           // 16-byte pieces of a row; the rest of DP is zeros

    __shared__ Segments segments;
    if (threadIdx.x == 0) first_segments(&segments);
    for (int number = 0;; ++number) {
        if (number % Segments::CAP == 0) {
            if (number && !segments.more) break;
            __syncthreads();
            if (threadIdx.x < 32) fill(a, &segments);
            __syncthreads();
        }
        if (number % Segments::CAP >= segments.count) break;
        const Segment& sg = segments.list[number % Segments::CAP];
        const int first = sg.first, len = sg.len, keys = sg.keys, rows = sg.rows, r0 = sg.row0, hk = sg.hk, k1 = sg.k1;
        const int* bt = a.block_table + (size_t)sg.s * a.bt_stride;
        const int t_last = (k1 - 1) / BK;                   // units are multiples of a tile
        const bool active = r0 + warp * RW < rows;          // a warp without rows only helps with the copies

        // the queries of this tile of rows
        const T* q = static_cast<const T*>(a.q);
        for (int i = threadIdx.x; i < S::ROWS * CH; i += WR * WK * 32) {
            const int r = i / CH, c = i % CH;
            const bool ok = r0 + r < rows && c < dh_ch;
            const int node = ok ? (r0 + r) / G : 0, h = hk * G + (ok ? (r0 + r) % G : 0);
            const T* src = q + (size_t)(first + node) * a.ldq + (size_t)h * a.dh + c * VEC;
            if (a.q_vec) {
                cp_async16(sQ + r * ROW + c * VEC, ok ? src : q, ok);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) sQ[r * ROW + c * VEC + e] = ok ? src[e] : from_f32<T>(0.f);
            }
        }
        cp_commit();

        // A lane looks up the rows of the tile's keys lane, lane + 32.
        unsigned int row_id[BK / 32];
        auto look_up = [&](int t) {
#pragma unroll
            for (int x = 0; x < BK / 32; ++x) {
                const int kp = t * BK + x * 32 + lane;
                row_id[x] = NO_ROW;
                if (kp < k1) {
                    const int p = a.page_shift >= 0 ? kp >> a.page_shift : kp / a.page_size;
                    row_id[x] = ((unsigned int)bt[p] * a.Hkv + hk) * a.page_size + (kp - p * a.page_size);
                }
            }
        };
        auto load = [&](T* dst, const T* pages) {             // the rows that look_up() brought
#pragma unroll
            for (int it = 0; it < BK * CH / NT; ++it) {
                const int i = gtid + it * NT, r = i / CH, c = i % CH;
                unsigned int id = __shfl_sync(0xffffffffu, row_id[0], r & 31);
                if (BK > 32) {                                // all rows of one step of the loop may lie in one half, or not
                    const unsigned int other = __shfl_sync(0xffffffffu, row_id[BK / 32 - 1], r & 31);
                    id = r >= 32 ? other : id;
                }
                const bool ok = id != NO_ROW && c < dh_ch;
                cp_async16(dst + r * ROW + c * VEC, pages + (ok ? (size_t)id * a.dh + c * VEC : 0), ok);
            }
        };
        int t = sg.k0 / BK + group;
#pragma unroll
        for (int st = 0; st < ST; ++st) {
            look_up(t + st * WK);
            if (t + st * WK <= t_last) load(sK + st * BK * ROW, k_pages);
            cp_commit();
            if (t + st * WK <= t_last) load(sV + st * BK * ROW, v_pages);
            cp_commit();
        }
        look_up(t + ST * WK);
        cp_wait<2 * ST>();                                    // the queries are in
        __syncthreads();

        // ---- running state
        float o[F32 ? 1 : ON];                                // bfloat16: the accumulators' fragments
        unsigned long long o2[F32 ? ON / 2 : 1];              // float32: [MN][DP / 32][2] pairs of columns
#pragma unroll
        for (int i = 0; i < (F32 ? 1 : ON); ++i) o[i] = 0.f;
#pragma unroll
        for (int i = 0; i < (F32 ? ON / 2 : 1); ++i) o2[i] = 0ull;
        float m_run[MN], l_run[MN];
#pragma unroll
        for (int i = 0; i < MN; ++i) { m_run[i] = -INFINITY; l_run[i] = 0.f; }
        const int g = lane >> 2, tq = lane & 3;               // bfloat16: fragment row and column
        const int rg = lane >> 3, kg = lane & 7;              // float32: row and key (or column) of a lane
        uint32_t qa[F32 ? 1 : DP / 16][4];
        if constexpr (!F32) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) ldsm_x4(qa[ks], sQ + (warp * 16 + (lane & 15)) * ROW + ks * 16 + (lane >> 4) * 8);
        }
        auto row_of = [&](int i) { return r0 + warp * RW + (F32 ? rg + 4 * i : g + 8 * i); };      // the query row of a thread's i-th state
        auto words_of = [&](int r) { return a.ancestors + (size_t)(first + (r < rows ? r / G : 0)) * a.words; };

        int stage = 0;
        for (; t <= t_last; t += WK, stage = stage + 1 == ST ? 0 : stage + 1) {
            T* tK = sK + stage * BK * ROW;
            T* tV = sV + stage * BK * ROW;
            const int key0 = t * BK;
            const bool tail = key0 + BK > min(len, keys);     // the tile reaches into the tree or past the keys
            mask_t seen[MN];
            if (tail) {
#pragma unroll
                for (int i = 0; i < MN; ++i)
                    seen[i] = (mask_t)tile_mask(words_of(row_of(i)), a.words, len, keys, key0, row_of(i) < rows);
            }
            cp_wait<2 * ST - 1>();                            // the tile's keys
            group_sync<WR>(group);
            float sc[F32 ? 4 * MN : BK / 2];                  // scores, then weights
            if (active) {
                if constexpr (!F32) {
                    // ---- S = Q K^T: 16 rows x BK keys
#pragma unroll
                    for (int i = 0; i < BK / 2; ++i) sc[i] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
                        for (int np = 0; np < BK / 16; ++np) {
                            uint32_t b[4];
                            ldsm_x4(b, tK + (np * 16 + (lane & 7) + ((lane >> 4) << 3)) * ROW + ks * 16 + ((lane >> 3) & 1) * 8);
                            mma16816(*reinterpret_cast<float (*)[4]>(&sc[8 * np]), qa[ks], b[0], b[1]);
                            mma16816(*reinterpret_cast<float (*)[4]>(&sc[8 * np + 4]), qa[ks], b[2], b[3]);
                        }
                    }
                } else {
                    // ---- S: rows rg + 4 i, keys kg + 8 j; even and odd columns in the halves of a pair
                    unsigned long long s2[MN][4];
#pragma unroll
                    for (int i = 0; i < MN; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s2[i][j] = 0ull;
                    const float* kr = reinterpret_cast<const float*>(tK) + kg * ROW;
                    const float* qr = reinterpret_cast<const float*>(sQ) + (warp * RW + rg) * ROW;
#pragma unroll 4
                    for (int d = 0; d < DP; d += 4) {
                        ulonglong2 qv[MN];
#pragma unroll
                        for (int i = 0; i < MN; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(qr + 4 * i * ROW + d);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const ulonglong2 kv = *reinterpret_cast<const ulonglong2*>(kr + 8 * j * ROW + d);
#pragma unroll
                            for (int i = 0; i < MN; ++i) { fma2(s2[i][j], qv[i].x, kv.x); fma2(s2[i][j], qv[i].y, kv.y); }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MN; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { const float2 h = halves(s2[i][j]); sc[4 * i + j] = h.x + h.y; }
                }
            }
            group_sync<WR>(group);                            // the keys' buffer is free
            if (t + ST * WK <= t_last) load(tK, k_pages);
            cp_commit();

            if (active) {
                // ---- weights, and what they do to the state
                float alpha[MN];
                bool moved = false;
#pragma unroll
                for (int i = 0; i < MN; ++i) {
                    float mx = -INFINITY;
                    if constexpr (F32) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (tail && !(seen[i] >> (kg + 8 * j) & 1)) sc[4 * i + j] = -INFINITY;
                            mx = fmaxf(mx, sc[4 * i + j]);
                        }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    } else {
#pragma unroll
                        for (int nt = 0; nt < BK / 8; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (tail && !(seen[i] >> (nt * 8 + 2 * tq + e) & 1)) sc[4 * nt + 2 * i + e] = -INFINITY;
                                mx = fmaxf(mx, sc[4 * nt + 2 * i + e]);
                            }
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float m_new = fmaxf(m_run[i], mx), use = m_new == -INFINITY ? 0.f : m_new;
                    if constexpr (F32) {
                        alpha[i] = exp2f((m_run[i] - use) * a.scale_log2);
                        float sum = 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float p = exp2f((sc[4 * i + j] - use) * a.scale_log2);
                            sP[(rg + 4 * i) * P_ROW + kg + 8 * j] = p;
                            sum += p;
                        }
                        l_run[i] = l_run[i] * alpha[i] + sum;          // this lane's keys; the lanes meet at the end
                    } else {
                        alpha[i] = fast_exp2((m_run[i] - use) * a.scale_log2);
                        float sum = 0.f;
#pragma unroll
                        for (int nt = 0; nt < BK / 8; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float& p = sc[4 * nt + 2 * i + e];
                                p = fast_exp2((p - use) * a.scale_log2);
                                sum += p;
                            }
                        l_run[i] = l_run[i] * alpha[i] + sum;
                    }
                    moved |= alpha[i] != 1.f;
                    m_run[i] = m_new;
                }
                if (__any_sync(0xffffffffu, moved)) {
                    if constexpr (F32) {
#pragma unroll
                        for (int i = 0; i < MN; ++i)
#pragma unroll
                            for (int c = 0; c < DP / 16; ++c) {
                                const float2 h = halves(o2[i * (DP / 16) + c]);
                                o2[i * (DP / 16) + c] = pair_of(h.x * alpha[i], h.y * alpha[i]);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < ON; ++i) o[i] *= alpha[i >> 1 & 1];
                    }
                }
            }

            cp_wait<2 * ST - 1>();                            // the tile's values
            bool odd = false;
            if (tail) {
                // infinite and NaN values of the tree: taken out before the group reads the tile
                group_sync<WR>(group);
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
            }
            group_sync<WR>(group);
            if (active) {
                // ---- O += P V
                if constexpr (!F32) {
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk) {
                        uint32_t pa[4], pb[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p0 = sc[8 * kk + 2 * e], p1 = sc[8 * kk + 2 * e + 1];
                            pa[e] = pack_bf16(p0, p1);
                            pb[e] = pack_bf16(p0 - __uint_as_float(pa[e] << 16), p1 - __uint_as_float(pa[e] & 0xffff0000u));
                        }
#pragma unroll
                        for (int dp = 0; dp < DP / 16; ++dp) {
                            uint32_t b[4];
                            ldsm_x4_trans(b, tV + (kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * ROW + dp * 16 + (lane >> 4) * 8);
                            float (&c0)[4] = *reinterpret_cast<float (*)[4]>(&o[8 * dp]);
                            float (&c1)[4] = *reinterpret_cast<float (*)[4]>(&o[8 * dp + 4]);
                            mma16816(c0, pa, b[0], b[1]);
                            mma16816(c1, pa, b[2], b[3]);
                            mma16816(c0, pb, b[0], b[1]);
                            mma16816(c1, pb, b[2], b[3]);
                        }
                    }
                } else {
                    __syncwarp();
                    const float* vr = reinterpret_cast<const float*>(tV) + kg * 4;
                    const float* pr = sP + rg * P_ROW;
#pragma unroll 2
                    for (int k = 0; k < BK; k += 4) {
                        float4 p[MN];
#pragma unroll
                        for (int i = 0; i < MN; ++i) p[i] = *reinterpret_cast<const float4*>(pr + 4 * i * P_ROW + k);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            unsigned long long pp[MN];
#pragma unroll
                            for (int i = 0; i < MN; ++i) {
                                const float x = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                                pp[i] = pair_of(x, x);
                            }
#pragma unroll
                            for (int c = 0; c < DP / 32; ++c) {
                                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(vr + (k + e) * ROW + c * 32);
#pragma unroll
                                for (int i = 0; i < MN; ++i) {
                                    fma2(o2[i * (DP / 16) + 2 * c], pp[i], v.x);
                                    fma2(o2[i * (DP / 16) + 2 * c + 1], pp[i], v.y);
                                }
                            }
                        }
                    }
                }
                if (tail && odd) {
                    // infinite and NaN elements, from memory, to the rows that see them
                    for (int b = max(0, len - key0); b < min(BK, k1 - key0); ++b) {
                        const int kp = key0 + b, p = kp / a.page_size;
                        const T* vrow = v_pages + (((size_t)bt[p] * a.Hkv + hk) * a.page_size + kp % a.page_size) * a.dh;
#pragma unroll
                        for (int i = 0; i < MN; ++i) {
                            if (!(seen[i] >> b & 1)) continue;
#pragma unroll
                            for (int e = 0; e < (F32 ? DP / 16 : DP / 8); ++e) {
                                const int d = F32 ? (e >> 1) * 32 + kg * 4 + 2 * (e & 1) : e * 8 + 2 * tq;
                                if (d >= a.dh) continue;
                                float x = to_f32(vrow[d]), y = to_f32(vrow[d + 1]);
                                x = fabsf(x) < INFINITY ? 0.f : x;
                                y = fabsf(y) < INFINITY ? 0.f : y;
                                if constexpr (F32) {
                                    const float2 h = halves(o2[i * (DP / 16) + e]);
                                    o2[i * (DP / 16) + e] = pair_of(h.x + x, h.y + y);
                                } else {
                                    o[e * 4 + 2 * i] += x;
                                    o[e * 4 + 2 * i + 1] += y;
                                }
                            }
                        }
                    }
                }
            }
            group_sync<WR>(group);                            // the values' buffer is free
            if (t + ST * WK <= t_last) load(tV, v_pages);
            cp_commit();
            look_up(t + (ST + 1) * WK);
        }
        cp_wait<0>();
        // the lanes' shares of the sums
#pragma unroll
        for (int i = 0; i < MN; ++i) {
            if (F32) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 4);
            l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
            l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
        }
        float res[ON];                                        // [MN][columns], a pair of neighbours after the other
#pragma unroll
        for (int i = 0; i < MN; ++i)
#pragma unroll
            for (int e = 0; e < ON / MN / 2; ++e) {
                if constexpr (F32) {
                    const float2 h = halves(o2[i * (DP / 16) + e]);
                    res[i * (ON / MN) + 2 * e] = h.x;
                    res[i * (ON / MN) + 2 * e + 1] = h.y;
                } else {
                    res[i * (ON / MN) + 2 * e] = o[e * 4 + 2 * i];
                    res[i * (ON / MN) + 2 * e + 1] = o[e * 4 + 2 * i + 1];
                }
            }
        // ---- out: a thread's own elements where the block is one group; else the groups' rows meet in shared memory, in order, and
        // every thread finishes neighbours of a row
        auto put = [&](int r, int d, float x, float y, float m, float l, bool first_of_row) {
            if (sg.slot >= 0) {
                const size_t pr = (size_t)sg.slot * a.tile_rows + (r - r0);
                if (first_of_row) *reinterpret_cast<float2*>(a.part_ml + 2 * pr) = make_float2(m, l);
                *reinterpret_cast<float2*>(a.part_o + pr * a.dh + d) = make_float2(x, y);
                return;
            }
            const float inv = inverse_sum(l);
            T* orow = static_cast<T*>(a.out) + (size_t)(first + r / G) * a.ldo + (size_t)(hk * G + r % G) * a.dh;
            if (F32 && a.out_vec >= 2) *reinterpret_cast<float2*>(orow + d) = make_float2(x * inv, y * inv);
            else if (!F32 && a.out_vec >= 2) *reinterpret_cast<uint32_t*>(orow + d) = pack_bf16(x * inv, y * inv);
            else { orow[d] = from_f32<T>(x * inv); orow[d + 1] = from_f32<T>(y * inv); }
        };
        if constexpr (WK > 1) {
            constexpr int X = S::X_ROW;
            float* xch = reinterpret_cast<float*>(shared_rest);            // [WK][ROWS][X], then maxima and sums [WK][ROWS][2]
            float* xml = xch + WK * S::ROWS * X;
            __syncthreads();
            if (active) {
#pragma unroll
                for (int i = 0; i < MN; ++i) {
                    const int r = group * S::ROWS + row_of(i) - r0;
                    if ((F32 ? kg : tq) == 0) *reinterpret_cast<float2*>(xml + 2 * r) = make_float2(m_run[i], l_run[i]);
#pragma unroll
                    for (int e = 0; e < ON / MN / 2; ++e) {
                        const int d = F32 ? (e >> 1) * 32 + kg * 4 + 2 * (e & 1) : e * 8 + 2 * tq;
                        *reinterpret_cast<float2*>(xch + r * X + d) = make_float2(res[i * (ON / MN) + 2 * e], res[i * (ON / MN) + 2 * e + 1]);
                    }
                }
            }
            __syncthreads();
            const int pairs = a.dh / 2, here = min(S::ROWS, rows - r0);
            for (int i = threadIdx.x; i < here * pairs; i += WR * WK * 32) {
                const int r = i / pairs, d = 2 * (i % pairs);
                float2 ml[WK];
                float m = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    ml[w] = *reinterpret_cast<const float2*>(xml + 2 * (w * S::ROWS + r));
                    m = fmaxf(m, ml[w].x);
                }
                const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    const float f = exp2f((ml[w].x - use) * a.scale_log2);
                    const float2 v = *reinterpret_cast<const float2*>(xch + (w * S::ROWS + r) * X + d);
                    l = fmaf(ml[w].y, f, l);
                    x = fmaf(v.x, f, x);
                    y = fmaf(v.y, f, y);
                }
                put(r0 + r, d, x, y, m, l, d == 0);
            }
        } else if (active) {
#pragma unroll
            for (int i = 0; i < MN; ++i) {
                const int r = row_of(i);
                if (r >= rows) continue;
#pragma unroll
                for (int e = 0; e < ON / MN / 2; ++e) {
                    const int d = F32 ? (e >> 1) * 32 + kg * 4 + 2 * (e & 1) : e * 8 + 2 * tq;
                    if (d < a.dh) put(r, d, res[i * (ON / MN) + 2 * e], res[i * (ON / MN) + 2 * e + 1], m_run[i], l_run[i], d == 0);
                }
            }
        }
        __syncthreads();                                      // shared memory is free for the next segment
    }
}

// The segments of the pairs that more than one block worked on meet, in order of position: a block per boundary between two blocks'
// shares (the first one inside a pair does the pair) and four rows of the tile, a warp per row.  VD: columns of a lane.
// Four segments' rows are in flight at once.
template <typename T, int VD>
__global__ void __launch_bounds__(128)
tree_attention_join_kernel(const Args a) {
    pdl_wait();
    pdl_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.G;
    const Line line = line_of(a);
    const unsigned int c = blockIdx.x + 1, u = line.begin(c);
    if (u >= line.units || line.begin(c - 1) == u) return;          // nothing behind the boundary, or the one before says the same
    unsigned int base;
    const Request r = find(a, line, u, &base);
    const unsigned int pair = (u - base) / r.units, from = base + pair * r.units;
    if (from == u || line.begin(c - 1) > from) return;              // between two pairs, or not the pair's first boundary
    const int hk = (int)(pair / r.tiles), tile = (int)(pair % r.tiles);
    const unsigned int c0 = c - 1, c1 = line.block_of(from + r.units - 1);
    const int parts = (int)(c1 - c0) + 1;
    const unsigned int shift = line.begin(c0) < from ? 1 : 0;       // block c0's segment is its last one, unless it begins here
    const int here_rows = min(a.tile_rows, r.n * G - tile * a.tile_rows);
    for (int row = blockIdx.y * 4 + warp; row < here_rows; row += gridDim.y * 4) {
        auto at = [&](int p) { return (size_t)(2 * (c0 + p) + (p == 0 ? shift : 0)) * a.tile_rows + row; };
        float m = -INFINITY, l = 0.f, o[VD];
#pragma unroll
        for (int x = 0; x < VD; ++x) o[x] = 0.f;
        for (int p0 = 0; p0 < parts; p0 += 32) {
            float2 ml = make_float2(-INFINITY, 0.f);
            if (p0 + lane < parts) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at(p0 + lane));
            const float m_new = fmaxf(m, warp_max(ml.x)), use = m_new == -INFINITY ? 0.f : m_new;
            const float keep = exp2f((m - use) * a.scale_log2), w = exp2f((ml.x - use) * a.scale_log2);
            m = m_new;
            l = l * keep + warp_sum(ml.y * w);
#pragma unroll
            for (int x = 0; x < VD; ++x) o[x] *= keep;
            const int here = min(32, parts - p0);
            for (int k = 0; k < here; k += 4) {
                float v[4][VD], we[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    we[e] = __shfl_sync(0xffffffffu, w, (k + e) & 31);
                    const float* po = a.part_o + at(p0 + min(k + e, here - 1)) * a.dh;
#pragma unroll
                    for (int x = 0; x < VD; ++x) v[e][x] = x * 32 + lane < a.dh ? po[x * 32 + lane] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + e < here && we[e] != 0.f) {
#pragma unroll
                        for (int x = 0; x < VD; ++x) o[x] = fmaf(v[e][x], we[e], o[x]);
                    }
            }
        }
        const float inv = inverse_sum(l);
        const int q = tile * a.tile_rows + row;
        T* orow = static_cast<T*>(a.out) + (size_t)(r.first + q / G) * a.ldo + (size_t)(hk * G + q % G) * a.dh;
#pragma unroll
        for (int x = 0; x < VD; ++x)
            if (x * 32 + lane < a.dh) orow[x * 32 + lane] = from_f32<T>(o[x] * inv);
    }
}
template <typename T>
int launch_join(const Args& a, cudaStream_t stream) {
    if (a.blocks < 2) return 0;
    const dim3 grid(a.blocks - 1, (a.max_rows + 3) / 4);
    if (a.dh <= 32) MLLM_CUDA(mllm_launch(tree_attention_join_kernel<T, 1>, grid, dim3(128), 0, stream, true, a));
    else if (a.dh <= 64) MLLM_CUDA(mllm_launch(tree_attention_join_kernel<T, 2>, grid, dim3(128), 0, stream, true, a));
    else if (a.dh <= 128) MLLM_CUDA(mllm_launch(tree_attention_join_kernel<T, 4>, grid, dim3(128), 0, stream, true, a));
    else MLLM_CUDA(mllm_launch(tree_attention_join_kernel<T, 8>, grid, dim3(128), 0, stream, true, a));
    return 0;
}

template <typename T, int DP, int RW, int WR, int WK, int BK, int ST, int PER_SM>
int launch(const Args& a, cudaStream_t stream) {
    using Sh = Shape<T, DP, RW, WR, WK, BK, ST>;
    static_assert(Sh::bytes + sizeof(Segments) <= 232448 && (Sh::bytes + sizeof(Segments) + 1024) * PER_SM <= 233472, "shared memory of an SM");
    auto kern = tree_attention_kernel<T, DP, RW, WR, WK, BK, ST, PER_SM>;
    static bool set = false;
    if (!set && Sh::bytes > 48 * 1024) {
        MLLM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::bytes));
        set = true;
    }
    MLLM_CUDA(mllm_launch(kern, grid_of(a), dim3(WR * WK * 32), Sh::bytes, stream, true, a));
    return a.blocks ? join(a, sizeof(T) == 4 ? MLLM_F32 : MLLM_BF16, stream) : 0;
}

// Blocks of a variant that an SM holds at once: what the work is shared among (mllm_tree_attention_per_sm).
template <int DP>
int by_rows(const Args* a, int dtype, int tile_rows, bool wide, int* per_sm, cudaStream_t stream) {
    using bf = __nv_bfloat16;
#define GO(T, RW, WR, WK, BK, ST, PER)                                                      \
    do {                                                                                    \
        if (per_sm) { *per_sm = PER; return 0; }                                            \
        return launch<T, DP, RW, WR, WK, BK, ST, PER>(*a, stream);                          \
    } while (0)
    if (dtype == MLLM_BF16) {
        if constexpr (DP <= 64) {
            if (tile_rows == 16 && wide) GO(bf, 16, 1, 8, 64, 1, 1);
            if (tile_rows == 16) GO(bf, 16, 1, 4, 64, 1, 3);
            if (tile_rows == 32) GO(bf, 16, 2, 4, 32, 2, 2);
            if (tile_rows == 64) GO(bf, 16, 4, 2, 32, 3, 2);
        } else if constexpr (DP == 128) {
            if (tile_rows == 16) GO(bf, 16, 1, 4, 32, 1, 2);
            if (tile_rows == 32) GO(bf, 16, 2, 2, 32, 2, 2);
            if (tile_rows == 64) GO(bf, 16, 4, 2, 32, 2, 1);
        } else {
            if (tile_rows == 16) GO(bf, 16, 1, 4, 32, 1, 1);
            if (tile_rows == 32) GO(bf, 16, 2, 4, 32, 1, 1);
            if (tile_rows == 64) GO(bf, 16, 4, 2, 32, 2, 1);
        }
    } else {
        if constexpr (DP <= 64) {
            if (tile_rows == 4) GO(float, 4, 1, 4, 32, 1, 3);
            if (tile_rows == 8) GO(float, 8, 1, 4, 32, 1, 3);
            if (tile_rows == 16) GO(float, 16, 1, 4, 32, 1, 2);
            if (tile_rows == 32) GO(float, 16, 2, 4, 32, 1, 2);
            if (tile_rows == 64) GO(float, 16, 4, 2, 32, 1, 2);
        } else if constexpr (DP == 128) {
            if (tile_rows == 4) GO(float, 4, 1, 3, 32, 1, 2);
            if (tile_rows == 8) GO(float, 8, 1, 3, 32, 1, 2);
            if (tile_rows == 16) GO(float, 16, 1, 4, 32, 1, 1);
            if (tile_rows == 32) GO(float, 16, 2, 4, 32, 1, 1);
            if (tile_rows == 64) GO(float, 16, 4, 2, 32, 1, 1);
        } else {
            if (tile_rows == 4) GO(float, 4, 1, 3, 32, 1, 1);
            if (tile_rows == 8) GO(float, 8, 1, 3, 32, 1, 1);
            if (tile_rows == 16) GO(float, 16, 1, 2, 32, 1, 1);
            if (tile_rows == 32) GO(float, 16, 2, 2, 32, 1, 1);
            if (tile_rows == 64) GO(float, 16, 4, 1, 32, 1, 1);
        }
    }
#undef GO
    return mllm_fail(1, "tree_attention: no kernel takes tiles of %d rows", tile_rows);
}
int by_head(const Args* a, int dh, int dtype, int tile_rows, bool wide, int* per_sm, cudaStream_t stream) {
    if (dh <= 32) return by_rows<32>(a, dtype, tile_rows, wide, per_sm, stream);
    if (dh <= 64) return by_rows<64>(a, dtype, tile_rows, wide, per_sm, stream);
    if (dh <= 128) return by_rows<128>(a, dtype, tile_rows, wide, per_sm, stream);
    return by_rows<256>(a, dtype, tile_rows, wide, per_sm, stream);
}

}  // namespace

int tree::join(const Args& a, int dtype, cudaStream_t stream) {
    return dtype == MLLM_F32 ? launch_join<float>(a, stream) : launch_join<__nv_bfloat16>(a, stream);
}

// Blocks of a tile size that one SM holds at once; 0: no kernel takes it.
MLLM_EXPORT int mllm_tree_attention_per_sm(int dh, int tile_rows, int dtype) {
    int per_sm = 0;
    if (dtype == MLLM_BF16 && tile_rows >= 128) return 1;
    return by_head(nullptr, dh, dtype, tile_rows, false, &per_sm, nullptr) ? 0 : per_sm;
}

// tile_rows: 128 or 256 (bfloat16, the kernel of tree_attention_tcgen05.cu), 16, 32 or 64 (bfloat16), 4, 8, 16, 32 or 64 (float32) query rows of a key/value head per tile; max_rows: those of
// the largest tree (as far as the host knows).  blocks: those that share all keys evenly, in units of `unit` keys (a power of two from 64 on); they
// need part_o [2 * blocks, tile_rows, dh] and part_ml [2 * blocks, tile_rows, 2].  0: a block for every pair of tile and head.
// The head size is a multiple of 16 up to 256.
MLLM_EXPORT int mllm_tree_attention(const void* q, long long ldq, const void* k_pages, const void* v_pages, long long pages,
                                    const int* block_table, int bt_stride, int width, const int* lengths, const int* cu_nodes,
                                    const int* ancestors, int words, void* out, long long ldo, float* part_o, float* part_ml, int S,
                                    int H, int Hkv, int dh, int page_size, float scale, int tile_rows, int max_rows, int unit,
                                    int blocks, int wide, int dtype, cudaStream_t stream) {
    if (S <= 0) return 0;
    if (Hkv <= 0 || H % Hkv != 0) return mllm_fail(1, "tree_attention: %d heads over %d key/value heads", H, Hkv);
    if (dh < 16 || dh > 256 || dh % 16) return mllm_fail(1, "tree_attention: head size %d is not a multiple of 16 in 16..256", dh);
    if (!(scale > 0.f)) return mllm_fail(1, "tree_attention: the score scale must be positive, got %g", (double)scale);
    if (dtype != MLLM_F32 && dtype != MLLM_BF16) return mllm_fail(1, "tree_attention: unknown dtype code %d", dtype);
    if (page_size <= 0 || width <= 0 || words <= 0 || unit < 64 || (unit & (unit - 1)) || blocks < 0 || max_rows <= 0 || tile_rows <= 0 ||
        (tile_rows & (tile_rows - 1)))
        return mllm_fail(1, "tree_attention: pages of %d, a table of %d columns, %d words, units of %d keys, %d blocks, %d rows", page_size,
                         width, words, unit, blocks, max_rows);
    const int max_tiles = (max_rows + tile_rows - 1) / tile_rows;
    if (pages * Hkv * page_size >= (long long)NO_ROW)
        return mllm_fail(1, "tree_attention: a pool of %lld rows of keys is more than 32-bit row numbers hold", pages * Hkv * page_size);
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) % 16) return mllm_fail(1, "tree_attention: pages must be 16-byte aligned");
    if (Hkv > 65535 || S > 65535 || (long long)Hkv * max_tiles > 0x7fffffffLL)
        return mllm_fail(1, "tree_attention: %d requests of %d tiles of %d heads are more than one launch takes", S, max_tiles, Hkv);
    if (blocks && (!part_o || !part_ml)) return mllm_fail(1, "tree_attention: keys shared among %d blocks need scratch to meet in", blocks);
    const int es = dtype == MLLM_F32 ? 4 : 2;
    int shift = -1;
    for (int b = 0; b < 31; ++b)
        if (page_size == 1 << b) shift = b;
    const int tile_shift = 31 - __builtin_clz(tile_rows), unit_shift = 31 - __builtin_clz(unit);
    int out_vec = 1;
    while (out_vec < 8 && (uintptr_t)out % (2 * out_vec * es) == 0 && ldo % (2 * out_vec) == 0) out_vec *= 2;
    const Args a{q, ldq, k_pages, v_pages, block_table, bt_stride, width, lengths, cu_nodes, ancestors, words, out, ldo, part_o,
                 part_ml, S, H, Hkv, H / Hkv, dh, page_size, shift, (uintptr_t)q % 16 == 0 && ldq * es % 16 == 0,
                 out_vec, tile_rows, tile_shift, max_rows < tile_rows ? max_rows : tile_rows, unit_shift, blocks, max_tiles, scale * LOG2E};
    if (dtype == MLLM_BF16 && tile_rows >= 128) return tcgen05(a, pages, stream);
    return by_head(&a, dh, dtype, tile_rows, wide != 0, nullptr, stream);
}
