// Attention of a few rows at a time over the paged cache in its 8-bit forms (kv8.cuh) or in bfloat16, and the write of the
// 8-bit forms; compiled for one head size: -DOE_HD=64 or 128.
//
// A row is a (token, query head of the group) pair.  A CTA (or a cluster of CTAs) has 16 rows of one KV head and a range of
// keys; its warps split the keys in tiles of 32, each with a ring of tiles of its own that cp.async fills and a running
// softmax of its own, and the results are added up in warp order, then in rank order, through shared memory.
//   S = Q K^T, O += P V     mma.sync m16n8k16 with float32 sums.
//     8-bit forms           float16: a code is a float16 exactly, so K and V enter as codes.  The turned queries are rounded to float16
//                           (2^-12 of themselves; a row is scaled by a power of two first), the key's scale multiplies the score's
//                           sum, and the weight p times the value's scale is rounded to float16: relative to R, the largest power of
//                           two above a value's scale so far, and times 2^8, so that what float16 cannot hold is below 2^-33 of the
//                           row's largest weight.  When R grows, O is scaled down with the step that a grown maximum takes anyway.
//     bfloat16              K and V as they are.  Turned queries and weights enter as the sum of two bfloat16 (2^-17 of themselves), which
//                           costs a second product each in a kernel that waits for memory.
//   Fragments               the dimensions of a product's inner axis and the columns of its result may be in any order that both
//                           operands keep, so a lane takes 4 dimensions of a row that lie together: K needs one 32-bit load of
//                           codes a k-step, V one for 4 dimensions of each of 4 keys, whose bytes are paired by permutes.
// Masks: key <= the row's position; window > 0 the last `window` keys, window < 0 the keys of the row's chunk.  A masked key's weight is
// set to zero whatever its score and scale are, so rows behind the last token of a page may hold anything.
// A page number outside the cache counts as a page without keys.
#include "kv8.cuh"

#ifndef OE_HD
#define OE_HD 128
#endif

namespace {

constexpr int HD = OE_HD;
static_assert(HD == 64 || HD == 128, "built for head_dim 64 or 128");
constexpr int KS = HD / 16;
constexpr int TB = 32;                           // keys per tile: half a page
constexpr int PARTS = OE_PAGE / TB;
constexpr float LOG2E = 1.4426950408889634f;

// ------------------------------------------------------------------------------------------------ the write
// keys and values of a step's tokens into the 8-bit cache.  HD / 16 lanes have a row: 8 dimensions of its lower half and the 8 that
// they are turned with.
template <int KIND>
__global__ void __launch_bounds__(256)
kv8_write_kernel(const bf16* qkv, long long stride, const float* __restrict__ cos_tab, const float* __restrict__ sin_tab,
                 uint8_t* codes, float* scales, long long n_pages, const int* __restrict__ tables, int max_pages,
                 const int* __restrict__ tok_seq, const int* __restrict__ tok_pos, int n_tokens, int H, int KVH) {
    constexpr int LANES = HD / 16;
    pdl_wait();
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long r = item / LANES;                        // (token, K or V, KV head)
    const int i = (int)(item % LANES) * 8;
    const long long per_token = 2 * KVH;
    const long long t = r / per_token;
    const int which = (int)(r % per_token) / KVH, kvh = (int)(r % KVH);
    const bool here = t < n_tokens;
    const int b = here ? tok_seq[t] : -1;
    const int pos = b >= 0 ? tok_pos[t] : 0;
    const int page = b >= 0 && pos / OE_PAGE < max_pages ? tables[(long long)b * max_pages + pos / OE_PAGE] : -1;
    const bool ok = page >= 0 && page < n_pages;
    uint32_t lo[4] = {0, 0, 0, 0}, hi[4] = {0, 0, 0, 0};
    if (ok) {
        const bf16* row = qkv + t * stride + (long long)(H + which * KVH + kvh) * HD;
        const uint4 a = *(const uint4*)(row + i), c = *(const uint4*)(row + i + HD / 2);
        lo[0] = a.x; lo[1] = a.y; lo[2] = a.z; lo[3] = a.w;
        hi[0] = c.x; hi[1] = c.y; hi[2] = c.z; hi[3] = c.w;
        if (which == 0 && cos_tab != nullptr) {
            const float* cs = cos_tab + (long long)pos * (HD / 2) + i;
            const float* sn = sin_tab + (long long)pos * (HD / 2) + i;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t nl = 0, nh = 0;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float x0 = kv8_from_bits((lo[j] >> (16 * e)) & 0xffffu), x1 = kv8_from_bits((hi[j] >> (16 * e)) & 0xffffu);
                    const float c1 = cs[2 * j + e], s1 = sn[2 * j + e];
                    nl |= kv8_turned_bits(x0, c1, x1, s1) << (16 * e);
                    nh |= kv8_turned_bits(x0, s1, -x1, c1) << (16 * e);
                }
                lo[j] = nl;
                hi[j] = nh;
            }
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        m = max(m, max(lo[j] & 0x7fffu, (lo[j] >> 16) & 0x7fffu));
        m = max(m, max(hi[j] & 0x7fffu, (hi[j] >> 16) & 0x7fffu));
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (ok) {
        const Kv8Row q = kv8_row<KIND>(m);
        uint32_t w[4];
    #pragma unroll
        for (int j = 0; j < 4; j += 2) {
            w[j / 2] = kv8_code<KIND>(q, lo[j] & 0xffffu) | kv8_code<KIND>(q, lo[j] >> 16) << 8 |
                       kv8_code<KIND>(q, lo[j + 1] & 0xffffu) << 16 | kv8_code<KIND>(q, lo[j + 1] >> 16) << 24;
            w[2 + j / 2] = kv8_code<KIND>(q, hi[j] & 0xffffu) | kv8_code<KIND>(q, hi[j] >> 16) << 8 |
                           kv8_code<KIND>(q, hi[j + 1] & 0xffffu) << 16 | kv8_code<KIND>(q, hi[j + 1] >> 16) << 24;
    }
        const long long at = (((long long)page * 2 + which) * KVH + kvh) * OE_PAGE + pos % OE_PAGE;
        *(uint2*)(codes + at * HD + i) = make_uint2(w[0], w[1]);
        *(uint2*)(codes + at * HD + i + HD / 2) = make_uint2(w[2], w[3]);
        if (i == 0) scales[at] = q.scale;
    }
    // the kernel behind this one may ask for these rows before it waits
    __threadfence();
    pdl_launch_dependents();
}

// ------------------------------------------------------------------------------------------------ the attention
struct Args {
    bf16* out;                 // [T, H*HD]
    const bf16* q;             // rows of q_stride elements: the projections, queries first, not yet turned
    long long q_stride;
    const float* cos_tab;      // [max_pos, HD/2] or null
    const float* sin_tab;
    const void* cache;         // one cache entry's codes, or its bfloat16 rows
    const float* scales;       // of the 8-bit forms
    void* cache_w;             // the same two, where this kernel writes the step's new keys and values (one token a sequence); else null
    float* scales_w;
    long long n_pages;
    const int* tables;         // [B, max_pages]
    int max_pages;
    const int* cu_q;           // [B+1] first packed row of each sequence
    const int* seq_start;      // [B] cache length before the step
    const int* seq_qlen;       // [B]
    int H, KVH, window;
    float scale_log2;
    int cluster;               // CTAs that share a tile of rows
    int ahead;                 // rows of earlier tokens may be read before the wait
    // sequences that begin with the same pages: what attention_rows.cu has left of those pages
    const int* seq_pages;      // [B] pages of the sequence's prefix (0: none); null: no prefixes
    int splits;
    const float* part_o;       // [B * H, splits, HD]
    const float* part_ml;      // [B * H, splits, 2]
};

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t*)&h;
}
// What pack_bf16(lo, hi) = h leaves of the two, again as bfloat16.
__device__ __forceinline__ uint32_t rest_bf16(float lo, float hi, uint32_t h) {
    return pack_bf16(lo - __uint_as_float(h << 16), hi - __uint_as_float(h & 0xffff0000u));
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster calls it.
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float ld_peer_f32(const float* p, uint32_t rank) {
    uint32_t addr;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// A tile of 32 keys in shared memory: rows padded so that the loads of a fragment fall into different banks.
template <int KIND>
struct Tile {
    static constexpr int ELEM = KIND == OE_KV_BF16 ? 2 : 1;
    static constexpr int K_ROW = HD * ELEM + (KIND == OE_KV_BF16 ? 32 : 16), V_ROW = HD * ELEM + 16;
    static constexpr int V_AT = TB * K_ROW, S_AT = V_AT + TB * V_ROW;         // S: 32 scales of keys, 32 of values
    static constexpr int BYTES = S_AT + (KIND == OE_KV_BF16 ? 0 : 2 * TB * 4);
};

template <int KIND>
__device__ __forceinline__ void load_tile(uint8_t* st, const Args& a, int page, int part, int kvh, int lane) {
    using L = Tile<KIND>;
    if ((unsigned)page < (unsigned long long)a.n_pages) {
        const long long krow = (((long long)page * 2) * a.KVH + kvh) * OE_PAGE + part * TB, vrow = krow + (long long)a.KVH * OE_PAGE;
        constexpr int PER_ROW = HD * L::ELEM / 16;
        const uint8_t* kg = (const uint8_t*)a.cache + krow * (HD * L::ELEM);
        const uint8_t* vg = (const uint8_t*)a.cache + vrow * (HD * L::ELEM);
#pragma unroll
        for (int c0 = 0; c0 < TB * PER_ROW; c0 += 32) {
            const int c = c0 + lane, row = c / PER_ROW, col = c % PER_ROW;
            cp_async16(st + row * L::K_ROW + col * 16, kg + (size_t)c * 16);
            cp_async16(st + L::V_AT + row * L::V_ROW + col * 16, vg + (size_t)c * 16);
        }
        if (KIND != OE_KV_BF16 && lane < 2 * TB / 4)
            cp_async16(st + L::S_AT + lane * 16, a.scales + (lane < TB / 4 ? krow : vrow - TB) + lane * 4);
    }
}

__device__ __forceinline__ int page_at(const int* trow, int j, int max_pages) { return j < max_pages ? trow[j] : -1; }

// The new token's key and value, made by one warp: its cache rows' bytes, PP pairs (d, d + HD/2) a lane at d = PP lane.
template <int KIND>
struct NewToken {
    static constexpr int PP = HD / 64;
    uint32_t k0[PP], k1[PP], v0[PP], v1[PP];       // bfloat16 bits, or codes
    float ks, vs;
    __device__ __forceinline__ void make(const Args& a, const bf16* row, int pos, int kvh, int lane) {
        const bf16* kr = row + (size_t)(a.H + kvh) * HD;
        const bf16* vr = kr + (size_t)a.KVH * HD;
        uint32_t mk = 0, mv = 0;
#pragma unroll
        for (int u = 0; u < PP; u++) {
            const int d = lane * PP + u;
            k0[u] = __bfloat16_as_ushort(kr[d]); k1[u] = __bfloat16_as_ushort(kr[d + HD / 2]);
            v0[u] = __bfloat16_as_ushort(vr[d]); v1[u] = __bfloat16_as_ushort(vr[d + HD / 2]);
            if (a.cos_tab != nullptr) {
                const float c = a.cos_tab[(size_t)pos * (HD / 2) + d], s = a.sin_tab[(size_t)pos * (HD / 2) + d];
                const float x0 = kv8_from_bits(k0[u]), x1 = kv8_from_bits(k1[u]);
                k0[u] = kv8_turned_bits(x0, c, x1, s);
                k1[u] = kv8_turned_bits(x0, s, -x1, c);
            }
            mk = max(mk, max(k0[u] & 0x7fffu, k1[u] & 0x7fffu));
            mv = max(mv, max(v0[u] & 0x7fffu, v1[u] & 0x7fffu));
        }
        if (KIND != OE_KV_BF16) {
            const Kv8Row qk = kv8_row<KIND>(__reduce_max_sync(0xffffffffu, mk)), qv = kv8_row<KIND>(__reduce_max_sync(0xffffffffu, mv));
#pragma unroll
            for (int u = 0; u < PP; u++) {
                k0[u] = kv8_code<KIND>(qk, k0[u]); k1[u] = kv8_code<KIND>(qk, k1[u]);
                v0[u] = kv8_code<KIND>(qv, v0[u]); v1[u] = kv8_code<KIND>(qv, v1[u]);
            }
            ks = qk.scale; vs = qv.scale;
        }
    }
    __device__ __forceinline__ void store(uint8_t* krow, uint8_t* vrow, int lane) const {
#pragma unroll
        for (int u = 0; u < PP; u++) {
            const int d = lane * PP + u;
            if (KIND == OE_KV_BF16) {
                ((uint16_t*)krow)[d] = (uint16_t)k0[u]; ((uint16_t*)krow)[d + HD / 2] = (uint16_t)k1[u];
                ((uint16_t*)vrow)[d] = (uint16_t)v0[u]; ((uint16_t*)vrow)[d + HD / 2] = (uint16_t)v1[u];
            } else {
                krow[d] = (uint8_t)k0[u]; krow[d + HD / 2] = (uint8_t)k1[u];
                vrow[d] = (uint8_t)v0[u]; vrow[d + HD / 2] = (uint8_t)v1[u];
            }
        }
    }
};

// The rows are those of one sequence's new tokens (blockIdx.z), the keys its own, from behind its prefix on if it has one, whose
// parts are joined with the result.
template <int KIND, int NW, int ST>
__global__ void __launch_bounds__(NW * 32)
attn_kv8_kernel(const Args a) {
    using L = Tile<KIND>;
    constexpr int WARP_BYTES = ST * L::BYTES;
    static_assert((NW + 1) * 16 * (HD + 2) * 4 <= NW * WARP_BYTES, "the parts lie where the rings were");
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.H / a.KVH, kvh = blockIdx.y;
    const int CR = a.cluster, rank = CR > 1 ? (int)cluster_ctarank() : 0;
    const int bx = blockIdx.x / CR;
    const int b = blockIdx.z, row0 = bx * 16, qlen = a.seq_qlen[b], n_rows = qlen > 0 ? qlen * G : 0;
    if (row0 >= n_rows) {                                            // the whole cluster
        pdl_wait();
        return;
    }
    const int start = a.seq_start[b];
    const long long packed0 = a.cu_q[b];
    int key_lo = oe_first_key(start + row0 / G, a.window);
    const int key_hi = start + min(row0 + 15, n_rows - 1) / G;
    const int common = a.seq_pages != nullptr ? a.seq_pages[b] : 0;
    key_lo = max(key_lo, common * OE_PAGE);
    const int* trow = a.tables + (size_t)b * a.max_pages;
    uint8_t* mine = smem + (size_t)warp * WARP_BYTES;
    const int gw = rank * NW + warp, stride = NW * CR;
    const int t_lo = key_lo / TB, t_hi = key_hi >= key_lo ? key_hi / TB : t_lo - 1;
    const int n_my = t_lo + gw <= t_hi ? (t_hi - t_lo - gw) / stride + 1 : 0;
    const bool own_kv = a.cache_w != nullptr;
    // where the caller says so, keys and values of earlier steps are asked for before the wait: only the new token's q, k and v
    // come from the kernel before this one
    const bool ahead = a.ahead && own_kv;
    if (!ahead) pdl_wait();
#pragma unroll
    for (int pre = 0; pre < ST; pre++) {
        if (pre < n_my) {
            const int tile = t_lo + gw + pre * stride;
            load_tile<KIND>(mine + pre * L::BYTES, a, page_at(trow, tile / PARTS, a.max_pages), tile % PARTS, kvh, lane);
        }
        cp_async_commit();
    }
    if (ahead) pdl_wait();

    // this thread's two rows
    bool valid[2];
    int head[2], pos[2], low[2];
    long long tok[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = row0 + gid + i * 8;
        valid[i] = r < n_rows;
        const int rr = valid[i] ? r : row0;
        head[i] = kvh * G + rr % G;
        tok[i] = packed0 + rr / G;
        pos[i] = start + rr / G;
        low[i] = oe_first_key(pos[i], a.window);
    }
    // Q fragments, turned: qf, and for a 16-bit cache what its rounding leaves
    constexpr int KL = KIND == OE_KV_BF16 ? KS : 1;
    uint32_t qf[KS][4], ql[KL][4];
    float row_scale[2] = {a.scale_log2, a.scale_log2};
    {
        float qv[KS][4][2];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint2 w = make_uint2(0u, 0u);
                if (valid[i]) w = *(const uint2*)(a.q + tok[i] * a.q_stride + (size_t)head[i] * HD + ks * 16 + tig * 4);
                qv[ks][i][0] = kv8_from_bits(w.x & 0xffffu); qv[ks][i][1] = kv8_from_bits(w.x >> 16);
                qv[ks][i + 2][0] = kv8_from_bits(w.y & 0xffffu); qv[ks][i + 2][1] = kv8_from_bits(w.y >> 16);
            }
        }
        if (a.cos_tab != nullptr) {
#pragma unroll
            for (int ks = 0; ks < KS / 2; ks++) {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int d = ks * 16 + tig * 4 + (x >> 1) * 2;
                    const float2 cs = *(const float2*)(a.cos_tab + (size_t)pos[x & 1] * (HD / 2) + d);
                    const float2 sn = *(const float2*)(a.sin_tab + (size_t)pos[x & 1] * (HD / 2) + d);
                    const float x0 = qv[ks][x][0], x1 = qv[ks][x][1], y0 = qv[ks + KS / 2][x][0], y1 = qv[ks + KS / 2][x][1];
                    qv[ks][x][0] = x0 * cs.x - y0 * sn.x;
                    qv[ks][x][1] = x1 * cs.y - y1 * sn.y;
                    qv[ks + KS / 2][x][0] = x0 * sn.x + y0 * cs.x;
                    qv[ks + KS / 2][x][1] = x1 * sn.y + y1 * cs.y;
                }
            }
        }
        if (KIND == OE_KV_BF16) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    qf[ks][x] = pack_bf16(qv[ks][x][0], qv[ks][x][1]);
                    ql[ks < KL ? ks : 0][x] = rest_bf16(qv[ks][x][0], qv[ks][x][1], qf[ks][x]);
                }
            }
        } else {
            float most[2] = {0.f, 0.f}, down[2];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int x = 0; x < 4; x++) most[x & 1] = fmaxf(most[x & 1], fmaxf(fabsf(qv[ks][x][0]), fabsf(qv[ks][x][1])));
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 1));
                most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 2));
                float up;
                down[i] = kv8_row_factor(most[i], &up);
                row_scale[i] *= up;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int x = 0; x < 4; x++) qf[ks][x] = pack_f16(qv[ks][x][0] * down[x & 1], qv[ks][x][1] * down[x & 1]);
            }
        }
    }
    // the warp that meets the new token's tile makes that token's rows and stores them in the cache
    const bool owner = own_kv && n_my > 0 && (t_hi - t_lo - gw) % stride == 0;
    NewToken<KIND> fresh;
    if (owner) {
        fresh.make(a, a.q + packed0 * a.q_stride, start, kvh, lane);
        const int page = page_at(trow, start / OE_PAGE, a.max_pages);
        if ((unsigned)page < (unsigned long long)a.n_pages) {
            const long long krow = (((long long)page * 2) * a.KVH + kvh) * OE_PAGE + start % OE_PAGE, vrow = krow + (long long)a.KVH * OE_PAGE;
            fresh.store((uint8_t*)a.cache_w + krow * (HD * L::ELEM), (uint8_t*)a.cache_w + vrow * (HD * L::ELEM), lane);
            if (KIND != OE_KV_BF16 && lane == 0) { a.scales_w[krow] = fresh.ks; a.scales_w[vrow] = fresh.vs; }
        }
    }

    float oacc[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; n++) { oacc[n][0] = oacc[n][1] = oacc[n][2] = oacc[n][3] = 0.f; }
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    float ref = kv8_above(0.f);                             // R: what O is relative to
    constexpr float HEADROOM = KIND == OE_KV_BF16 ? 0.f : 8.f;
    int stage = 0;
    for (int it = 0; it < n_my; it++) {
        const int tile = t_lo + gw + it * stride;
        uint8_t* cur = mine + (size_t)stage * L::BYTES;
        const uint8_t* vs_cur = cur + L::V_AT;
        cp_async_wait<ST - 1>();
        __syncwarp();
        if (own_kv && tile == t_hi) {
            const int r = start % TB;
            fresh.store(cur + r * L::K_ROW, cur + L::V_AT + r * L::V_ROW, lane);
            if (KIND != OE_KV_BF16 && lane == 0) { ((float*)(cur + L::S_AT))[r] = fresh.ks; ((float*)(cur + L::S_AT))[TB + r] = fresh.vs; }
            __syncwarp();
        }
        const bool mapped = (unsigned)page_at(trow, tile / PARTS, a.max_pages) < (unsigned long long)a.n_pages;
        if (mapped) {
            float s[TB / 8][4];
#pragma unroll
            for (int n = 0; n < TB / 8; n++) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const uint8_t* kr = cur + (n * 8 + gid) * L::K_ROW + tig * 4 * L::ELEM;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    if (KIND == OE_KV_BF16) {
                        const uint2 w = *(const uint2*)(kr + ks * 32);
                        mma_bf16(s[n], qf[ks], w.x, w.y);
                        mma_bf16(s[n], ql[ks < KL ? ks : 0], w.x, w.y);
                    } else {
                        const uint32_t w = kv8_word<KIND>(*(const uint32_t*)(kr + ks * 16));
                        mma_f16(s[n], qf[ks], kv8_pair<KIND>(w, 0), kv8_pair<KIND>(w, 2));
                    }
                }
            }
            const float* sc = (const float*)(cur + L::S_AT);
            const int k0 = tile * TB;
            // (key_lo: the first key of this CTA's range, beside each row's own)
            const bool whole = k0 >= key_lo && k0 + TB - 1 <= key_hi &&
                               k0 + TB - 1 <= min(pos[0], pos[1]) && k0 >= max(low[0], low[1]);
            const bool mask = !__all_sync(0xffffffffu, whole);
            float rmax[2] = {-INFINITY, -INFINITY}, sv_most = 0.f;
#pragma unroll
            for (int n = 0; n < TB / 8; n++) {
                float2 ksc = make_float2(1.f, 1.f), vsc = make_float2(0.f, 0.f);
                if (KIND != OE_KV_BF16) {
                    ksc = *(const float2*)(sc + n * 8 + tig * 2);
                    vsc = *(const float2*)(sc + TB + n * 8 + tig * 2);
                }
                const int key = k0 + n * 8 + tig * 2;
                if (KIND != OE_KV_BF16) {
                    if (!mask || (key >= key_lo && key <= key_hi)) sv_most = fmaxf(sv_most, vsc.x);
                    if (!mask || (key + 1 >= key_lo && key + 1 <= key_hi)) sv_most = fmaxf(sv_most, vsc.y);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = e >> 1, ke = key + (e & 1);
                    float v = s[n][e] * (KIND == OE_KV_BF16 ? row_scale[i] : (e & 1 ? ksc.y : ksc.x) * row_scale[i]);
                    if (mask) {
                        const bool seen = ke >= key_lo && ke <= pos[i] && ke >= low[i];
                        v = seen ? v : -INFINITY;
                    }
                    s[n][e] = v;
                    rmax[i] = fmaxf(rmax[i], v);
                }
            }
            float grown = 1.f, inv_ref = 1.f;
            if (KIND != OE_KV_BF16) {
                sv_most = fmaxf(sv_most, __shfl_xor_sync(0xffffffffu, sv_most, 1));
                sv_most = fmaxf(sv_most, __shfl_xor_sync(0xffffffffu, sv_most, 2));
                const float next = fmaxf(ref, kv8_above(sv_most));
                inv_ref = kv8_inverse(next);
                grown = ref * inv_ref;
                ref = next;
            }
            float alpha[2], m_use[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 1));
                rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], 2));
                const float m_new = fmaxf(m_run[i], rmax[i]);
                m_use[i] = m_new == -INFINITY ? 0.f : m_new;
                alpha[i] = exp2f(m_run[i] - m_use[i]);
                m_use[i] -= HEADROOM;                       // l and O carry 2^8 beside the maximum's 2^-m
                m_run[i] = m_new;
            }
            float rsum[2] = {0.f, 0.f};
#pragma unroll
            for (int n = 0; n < TB / 8; n++) {
                float2 vsc = make_float2(1.f, 1.f);
                if (KIND != OE_KV_BF16) vsc = *(const float2*)(sc + TB + n * 8 + tig * 2);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = exp2f(s[n][e] - m_use[e >> 1]);
                    rsum[e >> 1] += p;
                    float w = p;
                    if (KIND != OE_KV_BF16) w = mask && s[n][e] == -INFINITY ? 0.f : p * ((e & 1 ? vsc.y : vsc.x) * inv_ref);
                    s[n][e] = w;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                l_run[i] = l_run[i] * alpha[i] + rsum[i];
                alpha[i] *= grown;
            }
#pragma unroll
            for (int n = 0; n < HD / 8; n++) {
                oacc[n][0] *= alpha[0]; oacc[n][1] *= alpha[0];
                oacc[n][2] *= alpha[1]; oacc[n][3] *= alpha[1];
            }
#pragma unroll
            for (int kk = 0; kk < TB / 16; kk++) {
                uint32_t pa[4], pl[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float w0 = s[2 * kk + (x >> 1)][2 * (x & 1)], w1 = s[2 * kk + (x >> 1)][2 * (x & 1) + 1];
                    pa[x] = KIND == OE_KV_BF16 ? pack_bf16(w0, w1) : pack_f16(w0, w1);
                    if (KIND == OE_KV_BF16) pl[x] = rest_bf16(w0, w1, pa[x]);
                }
                const uint8_t* vr = vs_cur + (kk * 16 + tig * 2) * L::V_ROW + gid * 4 * L::ELEM;
#pragma unroll
                for (int c = 0; c < HD / 32; c++) {
                    if (KIND == OE_KV_BF16) {
                        uint2 w0 = *(const uint2*)(vr + c * 64), w1 = *(const uint2*)(vr + L::V_ROW + c * 64);
                        uint2 w2 = *(const uint2*)(vr + 8 * L::V_ROW + c * 64), w3 = *(const uint2*)(vr + 9 * L::V_ROW + c * 64);
                        if (mask) {            // a row behind the last token may hold anything, and 0 times that need not be 0
                            const int key = k0 + kk * 16 + tig * 2;
                            if (key < key_lo || key > key_hi) w0 = make_uint2(0u, 0u);
                            if (key + 1 < key_lo || key + 1 > key_hi) w1 = make_uint2(0u, 0u);
                            if (key + 8 < key_lo || key + 8 > key_hi) w2 = make_uint2(0u, 0u);
                            if (key + 9 < key_lo || key + 9 > key_hi) w3 = make_uint2(0u, 0u);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
                            const uint32_t b0 = j < 2 ? kv8_prmt(w0.x, w1.x, sel) : kv8_prmt(w0.y, w1.y, sel);
                            const uint32_t b1 = j < 2 ? kv8_prmt(w2.x, w3.x, sel) : kv8_prmt(w2.y, w3.y, sel);
                            mma_bf16(oacc[c * 4 + j], pa, b0, b1);
                            mma_bf16(oacc[c * 4 + j], pl, b0, b1);
                        }
                    } else {
                        const uint32_t w0 = kv8_word<KIND>(*(const uint32_t*)(vr + c * 32)), w1 = kv8_word<KIND>(*(const uint32_t*)(vr + L::V_ROW + c * 32));
                        const uint32_t w2 = kv8_word<KIND>(*(const uint32_t*)(vr + 8 * L::V_ROW + c * 32)), w3 = kv8_word<KIND>(*(const uint32_t*)(vr + 9 * L::V_ROW + c * 32));
                        const uint32_t x0 = kv8_prmt(w0, w1, 0x5140u), x1 = kv8_prmt(w0, w1, 0x7362u);
                        const uint32_t y0 = kv8_prmt(w2, w3, 0x5140u), y1 = kv8_prmt(w2, w3, 0x7362u);
                        mma_f16(oacc[c * 4 + 0], pa, kv8_pair<KIND>(x0, 0), kv8_pair<KIND>(y0, 0));
                        mma_f16(oacc[c * 4 + 1], pa, kv8_pair<KIND>(x0, 2), kv8_pair<KIND>(y0, 2));
                        mma_f16(oacc[c * 4 + 2], pa, kv8_pair<KIND>(x1, 0), kv8_pair<KIND>(y1, 0));
                        mma_f16(oacc[c * 4 + 3], pa, kv8_pair<KIND>(x1, 2), kv8_pair<KIND>(y1, 2));
                    }
                }
            }
        }
        __syncwarp();                                       // every lane has read the stage: refill it
        if (it + ST < n_my) {
            const int next = tile + ST * stride;
            load_tile<KIND>(cur, a, page_at(trow, next / PARTS, a.max_pages), next % PARTS, kvh, lane);
        }
        cp_async_commit();
        stage = stage + 1 == ST ? 0 : stage + 1;
    }
    cp_async_wait<0>();
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 1);
        l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], 2);
    }
    // the warps' parts, added in warp order
    __syncthreads();                                        // every warp has left its ring
    const int rows = min(16, n_rows - row0);
    const float out_scale = KIND == OE_KV_BF16 ? 1.f : ref;
    float* part = (float*)smem;                             // [NW][16][HD + 2]
    float* cpart = part + (size_t)NW * 16 * (HD + 2);       // [16][HD + 2]: this CTA's sum
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float* p = part + ((size_t)warp * 16 + gid + i * 8) * (HD + 2);
#pragma unroll
        for (int c = 0; c < HD / 32; c++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                p[c * 32 + tig * 8 + j] = oacc[c * 4 + j][2 * i] * out_scale;
                p[c * 32 + tig * 8 + 4 + j] = oacc[c * 4 + j][2 * i + 1] * out_scale;
            }
        }
        if (tig == 0) { p[HD] = m_run[i]; p[HD + 1] = l_run[i]; }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows * HD; idx += NW * 32) {
        const int r = idx / HD, d = idx % HD;
        float m = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) m = fmaxf(m, part[((size_t)w * 16 + r) * (HD + 2) + HD]);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float* p = part + ((size_t)w * 16 + r) * (HD + 2);
            if (p[HD] == -INFINITY && p[HD + 1] == 0.f) continue;          // no key of this row
            const float e = exp2f(p[HD] - (m == -INFINITY ? 0.f : m));
            l += p[HD + 1] * e;
            o += p[d] * e;
        }
        cpart[r * (HD + 2) + d] = o;
        if (d == 0) { cpart[r * (HD + 2) + HD] = m; cpart[r * (HD + 2) + HD + 1] = l; }
    }
    if (CR > 1) cluster_sync_all();
    else __syncthreads();
    const int n_pre = common > 0 ? a.splits : 0;
    for (int idx = threadIdx.x + rank * NW * 32; idx < rows * HD; idx += NW * 32 * CR) {
        const int r = idx / HD, d = idx % HD;
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (int q = 0; q < CR; q++) m = fmaxf(m, CR > 1 ? ld_peer_f32(cpart + r * (HD + 2) + HD, q) : cpart[r * (HD + 2) + HD]);
        const int h = kvh * G + (row0 + r) % G;
        const float* pre_o = a.part_o + ((long long)b * a.H + h) * a.splits * HD;
        const float2* pre_ml = (const float2*)a.part_ml + ((long long)b * a.H + h) * a.splits;
        for (int q = 0; q < n_pre; q++) m = fmaxf(m, pre_ml[q].x);
        const float mu = m == -INFINITY ? 0.f : m;
        for (int q = 0; q < CR; q++) {
            const float pm = CR > 1 ? ld_peer_f32(cpart + r * (HD + 2) + HD, q) : cpart[r * (HD + 2) + HD];
            const float pl = CR > 1 ? ld_peer_f32(cpart + r * (HD + 2) + HD + 1, q) : cpart[r * (HD + 2) + HD + 1];
            if (pm == -INFINITY && pl == 0.f) continue;
            const float e = exp2f(pm - mu);
            l += pl * e;
            o += (CR > 1 ? ld_peer_f32(cpart + r * (HD + 2) + d, q) : cpart[r * (HD + 2) + d]) * e;
        }
        for (int q = 0; q < n_pre; q++) {
            const float2 ml = pre_ml[q];
            if (ml.x == -INFINITY && ml.y == 0.f) continue;
            const float e = exp2f(ml.x - mu);
            l += ml.y * e;
            o += pre_o[q * HD + d] * e;
        }
        a.out[(packed0 + (row0 + r) / G) * (long long)(a.H * HD) + (long long)h * HD + d] = __float2bfloat16_rn(l > 0.f ? o / l : l == 0.f ? 0.f : l);
    }
    if (CR > 1) cluster_sync_all();                         // nobody leaves while its shared memory is read
}

template <int KIND>
int launch(const Args& a, int row_tiles, int n_seqs, cudaStream_t st) {
    constexpr int NW = KIND == OE_KV_BF16 ? 3 : 4, ST = KIND == OE_KV_BF16 ? 2 : 3;
    constexpr size_t smem = (size_t)NW * ST * Tile<KIND>::BYTES;
    const long long x = (long long)row_tiles * a.cluster;
    if (x > 0x7fffffffLL || a.KVH > 65535 || n_seqs > 65535) return OE_ERR_UNSUPPORTED;
    cudaError_t e = cudaFuncSetAttribute(attn_kv8_kernel<KIND, NW, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    const dim3 grid((unsigned)x, a.KVH, n_seqs);
    if (a.cluster > 1) return oe_launch_cluster(attn_kv8_kernel<KIND, NW, ST>, (unsigned)a.cluster, grid, dim3(NW * 32), smem, st, a);
    return oe_launch(attn_kv8_kernel<KIND, NW, ST>, grid, dim3(NW * 32), smem, st, a);
}

}  // namespace

extern "C" {

// Keys and values of n_tokens tokens (rows of `stride` bfloat16: H query heads, KVH keys, KVH values) into the 8-bit cache.
int oe_kv8_write(int kind, const bf16* qkv, long long stride, const float* cos_tab, const float* sin_tab, void* codes, float* scales,
                 long long n_pages, const int* tables, int max_pages, const int* tok_seq, const int* tok_pos, int n_tokens, int H,
                 int KVH, cudaStream_t st) {
    if (n_tokens <= 0) return 0;
    if (stride % 8 || ((uintptr_t)qkv & 15) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15)) return OE_ERR_UNSUPPORTED;
    const long long blocks = ((long long)n_tokens * 2 * KVH * (HD / 16) + 255) / 256;
    if (blocks > 0x7fffffffLL) return OE_ERR_UNSUPPORTED;
    if (kind == OE_KV_INT8)
        return oe_launch(kv8_write_kernel<OE_KV_INT8>, dim3((unsigned)blocks), dim3(256), 0, st, qkv, stride, cos_tab, sin_tab,
                         (uint8_t*)codes, scales, n_pages, tables, max_pages, tok_seq, tok_pos, n_tokens, H, KVH);
    if (kind == OE_KV_E4M3)
        return oe_launch(kv8_write_kernel<OE_KV_E4M3>, dim3((unsigned)blocks), dim3(256), 0, st, qkv, stride, cos_tab, sin_tab,
                         (uint8_t*)codes, scales, n_pages, tables, max_pages, tok_seq, tok_pos, n_tokens, H, KVH);
    return OE_ERR_UNSUPPORTED;
}

// Attention of the step's tokens over their sequences' caches (kind: OE_KV_*).  write != 0: every sequence brings one token, whose
// key and value this kernel writes.  With seq_pages the pages before a sequence's own are left out and the parts that
// oe_attn_rows_prefix left are added.
int oe_attn_kv8(int kind, bf16* out, const bf16* q, long long q_stride, const float* cos_tab, const float* sin_tab, void* cache,
                float* scales, int write, long long n_pages, const int* tables, int max_pages, const int* cu_q, const int* seq_start,
                const int* seq_qlen, int n_seqs, int max_qlen, int H, int KVH, int window, float scale, int cluster,
                const int* seq_pages, int splits, const float* part_o, const float* part_ml, int ahead, cudaStream_t st) {
    if (n_seqs <= 0 || max_qlen <= 0) return 0;
    if (H % KVH || q_stride % 8 || ((uintptr_t)q & 15) || ((uintptr_t)cache & 15) || ((uintptr_t)scales & 15)) return OE_ERR_UNSUPPORTED;
    if (cluster < 1 || cluster > 8 || (write && max_qlen != 1)) return OE_ERR_UNSUPPORTED;
    if (seq_pages != nullptr && (window != 0 || max_qlen != 1 || splits < 1 || part_o == nullptr || part_ml == nullptr)) return OE_ERR_UNSUPPORTED;
    Args a = {};
    a.out = out; a.q = q; a.q_stride = q_stride; a.cos_tab = cos_tab; a.sin_tab = sin_tab;
    a.cache = cache; a.scales = scales;
    if (write) { a.cache_w = cache; a.scales_w = scales; }
    a.n_pages = n_pages; a.tables = tables; a.max_pages = max_pages; a.cu_q = cu_q; a.seq_start = seq_start; a.seq_qlen = seq_qlen;
    a.H = H; a.KVH = KVH; a.window = window; a.scale_log2 = scale * LOG2E; a.cluster = cluster;
    a.seq_pages = seq_pages; a.splits = splits; a.part_o = part_o; a.part_ml = part_ml; a.ahead = ahead;
    const long long rows = (long long)max_qlen * (H / KVH), tiles = (rows + 15) / 16;
    if (tiles > 0x7fffffffLL) return OE_ERR_UNSUPPORTED;
    if (kind == OE_KV_BF16) return launch<OE_KV_BF16>(a, (int)tiles, n_seqs, st);
    if (kind == OE_KV_INT8) return launch<OE_KV_INT8>(a, (int)tiles, n_seqs, st);
    if (kind == OE_KV_E4M3) return launch<OE_KV_E4M3>(a, (int)tiles, n_seqs, st);
    return OE_ERR_UNSUPPORTED;
}

}  // extern "C"
