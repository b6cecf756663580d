// Decode attention over the 8-bit paged cache (kv_quant.cuh): one query token per request in bfloat16, the query heads of a kv
// head as the 16 rows of a tensor-core tile, the keys of a request split over blocks and merged by a second kernel.
//
//   s_k = scale q.K_k with K_k = c_k 2^e_k,  o = sum_k p_k V_k / sum_k p_k,  p_k = 2^(s_k log2 e - m),  V_k = d_k 2^f_k
//
// Codes become halves (exactly) in registers and go straight into m16n8k16 products with f32 sums; nothing is scaled before a
// product. The exponent of K multiplies the score; the exponent of V joins the softmax's: with t_k = s_k log2 e + f_k and the running
// maximum taken over t_k, the weight w_k = 2^(t_k - m) is what V's codes are multiplied by, at most 2^8 and therefore a half with 11 bits
// where they count, and the denominator adds w_k 2^-f_k in 32 bits. One exponential a score, as without a quantised cache. q goes to halves times a
// power of two of its row's (its largest magnitude then lies in 2^14 .. 2^15): what a half cannot hold of it is below 2^-39 of that.
//
//   grid (splits, kv heads * row tiles, entries), 4 warps a block. A warp walks pages p0 + w, p0 + w + 4, ... of its split; a page's record of
//   a kv head is one untiled bulk copy into the warp's own ring.
//   Q.K^T: a product step's 16 columns are four codes of each lane of a group of four, so a lane's 16-byte piece of a key row feeds four steps.
//   P.V: lane (g, q) of a warp takes columns g head_dim/8 .. of keys 2q, 2q + 1, 8 + 2q, 9 + 2q: the keys that its scores belong to; pairs of
//   keys are joined byte by byte, and tile t of the product holds column t of every lane's columns.
//
// Token t (= entry t) sits at position kvlen - 1 and sees positions max(0, kvlen - window) .. kvlen - 1 (window < 0: runs of -window; 0: all). No
// key to see: zeros. A block-table entry below 0 is never followed, its keys count as masked. A masked key's codes are replaced, so
// whatever a page holds behind a request's end does not matter.
#include "kv_quant.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=64, 128 or 256"
#endif
static_assert(HEAD_DIM == 64 || HEAD_DIM == 128 || HEAD_DIM == 256, "the 8-bit decode kernel takes head_dim 64, 128 or 256");

constexpr int DQ_HD = HEAD_DIM;
constexpr int DQ_WARPS = 4;
constexpr int DQ_REC = kvq_record(HEAD_DIM);
constexpr int DQ_STAGES = HEAD_DIM > 128 ? 3 : 4;
constexpr int DQ_KG = HEAD_DIM / 64;              // groups of four product steps of Q.K^T
constexpr int DQ_NT = HEAD_DIM / 8;               // tiles of eight columns of P.V
constexpr int DQ_VB = HEAD_DIM / 8 < 16 ? HEAD_DIM / 8 : 16;      // columns a lane takes of a key row at a time
constexpr int DQ_NVB = HEAD_DIM / 8 / DQ_VB;      // ... and how often
constexpr int DQ_MAX_SPLITS = 128;
constexpr int DQ_OS = HEAD_DIM + 4;
constexpr int DQ_PIPE = DQ_WARPS * DQ_STAGES * DQ_REC;
constexpr int DQ_MERGE = DQ_WARPS * 16 * (DQ_OS + 2) * 4;
constexpr int DQ_BARS = ((DQ_PIPE > DQ_MERGE ? DQ_PIPE : DQ_MERGE) + 15) / 16 * 16;
constexpr int DQ_SMEM = DQ_BARS + DQ_WARPS * DQ_STAGES * 8;
constexpr unsigned DQ_SPIN = 1u << 24;
constexpr float DQ_RAISE = 8.f;                   // the running maximum follows only when a page's is more than this above it (log2 units)

__device__ __forceinline__ void dq_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool dq_wait(uint32_t bar, uint32_t parity) {
    for (unsigned spin = 0; spin < DQ_SPIN; ++spin) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ float dq_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t dq_pack_half(float lo, float hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(hi), "f"(lo));
    return h;
}
__device__ __forceinline__ uint32_t dq_pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// (q, the newest token's slot of the cache, and o_part / ml_part in the merge, are written by the kernel before and read after a wait that is not the
// kernel's first statement: they are not declared __restrict__.)
template <int KIND>
__global__ void __launch_bounds__(DQ_WARPS * 32) attn_decode_quant_kernel(
    const __nv_bfloat16* q, long long q_stride, const unsigned char* cache, const int* __restrict__ block_table, int bt_stride,
    const int* __restrict__ entry_kvlen, int nh, int nkv, float scale_log2, int window, int n_splits, float* o_part, float* ml_part,
    __nv_bfloat16* out_direct, int* status, int early) {
    if (!early) il_pdl_wait();
    extern __shared__ __align__(128) unsigned char smem[];
    const int split = blockIdx.x, G = nh / nkv, row_tiles = (G + 15) / 16;
    const int head = blockIdx.y / row_tiles, rt = blockIdx.y - head * row_tiles, e = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane >> 2, lq = lane & 3;
    const int head0 = head * G + rt * 16, rows_valid = min(16, G - rt * 16);

    // early: the caller vouches that lengths, block tables and the pages of earlier tokens do not come from the kernel in front (which writes q and
    // the newest token's slot, in the last page). What depends only on them is then done before waiting for it.
    const int kvlen = entry_kvlen[e];
    const int lo = il_mask_lo(kvlen - 1, window);
    const int first_page = lo / KVQ_PAGE, last_page = kvlen > 0 ? (kvlen - 1) / KVQ_PAGE : first_page - 1;
    const int per_split = (last_page - first_page + n_splits) / n_splits;       // the request's pages, evenly over the splits
    const int p0 = first_page + split * per_split, p1 = min(p0 + per_split, last_page + 1);
    if (p0 >= p1 && (split > 0 || !out_direct)) return;       // no keys here: the merge knows; where there is none the block below writes zeros

    const int* bt = block_table + (size_t)e * bt_stride;
    const unsigned char* recs = cache + (size_t)head * DQ_REC;
    const size_t page_bytes = (size_t)nkv * DQ_REC;
    const int n_my = max(0, (p1 - p0 - warp + DQ_WARPS - 1) / DQ_WARPS);
    // Page ids of this warp's iterations, 32 at a time: lane l holds the id of iteration base + l.
    int ids_base = 0, my_ids = lane < n_my ? bt[p0 + warp + lane * DQ_WARPS] : 0;
    unsigned bad = 0;                             // bit (iteration % 32): the page is not there, its keys are masked
    const uint32_t pipe = (uint32_t)__cvta_generic_to_shared(smem) + warp * DQ_STAGES * DQ_REC;
    const uint32_t bars = (uint32_t)__cvta_generic_to_shared(smem) + DQ_BARS + warp * DQ_STAGES * 8;
    const auto issue = [&](int it) {
        if (it >= n_my) return;
        if (it >= ids_base + 32) {
            ids_base += 32;
            my_ids = ids_base + lane < n_my ? bt[p0 + warp + (ids_base + lane) * DQ_WARPS] : 0;
        }
        const int page = __shfl_sync(0xffffffffu, my_ids, it - ids_base);
        bad = page < 0 ? bad | 1u << (it & 31) : bad & ~(1u << (it & 31));
        if (lane == 0) {
            const uint32_t dst = pipe + (it % DQ_STAGES) * DQ_REC, bar = bars + (it % DQ_STAGES) * 8;
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");      // the record before was read by ordinary loads
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(DQ_REC) : "memory");
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                         ::"r"(dst), "l"(recs + (size_t)max(page, 0) * page_bytes), "r"(DQ_REC), "r"(bar) : "memory");
        }
    };
    if (lane == 0) {
        for (int s = 0; s < DQ_STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(bars + s * 8));
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    int issued = 0;
    if (early) {
        for (; issued < DQ_STAGES && p0 + warp + issued * DQ_WARPS < last_page; ++issued) issue(issued);
        il_pdl_wait();
    }
    for (; issued < DQ_STAGES; ++issued) issue(issued);

    // Q as the products' left operand: rows lg and lg + 8, of each group of 64 columns the 16 from 16 lq on.
    uint32_t qf[4 * DQ_KG][4];
    float s_scale[2];                             // what a row's score is multiplied by (its power of two taken back)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = lg + 8 * h;
        const __nv_bfloat16* row = q + (size_t)e * q_stride + (size_t)(head0 + r) * DQ_HD;
        uint32_t x[8 * DQ_KG], most = 0u;
#pragma unroll
        for (int kg = 0; kg < DQ_KG; ++kg)
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                x[8 * kg + c] = r < rows_valid ? *reinterpret_cast<const uint32_t*>(row + 64 * kg + 16 * lq + 2 * c) : 0u;
                most = max(most, max(x[8 * kg + c] & 0x7fffu, x[8 * kg + c] >> 16 & 0x7fffu));
            }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int ex = max((int)(most >> 7) - 127, -100);
        const float up = __int_as_float((127 + 14 - ex) << 23);
        s_scale[h] = scale_log2 * __int_as_float((127 - 14 + ex) << 23);
#pragma unroll
        for (int i = 0; i < 4 * DQ_KG; ++i) {
            const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&x[2 * i]), b = *reinterpret_cast<const __nv_bfloat162*>(&x[2 * i + 1]);
            qf[i][h] = dq_pack_half(__low2float(a) * up, __high2float(a) * up);
            qf[i][2 + h] = dq_pack_half(__low2float(b) * up, __high2float(b) * up);
        }
    }

    float o[DQ_NT][4];
#pragma unroll
    for (int i = 0; i < DQ_NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int it = 0; it < n_my; ++it) {
        if (!dq_wait(bars + (it % DQ_STAGES) * 8, (it / DQ_STAGES) & 1)) {
            if (lane == 0) atomicExch(status, 91);
            for (int k = it + 1; k < min(it + DQ_STAGES, n_my); ++k) dq_wait(bars + (k % DQ_STAGES) * 8, (k / DQ_STAGES) & 1);
            break;
        }
        const unsigned char* rec = smem + (size_t)(warp * DQ_STAGES + it % DQ_STAGES) * DQ_REC;
        // ---- scores of the page's 16 keys: s[n] holds keys 8 n + 2 lq, + 1 of rows lg (0, 1) and lg + 8 (2, 3)
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
#pragma unroll
        for (int kg = 0; kg < DQ_KG; ++kg)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int key = 8 * n + lg, piece = (key * (DQ_HD / 16) + 4 * kg + lq) ^ kvq_turn(DQ_HD, false, key);
                const uint4 w = *reinterpret_cast<const uint4*>(rec + piece * 16);
                const uint32_t c[4] = {kvq_raw<KIND>(w.x), kvq_raw<KIND>(w.y), kvq_raw<KIND>(w.z), kvq_raw<KIND>(w.w)};
#pragma unroll
                for (int i = 0; i < 4; ++i) dq_mma(s[n], qf[4 * kg + i], kvq_low<KIND>(c[i]), kvq_high<KIND>(c[i]));
            }
        // ---- exponents of this lane's four keys, softmax in base 2
        uint32_t ke[2], ve[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            ke[n] = *reinterpret_cast<const uint16_t*>(rec + 2 * KVQ_PAGE * DQ_HD + 8 * n + 2 * lq);
            ve[n] = *reinterpret_cast<const uint16_t*>(rec + 2 * KVQ_PAGE * DQ_HD + KVQ_PAGE + 8 * n + 2 * lq);
        }
        const int key0 = (p0 + warp + it * DQ_WARPS) * KVQ_PAGE + 2 * lq;
        const bool gone = (bad >> (it & 31)) & 1;
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};        // a byte a key: 2 lq, 2 lq + 1 of either half of the page
        float inv_v[2][2];
        const bool edge = gone || key0 - 2 * lq < lo || key0 - 2 * lq + KVQ_PAGE > kvlen;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int kb = ke[n] >> (8 * j) & 255, vb = ve[n] >> (8 * j) & 255, key = key0 + 8 * n + j;
                const float kp = kvq_power(kb), add = vb == KVQ_NAN ? __int_as_float(0x7fc00000) : (float)(vb - 127);
                const bool there = !edge || (!gone && key >= lo && key < kvlen);
                inv_v[n][j] = __int_as_float((254 - vb) << 23);
#pragma unroll
                for (int h = 0; h < 2; ++h) s[n][2 * h + j] = there ? fmaf(s[n][2 * h + j], s_scale[h] * kp, add) : -INFINITY;
                if (!there) seen[n] &= j ? 0x00ff00ffu : 0xff00ff00u, inv_v[n][j] = 0.f;
            }
        uint32_t pf[4];
        float corr[2];
        bool raise = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const bool up = mx > m[h] + DQ_RAISE;             // also the first keys of a row (m = -inf)
            const float mn = up ? mx : m[h];
            corr[h] = up ? dq_ex2(m[h] - mn) : 1.f;           // 0 when nothing was summed yet
            raise |= up;
            const float ms = mn == -INFINITY ? 0.f : mn;
            float w[2][2], rs = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    w[n][j] = dq_ex2(s[n][2 * h + j] - ms);
                    rs = fmaf(w[n][j], inv_v[n][j], rs);
                }
            l[h] = l[h] * corr[h] + rs;                       // (this lane's keys; the lanes of a row are added at the end)
            m[h] = mn;
            pf[h] = dq_pack_half(w[0][0], w[0][1]);
            pf[2 + h] = dq_pack_half(w[1][0], w[1][1]);
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int t = 0; t < DQ_NT; ++t) o[t][0] *= corr[0], o[t][1] *= corr[0], o[t][2] *= corr[1], o[t][3] *= corr[1];
        }
        // ---- P.V: this lane's four keys, DQ_VB columns at a time
#pragma unroll
        for (int vb = 0; vb < DQ_NVB; ++vb) {
            uint32_t x[4][DQ_VB / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int key = 2 * lq + (k & 1) + 8 * (k >> 1), col = vb * 8 * DQ_VB + lg * DQ_VB;
                const int piece = (key * (DQ_HD / 16) + col / 16) ^ kvq_turn(DQ_HD, true, key);
                const unsigned char* at = rec + KVQ_PAGE * DQ_HD + piece * 16 + col % 16;
                if constexpr (DQ_VB == 16) {
                    const uint4 w = *reinterpret_cast<const uint4*>(at);
                    x[k][0] = w.x, x[k][1] = w.y, x[k][2] = w.z, x[k][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(at);
                    x[k][0] = w.x, x[k][1] = w.y;
                }
            }
#pragma unroll
            for (int i = 0; i < DQ_VB / 4; ++i) {
                uint32_t a[2][2];                             // [keys 2 lq, + 1 | 8 + 2 lq, + 1][columns 0, 1 | 2, 3]: two keys of a column side by side
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    a[n][0] = __byte_perm(x[2 * n][i], x[2 * n + 1][i], 0x5140);
                    a[n][1] = __byte_perm(x[2 * n][i], x[2 * n + 1][i], 0x7362);
                    if (edge) a[n][0] &= seen[n], a[n][1] &= seen[n];
                    a[n][0] = kvq_raw<KIND>(a[n][0]), a[n][1] = kvq_raw<KIND>(a[n][1]);
                }
                const int t = vb * DQ_VB + 4 * i;
                dq_mma(o[t], pf, kvq_low<KIND>(a[0][0]), kvq_low<KIND>(a[1][0]));
                dq_mma(o[t + 1], pf, kvq_high<KIND>(a[0][0]), kvq_high<KIND>(a[1][0]));
                dq_mma(o[t + 2], pf, kvq_low<KIND>(a[0][1]), kvq_low<KIND>(a[1][1]));
                dq_mma(o[t + 3], pf, kvq_high<KIND>(a[0][1]), kvq_high<KIND>(a[1][1]));
            }
        }
        __syncwarp();
        issue(it + DQ_STAGES);                    // refill the stage this record came from
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    __syncthreads();                              // the pipeline memory is reused for the merge

    // The four warps' sums, brought to the rows' common maximum, then added in warp order.
    float* sm_ml = reinterpret_cast<float*>(smem);                     // [warp][16 rows][m, l]
    float* sm_o = sm_ml + DQ_WARPS * 16 * 2;                           // [warp][16 rows][DQ_OS]
    if (lq == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sm_ml[(warp * 16 + lg + 8 * h) * 2] = m[h];
            sm_ml[(warp * 16 + lg + 8 * h) * 2 + 1] = l[h];
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = lg + 8 * h;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < DQ_WARPS; ++w) M = fmaxf(M, sm_ml[(w * 16 + r) * 2]);
        const float f = m[h] == -INFINITY ? 0.f : dq_ex2(m[h] - M);
        float* row = sm_o + (size_t)(warp * 16 + r) * DQ_OS;
#pragma unroll
        for (int vb = 0; vb < DQ_NVB; ++vb)
#pragma unroll
            for (int j = 0; j < 2; ++j)           // tile columns 2 lq + j: columns DQ_VB (2 lq + j) .. of this block of columns
#pragma unroll
                for (int t = 0; t < DQ_VB; t += 4)
                    *reinterpret_cast<float4*>(row + vb * 8 * DQ_VB + (2 * lq + j) * DQ_VB + t) =
                        make_float4(f * o[vb * DQ_VB + t][2 * h + j], f * o[vb * DQ_VB + t + 1][2 * h + j], f * o[vb * DQ_VB + t + 2][2 * h + j],
                                    f * o[vb * DQ_VB + t + 3][2 * h + j]);
    }
    il_pdl_tail();
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows_valid * (DQ_HD / 4); idx += DQ_WARPS * 32) {
        const int r = idx / (DQ_HD / 4), d = (idx - r * (DQ_HD / 4)) * 4;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < DQ_WARPS; ++w) M = fmaxf(M, sm_ml[(w * 16 + r) * 2]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < DQ_WARPS; ++w) {
            const float mw = sm_ml[(w * 16 + r) * 2];
            L += (mw == -INFINITY ? 0.f : dq_ex2(mw - M)) * sm_ml[(w * 16 + r) * 2 + 1];
            const float4 v = *reinterpret_cast<const float4*>(sm_o + (size_t)(w * 16 + r) * DQ_OS + d);
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
        const size_t row = (size_t)e * nh + head0 + r;
        if (out_direct) {
            const float inv = L == 0.f ? 0.f : 1.f / L;       // (no key seen: zeros)
            *reinterpret_cast<uint2*>(out_direct + row * DQ_HD + d) = make_uint2(dq_pack_bf16(acc.x * inv, acc.y * inv), dq_pack_bf16(acc.z * inv, acc.w * inv));
        } else {
            *reinterpret_cast<float4*>(o_part + (row * n_splits + split) * DQ_HD + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(ml_part + (row * n_splits + split) * 2) = make_float2(M, L);
        }
    }
}

// The merge: a warp a (token, head) row, a lane four columns at a time; the splits are added in order.
__global__ void __launch_bounds__(128) attn_decode_quant_merge_kernel(const float* o_part, const float* ml_part, const int* __restrict__ entry_kvlen, int nh,
                                                                      int n_rows, int window, int n_splits, __nv_bfloat16* out) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int kvlen = row < n_rows ? entry_kvlen[row / nh] : 0;
    il_pdl_wait();
    if (row >= n_rows) return;
    int n_valid = 0;                              // splits that have keys
    if (kvlen > 0) {
        const int n_pages = (kvlen - 1) / KVQ_PAGE - il_mask_lo(kvlen - 1, window) / KVQ_PAGE + 1, per_split = (n_pages + n_splits - 1) / n_splits;
        n_valid = (n_pages + per_split - 1) / per_split;
    }
    const float* ml = ml_part + (size_t)row * n_splits * 2;
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < n_valid; s += 32) M = fmaxf(M, ml[2 * s]);
    M = il_warp_max(M);
    for (int s = lane; s < n_valid; s += 32) L += (ml[2 * s] == -INFINITY ? 0.f : dq_ex2(ml[2 * s] - M)) * ml[2 * s + 1];
    L = il_warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int d = lane * 4; d < DQ_HD; d += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < n_valid; ++s) {
            const float f = ml[2 * s] == -INFINITY ? 0.f : dq_ex2(ml[2 * s] - M);
            const float4 v = *reinterpret_cast<const float4*>(o_part + ((size_t)row * n_splits + s) * DQ_HD + d);
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
        }
        *reinterpret_cast<uint2*>(out + (size_t)row * DQ_HD + d) = make_uint2(dq_pack_bf16(acc.x * inv, acc.y * inv), dq_pack_bf16(acc.z * inv, acc.w * inv));
    }
}

static int dq_prepare(int dev) {
    static bool done[64];
    if (dev < 0 || dev >= 64 || done[dev]) return IL_OK;
    cudaError_t e = cudaFuncSetAttribute(attn_decode_quant_kernel<KVQ_E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, DQ_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_decode_quant_kernel<KVQ_INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, DQ_SMEM);
    if (e != cudaSuccess) return 1000 + (int)e;
    done[dev] = true;
    return IL_OK;
}

// Blocks that this device runs at once; 0 if the query fails. The caller sizes the number of splits by it.
IL_EXPORT int il_attn_decode_quant_resident_blocks() {
    int dev = 0, per_sm = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dq_prepare(dev) != IL_OK ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attn_decode_quant_kernel<KVQ_E4M3>, DQ_WARPS * 32, DQ_SMEM) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return per_sm * sms;
}

// Scratch for more than one split: o_part float32 [n_decode * nh * n_splits * head_dim], ml_part [n_decode * nh * n_splits * 2].
IL_EXPORT int il_attn_decode_quant(const void* q, long long q_stride, void* out, const void* cache, int kind, const int* block_table, int bt_stride,
                                   const int* entry_kvlen, int n_decode, int nh, int nkv, int hd, float scale, int window, int n_splits, float* o_part,
                                   float* ml_part, int* status, int early, cudaStream_t stream) {
    if (n_decode <= 0) return IL_OK;
    if (hd != HEAD_DIM || n_splits > DQ_MAX_SPLITS || n_decode > 65535) return IL_UNSUPPORTED;
    if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || n_splits <= 0 || (kind != KVQ_E4M3 && kind != KVQ_INT8) || !status) return IL_BAD_ARG;
    if ((((uintptr_t)cache | (uintptr_t)q | (uintptr_t)out) & 15) || (q_stride & 7) || q_stride < (long long)nh * hd) return IL_BAD_ARG;
    const int row_tiles = (nh / nkv + 15) / 16;
    if ((long long)nkv * row_tiles > 65535) return IL_UNSUPPORTED;
    int dev = 0;
    cudaGetDevice(&dev);
    const int rc = dq_prepare(dev);
    if (rc != IL_OK) return rc;
    const dim3 grid(n_splits, nkv * row_tiles, n_decode);
    __nv_bfloat16* direct = n_splits == 1 ? (__nv_bfloat16*)out : nullptr;
#define DQ_GO(KIND)                                                                                                                               \
    IL_LAUNCH((attn_decode_quant_kernel<KIND>), grid, DQ_WARPS * 32, DQ_SMEM, stream, (const __nv_bfloat16*)q, q_stride, (const unsigned char*)cache, \
              block_table, bt_stride, entry_kvlen, nh, nkv, scale * 1.4426950408889634f, window, n_splits, o_part, ml_part, direct, status, early)
    if (kind == KVQ_E4M3) DQ_GO(KVQ_E4M3);
    else DQ_GO(KVQ_INT8);
#undef DQ_GO
    if (n_splits > 1) {
        const int n_rows = n_decode * nh;
        IL_LAUNCH(attn_decode_quant_merge_kernel, (n_rows + 3) / 4, 128, 0, stream, (const float*)o_part, (const float*)ml_part, entry_kvlen, nh, n_rows,
                  window, n_splits, (__nv_bfloat16*)out);
    }
    IL_LAUNCH_CHECK();
    return IL_OK;
}
