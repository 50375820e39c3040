// Attention of drafted tokens over a paged cache (dsv41_tree_attention): the mathematics, and the kernel for head
// sizes over 128 (tree_attn_tc.cu has the others).
//
// For request b with s_b keys in the cache, the last n_b of them its new tokens, token i and query head
// hq = h * G + g:
//     out[i, hq] = sum_j p_ij v[j, h] / sum_j p_ij,   p_ij = exp(scale * q[i, hq] . k[j, h] - m_i)
// over the keys j that i sees: all of the context, and among the new tokens its ancestors and itself (a bit
// mask per token), or the tokens before it and itself (no mask). A row that sees nothing is zero.
//
// All G query heads of a KV head and all new tokens of a request share its keys, so they are the rows
// (r = i * G + g) of one product: each key and value is read once per tile of rows, and the softmax runs over
// the keys in one pass (running maximum m and sum l in fp32, the accumulator rescaled when m grows).
//
// Split: the (request, KV head, row tile, key tile) units of the call are cut into equal runs, one per
// resident CTA, whatever the lengths are; the cut is computed in the kernel from the lengths (the host does
// not know them). A segment (the units of one row tile) that crosses CTAs leaves (m, l, O) per part in the
// workspace and the CTA that arrives last joins the parts in order: one launch, results independent of timing.
//
// Here: warp-level matrix instructions with Q and O in registers, keys and values through a three-stage ring of
// cp.async copies. For few rows the warps share a tile's keys (WN = 4 / WM of them per row tile) and are joined at the
// end of a segment.
#include "internal.h"
#include "tree_attn.cuh"

namespace dsv41 {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;

template <int DT, int WM>
struct AttnCfg {
    static constexpr int kt = WM > 1 ? 32 : 64;                      // keys per tile
    static constexpr int rt = 16 * WM;                               // rows per tile
    static constexpr int wn = kAttnWarps / WM;                       // warps that share a row tile's keys
    static constexpr int tn = kt / wn;                               // keys of a tile per warp
    static constexpr int row_b = DT * 2;
    static constexpr int tile_b = kt * row_b;                        // one K or V tile
    static constexpr int stages = 3;
    static constexpr int buf_b = wn > 1 ? rt * DT * 4 : kAttnWarps * 16 * tn * 4;   // joins of warps / P of a dirty tile
    static constexpr int ml_off = stages * 2 * tile_b + buf_b;
    static constexpr int smem = ml_off + wn * rt * 8;
    static constexpr int per_sm = smem <= 113 * 1024 ? 2 : 1;
    static_assert(tn >= 16 && tn % 16 == 0, "a warp's keys are whole k16 steps");
    static_assert(kMaxRequests * 8 <= stages * 2 * tile_b, "the prefix sums live in the stages");
};

template <typename T, int DT, int WM>
__global__ void __launch_bounds__(kAttnThreads, AttnCfg<DT, WM>::per_sm) tree_attn_kernel(const TreeAttnParams p)
{
    using Cfg = AttnCfg<DT, WM>;
    constexpr int KT = Cfg::kt, RT = Cfg::rt, WN = Cfg::wn, TN = Cfg::tn, NT = DT / 8, CPR = DT / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t warp_tot[kAttnWarps];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wm = warp % WM, wk = warp / WM;
    float* buf = reinterpret_cast<float*>(smem + Cfg::stages * 2 * Cfg::tile_b);
    float2* ml = reinterpret_cast<float2*>(smem + Cfg::ml_off);
    const uint32_t sbase = smem_addr(smem);

    // ---- this CTA's run of units -------------------------------------------------------------
    int64_t* pre = reinterpret_cast<int64_t*>(smem);   // exclusive prefix sums of units
    int64_t total;
    {
        const int per = (p.batch + kAttnThreads - 1) / kAttnThreads;
        const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
        auto units = [&](int b) -> int64_t {
            const AttnReq r = attn_req(p, b);
            return r.n > 0 ? (int64_t)((r.n * p.group + RT - 1) / RT) * max((r.seq + KT - 1) / KT, 1) * p.kv_heads : 0;
        };
        int64_t sum = 0;
        for (int b = b0; b < b1; ++b) sum += units(b);
        int64_t inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) warp_tot[warp] = inc;
        __syncthreads();
        int64_t base = inc - sum;
        total = 0;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            if (w < warp) base += warp_tot[w];
            total += warp_tot[w];
        }
        for (int b = b0; b < b1; ++b) {
            pre[b] = base;
            base += units(b);
        }
        __syncthreads();
    }
    const int64_t run = (total + gridDim.x - 1) / gridDim.x;
    const int64_t u0 = run * blockIdx.x;
    const int count = (int)max(min(run, total - u0), (int64_t)0);
    if (count <= 0) return;
    UnitCursor<RT, KT> cur;
    {
        int lo = 0, hi = p.batch;   // last b with pre[b] <= u0: requests without units share a start with the next
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= u0) lo = mid;
            else hi = mid;
        }
        cur.b = lo;
        cur.enter(p);
        int64_t at = u0 - pre[lo];
        const int64_t per_head = (int64_t)cur.nrt * cur.nkt;
        cur.h = (int)(at / per_head);
        at -= cur.h * per_head;
        cur.rt = (int)(at / cur.nkt);
        cur.kt = (int)(at - (int64_t)cur.rt * cur.nkt);
    }
    __syncthreads();
    if (p.head_dim < DT) {   // columns past the head size stay zero: no load writes them
        for (int i = tid; i < Cfg::stages * 2 * Cfg::tile_b / 16; i += kAttnThreads)
            reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    // ---- loads: key tile of the load cursor into a stage ---------------------------------------
    UnitCursor<RT, KT> ld = cur;
    const int ld_chunk = tid % CPR, ld_row = tid / CPR;
    constexpr int kRowStep = kAttnThreads / CPR;
    auto load_tile = [&](int stage) {
        if (ld_chunk * 8 < p.head_dim) {
            const uint32_t dst = sbase + stage * 2 * Cfg::tile_b;
            const int64_t head = ld.h * p.stride_head + ld_chunk * 8;
            const int* table = p.block_table + (int64_t)ld.b * p.table_stride;
            const int pos0 = ld.kt * KT;
            int64_t off[KT / kRowStep];
            bool live[KT / kRowStep];
#pragma unroll
            for (int i = 0; i < KT / kRowStep; ++i) {
                const int pos = pos0 + ld_row + i * kRowStep;
                const int pg = p.page_div.div(pos);
                live[i] = pos < ld.r.seq;
                const int id = live[i] ? __ldg(table + pg) : 0;
                if ((unsigned)id >= (unsigned)p.num_pages) live[i] = false;   // not a page of this cache
                off[i] = live[i] ? id * p.stride_page + (pos - pg * p.page_size) * p.stride_slot + head : 0;
            }
#pragma unroll
            for (int i = 0; i < KT / kRowStep; ++i) {
                const int row = ld_row + i * kRowStep;
                const uint32_t at = dst + row * Cfg::row_b + ((ld_chunk ^ (row & 7)) << 4);
                cp_async16(at, static_cast<const T*>(p.k_cache) + off[i], live[i]);
                cp_async16(at + Cfg::tile_b, static_cast<const T*>(p.v_cache) + off[i], live[i]);
            }
        }
        ld.next(p);
    };
    int loaded = 0;
#pragma unroll
    for (int s = 0; s < Cfg::stages - 1; ++s) {
        if (loaded < count) load_tile(s), ++loaded;
        cp_async_commit();
    }

    const float scale = p.flip ? -p.scale_log2 : p.scale_log2;
    uint32_t qf[DT / 16][4];
    float o[NT][4];
    float m[2], l[2];
    const int row0 = wm * 16 + (lane >> 2), col0 = 2 * (lane & 3);

    for (int it = 0; it < count; ++it) {
        const int ctx = cur.r.seq - cur.r.n;             // negative for a refused request (seq 0)
        const int rows = min(RT, cur.r.n * p.group - cur.rt * RT);
        if (it == 0 || cur.kt == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.0f;
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.0f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = row0 + 8 * half;
                const int at = cur.rt * RT + row, i = at / p.group, g = at - i * p.group;
                const T* q = static_cast<const T*>(p.q) + (int64_t)(cur.r.q0 + i) * p.q_stride_token +
                             (int64_t)(cur.h * p.group + g) * p.q_stride_head;
#pragma unroll
                for (int kk = 0; kk < DT / 16; ++kk) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int d = kk * 16 + c * 8 + col0;
                        qf[kk][half + 2 * c] =
                            (row < rows && d < p.head_dim) ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                    }
                }
            }
        }
        const int stage = it % Cfg::stages;
        cp_async_wait<Cfg::stages - 2>();
        __syncthreads();
        if (loaded < count) load_tile((it + Cfg::stages - 1) % Cfg::stages), ++loaded;
        cp_async_commit();
        const uint32_t sk = sbase + stage * 2 * Cfg::tile_b, sv = sk + Cfg::tile_b;
        const unsigned char* gv = smem + stage * 2 * Cfg::tile_b + Cfg::tile_b;

        // ---- S = Q K^T for this warp's TN keys ----
        float s[TN / 8][4];
#pragma unroll
        for (int j = 0; j < TN / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
            if (kk * 16 >= p.head_dim) break;
#pragma unroll
            for (int j = 0; j < TN / 16; ++j) {
                const int row = wk * TN + j * 16 + ((lane >> 4) << 3) + (lane & 7);
                const int chunk = kk * 2 + ((lane >> 3) & 1);
                uint32_t kf[4];
                ldmatrix_x4(kf, sk + row * Cfg::row_b + ((chunk ^ (row & 7)) << 4));
                mma_t<T>(s[2 * j], qf[kk], kf[0], kf[1]);
                mma_t<T>(s[2 * j + 1], qf[kk], kf[2], kf[3]);
            }
        }
        // ---- masks: only tiles that reach the new tokens or the end ----
        const int pos0 = cur.kt * KT;
        const bool tail = pos0 + KT > ctx;
        bool dirty = false;
        uint64_t win[2] = {~0ull, ~0ull};
        if (tail) {
            bool bad = false;
            for (int c = tid; c < Cfg::tile_b / 16; c += kAttnThreads)
                bad |= any_nonfinite<T>(*reinterpret_cast<const uint4*>(gv + c * 16));
            dirty = __syncthreads_or(bad);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = min(cur.rt * RT + row0 + 8 * half, cur.r.n * p.group - 1) / p.group;
                win[half] = cur.r.seq > 0 ? seen_window(p, cur.r, i, pos0 - ctx) : 0ull;
            }
        }
        // ---- running maximum, P = exp2(S - m), sums ----
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int j = 0; j < TN / 8; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float t = s[j][e] * scale;
                if (tail && !((win[e >> 1] >> (wk * TN + j * 8 + col0 + (e & 1))) & 1)) t = -INFINITY;
                s[j][e] = t;
                mx[e >> 1] = fmaxf(mx[e >> 1], t);
            }
        }
        float alpha[2], base[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
            mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
            base[half] = mx[half] == -INFINITY ? 0.0f : mx[half];
            alpha[half] = exp2_fast(m[half] - base[half]);
            m[half] = mx[half];
            l[half] *= alpha[half];
        }
        if (!__all_sync(0xffffffffu, alpha[0] == 1.0f && alpha[1] == 1.0f)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][0] *= alpha[0];
                o[nt][1] *= alpha[0];
                o[nt][2] *= alpha[1];
                o[nt][3] *= alpha[1];
            }
        }
        // P enters the second product in the cache's type; l sums the rounded values, so what is divided is
        // the weighted mean of the values with the weights that were used
        uint32_t pf[TN / 16][4];
#pragma unroll
        for (int j = 0; j < TN / 8; ++j) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float a = exp2_fast(s[j][2 * half] - base[half]), b = exp2_fast(s[j][2 * half + 1] - base[half]);
                const uint32_t u = pack2<T>(a, b);
                pf[j >> 1][(j & 1) * 2 + half] = u;
                const float2 f = unpack2<T>(u);
                l[half] += f.x + f.y;
            }
        }
        // ---- O += P V ----
#pragma unroll
        for (int j = 0; j < TN / 16; ++j) {
            const int row = wk * TN + j * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
            for (int n2 = 0; n2 < DT / 16; ++n2) {
                if (n2 * 16 >= p.head_dim) break;
                const int chunk = n2 * 2 + (lane >> 4);
                uint32_t vf[4];
                ldmatrix_x4_trans(vf, sv + row * Cfg::row_b + ((chunk ^ (row & 7)) << 4));
                if (dirty) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) vf[e] = finite2<T>(vf[e]);
                }
                mma_t<T>(o[2 * n2], pf[j], vf[0], vf[1]);
                mma_t<T>(o[2 * n2 + 1], pf[j], vf[2], vf[3]);
            }
        }
        if (dirty) {
            // infinities and NaN among this tile's values: a row takes them only from keys that it sees (0 * NaN
            // would carry a rejected branch's values into its siblings)
            float* pw = buf + warp * 16 * TN;
#pragma unroll
            for (int j = 0; j < TN / 8; ++j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float2 f = unpack2<T>(pf[j >> 1][(j & 1) * 2 + half]);
                    pw[((lane >> 2) + 8 * half) * TN + j * 8 + col0] = f.x;
                    pw[((lane >> 2) + 8 * half) * TN + j * 8 + col0 + 1] = f.y;
                }
            }
            __syncwarp();
            for (int x = 0; x < TN; ++x) {
                const int row = wk * TN + x;
                const bool see0 = (win[0] >> row) & 1, see1 = (win[1] >> row) & 1;
                const float p0 = pw[(lane >> 2) * TN + x], p1 = pw[((lane >> 2) + 8) * TN + x];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t raw = *reinterpret_cast<const uint32_t*>(gv + row * Cfg::row_b + ((nt ^ (row & 7)) << 4) + col0 * 2);
                    if (raw != finite2<T>(raw)) {
                        const float2 v = unpack2<T>(raw), f = unpack2<T>(finite2<T>(raw));
                        if (v.x != f.x) {
                            if (see0) o[nt][0] += p0 * v.x;
                            if (see1) o[nt][2] += p1 * v.x;
                        }
                        if (v.y != f.y) {
                            if (see0) o[nt][1] += p0 * v.y;
                            if (see1) o[nt][3] += p1 * v.y;
                        }
                    }
                }
            }
            __syncwarp();
        }

        if (cur.kt == cur.nkt - 1 || it == count - 1) {
            // ---- end of the segment, or of this CTA's run ----
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
                l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
            }
            if (WN > 1) {   // join the warps that shared the row tile's keys
                if ((lane & 3) == 0) {
                    ml[wk * RT + row0] = make_float2(m[0], l[0]);
                    ml[wk * RT + row0 + 8] = make_float2(m[1], l[1]);
                }
                __syncthreads();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                    for (int w = 0; w < WN; ++w) mm = fmaxf(mm, ml[w * RT + row0 + 8 * half].x);
                    const float safe = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
                    for (int w = 0; w < WN; ++w) {
                        const float2 v = ml[w * RT + row0 + 8 * half];
                        ll += v.y * exp2_fast(v.x - safe);
                    }
                    const float f = exp2_fast(m[half] - safe);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        o[nt][2 * half] *= f;
                        o[nt][2 * half + 1] *= f;
                    }
                    m[half] = mm;
                    l[half] = ll;
                }
#pragma unroll
                for (int w = 1; w < WN; ++w) {
                    if (wk == w) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            *reinterpret_cast<float2*>(buf + row0 * DT + nt * 8 + col0) = make_float2(o[nt][0], o[nt][1]);
                            *reinterpret_cast<float2*>(buf + (row0 + 8) * DT + nt * 8 + col0) = make_float2(o[nt][2], o[nt][3]);
                        }
                    }
                    __syncthreads();
                    if (wk == 0) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float2 a = *reinterpret_cast<const float2*>(buf + row0 * DT + nt * 8 + col0);
                            const float2 c = *reinterpret_cast<const float2*>(buf + (row0 + 8) * DT + nt * 8 + col0);
                            o[nt][0] += a.x, o[nt][1] += a.y, o[nt][2] += c.x, o[nt][3] += c.y;
                        }
                    }
                    __syncthreads();
                }
            }
            const int64_t seg0 = u0 + it - cur.kt, seg1 = seg0 + cur.nkt;   // units of the segment
            const bool whole = seg0 >= u0 && seg1 <= u0 + count;
            auto emit = [&](int row, int d, float a, float b, float inv) {   // two neighbouring outputs of one row
                const int at = cur.rt * RT + row, i = at / p.group, g = at - i * p.group;
                T* dst = static_cast<T*>(p.out) + (int64_t)(cur.r.q0 + i) * p.out_stride_token +
                         (int64_t)(cur.h * p.group + g) * p.out_stride_head + d;
                *reinterpret_cast<uint32_t*>(dst) = pack2<T>(a * inv, b * inv);
            };
            auto emit_lse = [&](int row, float mm, float ll) {
                const int at = cur.rt * RT + row, i = at / p.group, g = at - i * p.group;
                p.lse[(int64_t)(cur.r.q0 + i) * p.q_heads + cur.h * p.group + g] =
                    ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
            };
            if (whole) {
                if (wk == 0) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int row = row0 + 8 * half;
                        if (row >= rows) continue;
                        const float inv = l[half] == 0.0f ? 0.0f : 1.0f / l[half];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            if (nt * 8 < p.head_dim) emit(row, nt * 8 + col0, o[nt][2 * half], o[nt][2 * half + 1], inv);
                        if (p.lse && (lane & 3) == 0) emit_lse(row, m[half], l[half]);
                    }
                }
            } else {
                // a part: the first of the run (its segment began in an earlier CTA) or the last
                const int slot = 2 * blockIdx.x + (seg0 < u0 ? 0 : 1);
                if (wk == 0) {
                    float* po = p.part_o + (int64_t)slot * RT * DT;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        *reinterpret_cast<float2*>(po + row0 * DT + nt * 8 + col0) = make_float2(o[nt][0], o[nt][1]);
                        *reinterpret_cast<float2*>(po + (row0 + 8) * DT + nt * 8 + col0) = make_float2(o[nt][2], o[nt][3]);
                    }
                    if ((lane & 3) == 0) {
                        p.part_ml[slot * RT + row0] = make_float2(m[0], l[0]);
                        p.part_ml[slot * RT + row0 + 8] = make_float2(m[1], l[1]);
                    }
                }
                const int first = (int)(seg0 / run), last = (int)((seg1 - 1) / run);
                __threadfence();
                __syncthreads();
                if (tid == 0) s_last = atomicAdd(p.counters + first, 1) == last - first;
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    for (int e = tid; e < rows * (DT / 4); e += kAttnThreads) {
                        const int row = e / (DT / 4), d = (e - row * (DT / 4)) * 4;
                        float mm = -INFINITY, ll = 0.0f;
                        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
                        for (int c = first; c <= last; ++c) {
                            const int sl = 2 * c + (c == first ? 1 : 0);
                            const float2 v = __ldcg(p.part_ml + sl * RT + row);
                            const float4 po = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((int64_t)sl * RT + row) * DT + d));
                            const float top = fmaxf(mm, v.x), safe = top == -INFINITY ? 0.0f : top;
                            const float fa = exp2_fast(mm - safe), fb = exp2_fast(v.x - safe);
                            acc.x = acc.x * fa + po.x * fb;
                            acc.y = acc.y * fa + po.y * fb;
                            acc.z = acc.z * fa + po.z * fb;
                            acc.w = acc.w * fa + po.w * fb;
                            ll = ll * fa + v.y * fb;
                            mm = top;
                        }
                        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                        if (d < p.head_dim) {
                            emit(row, d, acc.x, acc.y, inv);
                            emit(row, d + 2, acc.z, acc.w, inv);
                        }
                        if (p.lse && d == 0) emit_lse(row, mm, ll);
                    }
                    if (tid == 0) p.counters[first] = 0;   // ready for the next call
                }
            }
        }
        cur.next(p);
    }
    cp_async_wait<0>();
}

template <typename T, int DT, int WM>
static cudaError_t launch_attn(const TreeAttnParams& p, cudaStream_t st)
{
    using Cfg = AttnCfg<DT, WM>;
    auto kernel = tree_attn_kernel<T, DT, WM>;
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem);
    if (err != cudaSuccess) return err;
    kernel<<<num_sms() * Cfg::per_sm, kAttnThreads, Cfg::smem, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int DT>
static cudaError_t launch_attn_rows(const TreeAttnParams& p, int rows, cudaStream_t st)
{
    if (rows <= 16) return launch_attn<T, DT, 1>(p, st);
    if (rows <= 32) return launch_attn<T, DT, 2>(p, st);
    return launch_attn<T, DT, 4>(p, st);
}

cudaError_t launch_tree_attn(const TreeAttnParams& p, int dtype, int max_rows, cudaStream_t st)
{
    if (p.head_dim <= 128) return launch_tree_attn_tc(p, dtype, max_rows, st);
    return dtype == 0 ? launch_attn_rows<__half, 256>(p, max_rows, st) : launch_attn_rows<__nv_bfloat16, 256>(p, max_rows, st);
}

// Most parts a call can leave: two per CTA (one CTA per SM and up to 256 rows on the tensor-memory path, two CTAs
// per SM and up to 64 rows on the other), of the padded head size.
AttnWorkspace tree_attn_workspace(int head_dim)
{
    const bool tc = head_dim <= 128;
    const int64_t dt = head_dim <= 64 ? 64 : tc ? 128 : 256;
    const int64_t ctas = (int64_t)num_sms() * (tc ? 1 : 2), rows = 2 * ctas * (tc ? 256 : 64);
    AttnWorkspace w;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    w.counters = 256;
    w.part_ml = w.counters + up(2 * ctas * sizeof(int));
    w.part_o = w.part_ml + up(rows * sizeof(float2));
    w.total = w.part_o + up(rows * dt * sizeof(float));
    return w;
}

}  // namespace dsv41
