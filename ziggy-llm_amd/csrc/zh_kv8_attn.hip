// zh_kv8_attn.hip -- attention over the cache held in 8 bits.
//
// o = sum_t w_t v_t / sum_t w_t, w_t = 2^(qscale q.k_t - max), in one pass with the running maximum and
// sum; a block's scale multiplies its scores and its weights, so the codes enter as they are.
#include "zh_longctx.h"

namespace zh {

namespace {

__device__ __forceinline__ uint32_t first_seen(uint32_t pos, uint32_t window) {
    return window && pos >= window ? pos + 1 - window : 0u;
}

// A workgroup takes one head of one query, 256 positions at a time.
template <int HD> __global__ void __launch_bounds__(256) kv8_attn_simple_kernel(Kv8Attn p) {
    __shared__ float q[HD], w[256], red[4];
    const int tid = threadIdx.x, head = blockIdx.x, kvh = head / (p.heads / p.c.nkv);
    const size_t base = (size_t)kvh * p.c.blocks;
    for (uint32_t qi = blockIdx.y; qi < p.queries; qi += gridDim.y) {
        const uint32_t pos = p.position + qi, lo = first_seen(pos, p.window);
        __syncthreads();
        for (int d = tid; d < HD; d += 256) q[d] = p.q[qi * p.q_stride + (size_t)head * HD + d] * p.qscale;
        __syncthreads();
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (uint32_t at = lo & ~31u; at <= pos; at += 256) {
            const uint32_t t = at + tid;
            const bool seen = t >= lo && t <= pos;
            float s = -INFINITY;
            if (seen) {
                const int8_t *k = p.c.kc + (base * kKv8Block + t) * HD;
                float a = 0.f;
                for (int d = 0; d < HD; d++) a += q[d] * (float)k[d];
                s = a * p.c.ks[base + t / kKv8Block];
            }
            float mx = wave_max_f32(s);
            if ((tid & 63) == 0) red[tid >> 6] = mx;
            __syncthreads();
            mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
            const float al = exp2f(m - mx), e = seen ? exp2f(s - mx) : 0.f;
            m = mx;
            w[tid] = e;
            __syncthreads();
            l *= al, o *= al;
            if (tid < HD) {
                const int n = (int)min(256u, pos - at + 1);
                for (int i = 0; i < n; i++) {
                    if (at + i < lo) continue;
                    const size_t b = base + (at + i) / kKv8Block;
                    l += w[i];
                    o += w[i] * p.c.vs[b] * (float)p.c.vc[b * (kKv8Block * HD) + tid * kKv8Block + ((at + i) & 31)];
                }
            }
            __syncthreads();
        }
        if (tid < HD) p.out[((size_t)qi * p.heads + head) * HD + tid] = o / l;
    }
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8Attn &p, int cus, hipStream_t s) {
    const dim3 grid(p.heads, p.queries < 32768u ? p.queries : 32768u);
    switch (p.c.hd) {
    case 64: hipLaunchKernelGGL(kv8_attn_simple_kernel<64>, grid, dim3(256), 0, s, p); break;
    case 96: hipLaunchKernelGGL(kv8_attn_simple_kernel<96>, grid, dim3(256), 0, s, p); break;
    case 128: hipLaunchKernelGGL(kv8_attn_simple_kernel<128>, grid, dim3(256), 0, s, p); break;
    case 256: hipLaunchKernelGGL(kv8_attn_simple_kernel<256>, grid, dim3(256), 0, s, p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace zh
