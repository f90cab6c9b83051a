// af_kv_pool.h — host checks of a paged pool, and where a layer's rows lie in it.
#pragma once

#include "af_common.h"

namespace af {

inline size_t pool_element_bytes(const af_kv_pool& p) {
    return p.dtype == AF_KV_FP8_E4M3 ? 1 : 2;
}
inline size_t pool_row_bytes(const af_kv_pool& p) {
    return size_t(p.n_kv_heads) * p.head_dim * pool_element_bytes(p);
}
// Bytes of one layer's K rows (or V rows).
inline size_t pool_slab_bytes(const af_kv_pool& p) {
    return size_t(p.total_blocks) * p.block_size * pool_row_bytes(p);
}

inline int check_pool(const af_kv_pool* p) {
    if (!p || !p->base || p->n_layers <= 0 || p->n_kv_heads <= 0 || p->head_dim <= 0 ||
        p->total_blocks <= 0 || p->block_size <= 0)
        return AF_ERR_INVALID_ARG;
    if (p->block_size & (p->block_size - 1)) return AF_ERR_UNSUPPORTED;
    if (p->dtype != AF_KV_FP16 && p->dtype != AF_KV_FP8_E4M3) return AF_ERR_UNSUPPORTED;
    if (p->flags & ~AF_KV_POOL_SHARED_BLOCKS) return AF_ERR_INVALID_ARG;
    if (pool_row_bytes(*p) % 16) return AF_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(p->base) % 16) return AF_ERR_INVALID_ARG;
    return AF_OK;
}

struct PoolLayer {
    uint8_t* k;
    uint8_t* v;
    const float* k_scales;  // FP8: [n_kv_heads] each
    const float* v_scales;
    PoolLayer(const af_kv_pool& p, int layer) {
        const size_t slab = pool_slab_bytes(p);
        k = static_cast<uint8_t*>(p.base) + size_t(2 * layer) * slab;
        v = k + slab;
        k_scales = v_scales = nullptr;
        if (p.dtype == AF_KV_FP8_E4M3 && p.scales) {
            k_scales = p.scales + size_t(layer) * 2 * p.n_kv_heads;
            v_scales = k_scales + p.n_kv_heads;
        }
    }
};

}  // namespace af
