// Checks shared by the entry points that take a paged cache.
#pragma once

#include "typed.cuh"

namespace b200 {

inline int check_paged(const b200_paged* c) {
    if (!c || c->requests < 0 || c->tokens < 0 || c->heads < 1 || c->kv_heads < 1 || c->heads % c->kv_heads != 0 || c->heads > 4096 ||
        c->head_dim < 1 || c->head_dim > 2048 || c->pages < 1 || c->page_size < 1 || c->table_width < 0 || c->table_stride < 0)
        return B200_EINVAL;
    if ((long long)c->table_width * c->page_size > 0x7fffffffll) return B200_ELIMIT;
    if (c->dtype != B200_DTYPE_F16 && c->dtype != B200_DTYPE_BF16) return B200_EUNSUPPORTED;
    if (!c->k_pages || !c->v_pages || !c->row_starts) return B200_EINVAL;
    if (c->requests > 0 && (!c->lengths || (c->table_width > 0 && !c->page_table))) return B200_EINVAL;
    return B200_OK;
}

}  // namespace b200
