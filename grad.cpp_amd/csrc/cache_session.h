// A session's context in and out of a paged cache (gh_session_store, gh_session_restore).
#pragma once

#include "kernels_common.h"

struct gh_cache;

namespace gh {

// A new sequence of the cache with the first `length` positions of sequence `seq` of a session, all layers.  Refuses a cache of
// another shape or device.  The work is enqueued on the session's stream.
int cache_from_session(gh_cache* cache, const KvLayout& kv, int layers, int seq, int length, hipStream_t stream);

// The first `length` positions of cache sequence seqs[b] become sequence b's, b < batch.
void cache_to_session(gh_cache* cache, const int32_t* seqs, int batch, const KvLayout& kv, int layers, int length, hipStream_t stream);

}  // namespace gh
