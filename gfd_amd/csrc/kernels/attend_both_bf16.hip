// Attention over the paged cache, a shared prefix and what follows: rows in Bf16, cache in Bf16.
#include "attend_both.h"

template int gfd::kv::launch_both<gfd::kv::Bf16, gfd::kv::Bf16>(const Call&, const Cache&, const Stage&, const Stage&, int,
                                                          bool, hipStream_t);
