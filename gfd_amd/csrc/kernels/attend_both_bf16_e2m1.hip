// Attention over the paged cache, a shared prefix and what follows: rows in Bf16, cache in E2m1.
#include "attend_both.h"

template int gfd::kv::launch_both<gfd::kv::Bf16, gfd::kv::E2m1>(const Call&, const Cache4&, const Stage&, const Stage&, int,
                                                          bool, hipStream_t);
