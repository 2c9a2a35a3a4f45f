// Attention over the paged cache, a shared prefix and what follows: rows in Fp16, cache in Fp16.
#include "attend_both.h"

template int gfd::kv::launch_both<gfd::kv::Fp16, gfd::kv::Fp16>(const Call&, const Cache&, const Stage&, const Stage&, int,
                                                          bool, hipStream_t);
