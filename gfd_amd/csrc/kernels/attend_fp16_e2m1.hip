// Attention over the paged cache: rows in Fp16, cache in E2m1 (one file per pair of types, compiled side by side).
#include "attend_rows.h"
#include "attend_tiles.h"

template int gfd::kv::launch_rows<gfd::kv::Fp16, gfd::kv::E2m1>(const Call&, const Cache4&, const Stage&, const Stage&, int,
                                                          bool, int, hipStream_t);
template int gfd::kv::launch_tiles<gfd::kv::Fp16, gfd::kv::E2m1>(const Call&, const Cache4&, const Stage&, const Stage&, int,
                                                           int, hipStream_t);
