// Attention over the paged cache: rows in Bf16, cache in E4m3 (one file per pair of types, compiled side by side).
#include "attend_rows.h"
#include "attend_tiles.h"

template int gfd::kv::launch_rows<gfd::kv::Bf16, gfd::kv::E4m3>(const Call&, const Cache&, const Stage&, const Stage&, int,
                                                          bool, int, hipStream_t);
template int gfd::kv::launch_tiles<gfd::kv::Bf16, gfd::kv::E4m3>(const Call&, const Cache&, const Stage&, const Stage&, int,
                                                           int, hipStream_t);
