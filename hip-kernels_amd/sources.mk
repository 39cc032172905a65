# The HIP sources of libgptoss_moe.so, for its own build and the sanitizer's.
SOURCES := moe_route moe_experts moe_decode moe_prefill moe_midstream moe_stages moe_checkpoint moe_stack moe_capi attn_append attn_decode attn_prefill attn_join attn_capi moe_select mx_quantize mx_product mx_tile mx_stream mx_capi
