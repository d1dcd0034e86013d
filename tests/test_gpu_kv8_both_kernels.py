"""Attention over the 8-bit cache with each of its two kernels at every size, not only where the call's own rule
takes it: the cases and tolerances of test_gpu_kv8.py (needs a B200)."""
import pytest

from test_gpu_kv8 import (test_a_layer_of_a_shared_pool, test_attention_at_the_edges_of_its_tiles,  # noqa: F401
                          test_attention_matches_64_bit, test_attention_scales, test_attention_with_value_scales_far_apart,
                          test_bf16_queries_outside_f16, test_c_calls_with_a_workspace_of_any_content,
                          test_contexts_longer_than_one_range_with_many_sequences,
                          test_device_side_errors_are_reported_and_the_rest_computed,
                          test_nan_reaches_only_the_rows_that_see_it, test_offsets_past_32_bits, test_ragged_rows_of_one_call,
                          test_repeats_streams_and_graphs_give_the_same_bits)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["few", "many"])
def kernel(request, monkeypatch):
    monkeypatch.setenv("BZB_KV8_ATTENTION", request.param)
