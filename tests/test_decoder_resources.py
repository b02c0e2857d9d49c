"""Scratch memory of the decoder's kernels, by the notes of the library's code objects: few instances keep some, and they are known."""
import re

import pytest

from tests.test_kernel_resources import scratch_bytes  # noqa: F401  (a fixture)

# what the heads' width, the rows of a tile, the waves that share the columns and the sixteens of columns a wave make of it, by kernel
KNOWN = [r"attn_forward_kernel<Shape<(F16|BF16), [012], 32, 128, 2, 2, 4>, \w+>", r"attn_forward_kernel<Shape<(F16|BF16), 0, 128, 64, 1, 2, 4>, \w+>",
         r"attn_grad_kv_kernel<Shape<BF16, 1, 32, 128, 2, 2, 4> ?>", r"attn_grad_kv_kernel<Shape<F16, 0, 64, 64, 1, 2, 4> ?>",
         r"attn_grad_kv_kernel<Shape<F16, [012], 64, 128, 4, 2, 4> ?>"]


@pytest.mark.parametrize("kernel,instances", [("attn_forward_kernel<", 150), ("attn_grad_q_kernel<", 76), ("attn_grad_kv_kernel<", 76),
                                              ("attn_join", 6), ("add_norm_", 97)])
def test_scratch_memory_of_the_decoders_kernels(scratch_bytes, kernel, instances):  # noqa: F811
    found = {name: size for name, size in scratch_bytes.items() if kernel in name}
    assert len(found) == instances, sorted(found)
    kept = {name: size for name, size in found.items() if size}
    assert all(any(re.search(known, name) for known in KNOWN) for name in kept), kept
    assert all(size <= 48 for size in kept.values()), kept
