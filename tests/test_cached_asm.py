"""The check of test_kernel_asm.py for the prompt kernel of the attention over a cache, whose
keys and values arrive by the same loads."""
import pytest

import test_kernel_asm as kernel_asm

asm_of = kernel_asm.asm_of


@pytest.mark.parametrize("wide", [1, 2, 3, 4])
@pytest.mark.parametrize("type", ["t", "f"])
def test_m0_only_feeds_the_lds_dma_loads(asm_of, type, wide):
    kernel_asm.test_m0_only_feeds_the_lds_dma_loads(
        asm_of, "cached_prompt.hip",
        f"_ZN3tfd12_GLOBAL__N_120cached_prompt_kernelI{type}Li{wide}E")
