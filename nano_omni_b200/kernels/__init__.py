"""Registry of kernel classes by ``name``: the reference's (src/nano_omni/kernels/__init__.py:11-29) and those without a
counterpart there (masked attention, the 8-bit cache)."""

from __future__ import annotations

import functools

from nano_omni_b200.core import Kernel


@functools.cache
def classes() -> dict[str, type[Kernel]]:
    from nano_omni_b200.kernels import (
        cache,
        dense_bf16,
        dense_int8_fp8,
        dense_nvfp4,
        masked,
        matmul,
        norm_rope,
        quantize,
        sol,
        sol_exact,
    )

    found: dict[str, type[Kernel]] = {}
    modules = (dense_bf16, dense_int8_fp8, dense_nvfp4, matmul, norm_rope, quantize, sol, sol_exact, masked, cache)
    for module in modules:
        for value in vars(module).values():
            if isinstance(value, type) and issubclass(value, Kernel) and value is not Kernel and value.name:
                assert value.name not in found or found[value.name] is value, f"duplicate kernel {value.name}"
                found[value.name] = value
    return found
