"""Errors on the GPU: one call's failure is not reported by the next."""
import numpy as np
import pytest

import shared_ref as ref
from test_gpu_shared import Case

pytestmark = pytest.mark.gpu


def test_a_failed_allocation_is_no_later_launch_s_error(ctx, qattn):
    """Device memory that runs out leaves an error in the HIP runtime, per thread; a launch after it is checked for
    its own."""
    c = Case(ctx, qattn, 150, [1] * 20, [1 + 37 * i % 90 for i in range(20)], page=16, form="int8")
    run = ctx.shared_run(c.desc())
    rows, cu = ref.to_bits(np.random.default_rng(1).standard_normal((20, 4096)), False), np.array([0, 7, 20], np.int32)
    x, y, positions = ctx.upload(rows), ctx.alloc(20 * 8192), ctx.upload(np.arange(20, dtype=np.int32))
    slots = ctx.upload(np.full(20, -1, np.int64))  # writes nothing, reads zeros
    old = ctx.run(qattn.make_desc(x.ptr, x.ptr, x.ptr, y.ptr, cu))
    calls = {
        "shared": run.encode,
        "rope": lambda: ctx.rope(qattn.make_rope_desc(positions.ptr, 20, (x.ptr, y.ptr, 16))),
        "write": lambda: ctx.kv_write(c.cache, x.ptr, x.ptr, slots.ptr, 20),
        "read": lambda: ctx.kv_read(c.cache, slots.ptr, 20, y.ptr, y.ptr),
        "run": old.encode,
        "prefill": lambda: ctx.prefill(qattn.make_desc(x.ptr, x.ptr, x.ptr, y.ptr, cu)),
        "norm and rope": lambda: ctx.qk_norm_rope_qkv(x.ptr, y.ptr, y.ptr + 20 * 4096, cu),
        "pool": lambda: ctx.pool_last_l2(x.ptr, 4096, 1024, cu, y.ptr),
    }
    for name, call in calls.items():
        print("after a failed allocation:", name, flush=True)
        with pytest.raises(qattn.QattnError) as e:
            ctx.alloc(1 << 50)
        assert e.value.code == qattn.ENOMEM
        call()
    ctx.synchronize()
    c.check()
    run.destroy()
    old.destroy()
    for b in (x, y, positions, slots):
        b.free()
    c.free()
