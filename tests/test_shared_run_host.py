"""Runs of the attention behind one shared prefix on the CPU: what their host side does with fields that nothing
reads.  The library runs over a stand-in for the HIP runtime (fake_hip.cc, preloaded into a child process)."""
import ctypes
import json
import os
import shutil
import subprocess
import sys

import pytest

from test_host_launches import HERE, ROCM, Launches

Q, O, K, V = 1 << 20, 1 << 30, 1 << 31, 1 << 32  # stand-in device addresses
LEAST, MOST = -(1 << 31), (1 << 31) - 1


def failure(h, call):
    """The error's message, or None."""
    try:
        call()
    except h.qattn.QattnError as e:
        return [e.code, str(e)]
    return None


def unread_cache_fields():
    """[[fields, failure of create, kernels launched, failure of a second batch, of a rebind, of a batch that
    reads pages]] of runs whose own keys are rows, with no prefix."""
    h, out = Launches(), []
    q = h.qattn
    for fields in (dict(), dict(page_size=-7), dict(page_size=48), dict(page_size=1 << 30), dict(page_size=(1 << 30) + 1),
                   dict(page_size=MOST), dict(page_size=LEAST), dict(pages=LEAST, page_size=MOST), dict(format=2),
                   dict(format=3), dict(format=LEAST), dict(format=MOST, page_size=MOST, pages=MOST),
                   dict(k=3, v=5, k_scale=7, v_scale=9)):
        cache = q.make_kv_cache(None, None, 0, 0)
        for name, value in fields.items():
            setattr(cache, name, value)
        names, run = [], []
        h.on = lambda name, *rest: names.append(name)
        made = failure(h, lambda: run.append(h.ctx.shared_run(q.make_shared_desc(Q, O, cache, [0, 40, 41], [40, 9], k=K, v=V))))
        row = [str(fields), made]
        if not made:
            run[0].encode()
            row += [names[:], failure(h, lambda: run[0].update([0, 3], [3])),
                    failure(h, lambda: run[0].rebind(Q + 64, O, cache, K, V)),
                    failure(h, lambda: run[0].update([0, 3], [3], prefix_pages=[0], prefix_len=1))]
            run[0].encode()
            run[0].destroy()
        out.append(row)
    return out


MANY = dict(cu_q=list(range(601)), own_len=[1] * 600, prefix_pages=[], prefix_len=0)  # a long plan, no partial results
LONG = dict(cu_q=[0, 1], own_len=[1], prefix_pages=[0] * 4000, prefix_len=64000)      # a short one, cut into many
BOTH = dict(cu_q=[0, 900, 901], own_len=[900, 1], prefix_pages=[0] * 10000, prefix_len=160000)
POINTERS = {name: 8 * i for i, name in enumerate(("items", "segs", "starts", "merges", "positions", "groups", "part_o", "part_ml"), 12)}


def failed_allocations():
    """[[step, failure, the run's info, launches: [kernel, grid, pointers, whether any points into freed memory]]] of
    a run whose device allocations fail now and then."""
    h, out = Launches(), []
    q, lib = h.qattn, h.qattn.lib()
    cache = q.make_kv_cache(K, V, 8, 16)

    def step(name, call, fails=0):
        lib.qattn_debug_fail_allocs(fails)
        error = failure(h, call)
        lib.qattn_debug_fail_allocs(0)
        launches = []

        def on(kernel, grid, block, args):
            at = {n: h.word(args, 0, ctypes.c_uint64, o) for n, o in POINTERS.items()}
            launches.append([kernel, grid, list(at.values()), any(h.fake.fake_hip_freed(x) for x in at.values())])

        h.on = on
        if run:
            run[0].encode()
        out.append([name, error, run[0].info().as_dict() if run else None, launches])

    run = []
    desc = lambda b: q.make_shared_desc(Q, O, cache, k=K, v=V, **b)  # noqa: E731
    step("create fails", lambda: run.append(h.ctx.shared_run(desc(LONG))), 1)
    step("create fails", lambda: run.append(h.ctx.shared_run(desc(LONG))), 2)
    step("create", lambda: run.append(h.ctx.shared_run(desc(MANY))))
    step("update", lambda: run[0].update(**MANY))  # both images hold a long plan now
    step("workspace fails", lambda: run[0].update(**LONG), 1)
    step("update", lambda: run[0].update(**LONG))
    step("image fails", lambda: run[0].update(**BOTH), 1)
    step("both fail", lambda: run[0].update(**BOTH), 2)
    step("update", lambda: run[0].update(**BOTH))
    step("update", lambda: run[0].update(**MANY))
    run[0].destroy()
    return out


def host_memory():
    """{call: how often it returned what}, each call again and again with its first, second, .. allocation on the host
    failing, until it makes no more."""
    h, new, out = Launches(), ctypes.CDLL(os.environ["FAIL_NEW"]), {}
    new.fail_new_at.argtypes = [ctypes.c_long]
    q, lib, ctx = h.qattn, h.qattn.lib(), h.ctx.handle
    cache = q.make_kv_cache(K, V, 8, 16)
    desc = lambda b: q.make_shared_desc(Q, O, cache, k=K, v=V, **b)  # noqa: E731
    first, second, refused, handle, words = desc(LONG), desc(BOTH), desc(LONG), ctypes.c_void_p(), ctypes.c_int64()
    refused.q_heads = 7

    def sweep(name, call, prepare=lambda: None, after=lambda: None):
        counts, n, more = {}, 0, True
        while more:
            n += 1
            prepare()
            new.fail_new_at(n)
            code = call()
            more = bool(new.fail_new_did())
            new.fail_new_at(0)
            if more and name != "destroy":
                counts[code] = counts.get(code, 0) + 1
            after()
        out[name] = [n, counts, code]

    def create():
        return lib.qattn_shared_run_create(ctx, ctypes.byref(first), ctypes.byref(handle))

    def destroy():
        lib.qattn_shared_run_destroy(handle)
        handle.value = None

    def used():  # a run with launches on two streams
        create()
        lib.qattn_shared_run_encode(handle, None)
        lib.qattn_shared_run_encode(handle, 0x5000)

    d = second
    sweep("create", create, after=destroy)
    sweep("update", lambda: lib.qattn_shared_run_update(handle, d.prefix_pages, d.prefix_len, d.cu_q, d.nseq, d.own_len, None), used, destroy)
    sweep("encode", lambda: lib.qattn_shared_run_encode(handle, 0x6000), used, destroy)
    sweep("describe", lambda: lib.qattn_shared_plan_describe(ctypes.byref(first), None, 0, ctypes.byref(words), None))
    sweep("refused", lambda: lib.qattn_shared_run_create(ctx, ctypes.byref(refused), ctypes.byref(handle)))
    sweep("destroy", destroy, used)
    return out


CASES = {f.__name__: f for f in (unread_cache_fields, failed_allocations, host_memory)}


@pytest.fixture(scope="module")
def run_child(tmp_path_factory):
    compiler = shutil.which("g++")
    if not compiler or not os.path.isdir(os.path.join(ROCM, "include", "hip")):
        pytest.skip("no g++ or HIP headers")
    lib = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-I" + os.path.join(ROCM, "include"), "-o", lib,
                    os.path.join(HERE, "fake_hip.cc")], check=True)
    new = os.path.join(os.path.dirname(lib), "libfail_new.so")
    subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", "-o", new, os.path.join(HERE, "fail_new.cc"), "-ldl"], check=True)

    def run(case, failing_new=False):
        preload = " ".join(v for v in (os.environ.get("LD_PRELOAD"), new if failing_new else None, lib) if v)
        out = subprocess.run([sys.executable, os.path.abspath(__file__), case], check=True, capture_output=True, text=True,
                             env=dict(os.environ, LD_PRELOAD=preload, FAKE_HIP=lib, FAIL_NEW=new), timeout=60)
        return json.loads(out.stdout)

    return run


def test_cache_fields_that_nothing_reads_may_hold_anything(run_child):
    """Runs that read no page need the cache's kv_heads, head_dim and dtype only: whatever the other fields hold, the
    run is planned, launched (by the kernel of 16-bit keys), updated and rebound; a batch that reads pages is
    refused for them."""
    seen = run_child("unread_cache_fields")
    assert len(seen) == 13
    for fields, made, kernels, updated, rebound, paged in seen:
        assert made is None and updated is None and rebound is None, (fields, made, updated, rebound)
        assert kernels and all("shared_" in k for k in kernels) and "ILb0ELi0ELi128E" in kernels[0], (fields, kernels)
        assert paged is not None and paged[0] == -1, fields


def test_a_failed_allocation_leaves_the_run_its_plan(run_child):
    """Device memory that runs out in a create or an update is an error of its own; the run goes on with the plan that
    it had, in memory that is still its own."""
    steps = run_child("failed_allocations")
    before = None
    for name, error, info, launches in steps:
        assert (error is not None) == ("fail" in name), (name, error)
        assert error is None or (error[0] == -3 and "hipMalloc" in error[1]), error
        assert not any(freed for *_, freed in launches), name
        if "fail" in name:
            assert before is None or [info, launches] == before, name
        elif before:
            assert [info, launches] != before
        before = info and [info, launches]
    assert [len(launches) for *_, launches in steps] == [0, 0, 1, 1, 1, 2, 2, 2, 2, 1]


def test_host_memory_that_runs_out_is_an_error_code(run_child):
    """No exception leaves a call, whichever of its allocations fails: planning and encoding report it, a refusal stays
    one, and a run is destroyed all the same."""
    if "QATTN_LIB" in os.environ:
        pytest.skip("an instrumented library brings its own operator new")
    seen = run_child("host_memory", failing_new=True)
    for name in ("create", "update", "encode", "describe"):
        n, counts, last = seen[name]
        assert last == 0 and set(counts) <= {"-3", "0"} and counts["-3"] >= (1 if name == "encode" else 20), (name, seen[name])
    n, counts, last = seen["refused"]
    assert last == -1 and set(counts) == {"-1"} and n > 1
    assert seen["destroy"][0] > 1


if __name__ == "__main__":
    print(json.dumps(CASES[sys.argv[1]]()))
