"""The checked build (RI_B200_CHECK_BOUNDS=1) of the kernels over a cache in 8 bits: silent on ordinary work, and it speaks, and follows
nothing, where a page, a slot or a position lies outside.  In a process of its own: the build is chosen when the package is imported."""
import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = textwrap.dedent("""
    import sys, math, torch, pathlib, tempfile
    sys.path.insert(0, {root!r}); sys.path.insert(0, {tests!r})
    from conftest import make_model, random_tokens, rel_err
    from test_quantized_cache_gpu import DEV, RUNS, ATTEND, Step, _write, _check_written
    from rust_inference_b200 import Model
    from rust_inference_b200.engine.engine import Engine
    from rust_inference_b200.kernels import attention, build, ops, quantized_cache as qc
    mine = ("quantized_cache", "attention_quantized", "token_logprobs")
    assert build.CHECKED and all(build.library_path(m).endswith(f"checked/libri_{{m}}.so") for m in mine)

    # ---- ordinary work ----
    model = make_model(pathlib.Path(tempfile.mkdtemp()), "A", std=0.08)
    toks = random_tokens(90, model.cfg["vocab_size"], seed=1)
    want = model.plain_logits(toks)
    for dtype in ("float32", "bfloat16"):
        eng = Engine.from_pretrained(model.folder, dtype=dtype, max_tokens=512, cache_dtype="int8")
        s = eng.alloc_slot()
        head = eng.step([s], [toks[:70]], "all").cpu()
        tail = torch.cat([eng.step([s], [[t]], "last").cpu() for t in toks[70:]])
        assert rel_err(torch.cat([head, tail]), want) <= 0.15          # (what 8 bits cost; the ordinary build's tests are exact)
        eng.check_device_status()
    scores = Model(eng).score(toks, top=5)
    assert len(scores.top) == 89
    assert set(mine) <= set(build.loaded_cuda_modules()) and ops.bounds_report() == []

    def call(step, dtype, n_heads, hd, **limits):
        q = torch.randn(step.n_tokens, n_heads * hd, device=DEV).to(dtype)
        out = torch.full_like(q, 7.0)
        attention.attention(q, step.layer, out, step.context(dtype), n_heads=n_heads, n_kv_heads=step.n_kv, head_dim=hd, scale=0.1, **limits)
        return out

    def limits_of(step):
        ops.bounds_set_limits(264, step.page_table.shape[0], step.layer.k.shape[0])

    for runs in RUNS.values():
        for hd, rot, dtype in ((64, 64, torch.bfloat16), (128, 0, torch.float32), (24, 24, torch.bfloat16)):
            step = Step(runs, 2, hd)
            step.fill()
            limits_of(step)
            rows = torch.randn(step.n_tokens, 8 * hd).to(dtype)
            before = step.host()
            q, _ = _write(step, rows, n_heads=4, rot=rot, style=0)
            _check_written(step, rows, before, q, n_heads=4, rot=rot, style=0)
    for runs in list(ATTEND.values()) + [[(31990, 1)], [(700, 300)], [(2000, 1)] * 9]:
        for n_heads, hd, dtype in ((4, 64, torch.bfloat16), (14, 128, torch.float32), (6, 24, torch.bfloat16)):
            step = Step(runs, 2, hd)
            step.arrays([(s + n, 0) for s, n in runs])
            step.fill() if max(s for s, _ in runs) < 1000 else [t.fill_(0.01) for t in (step.layer.k_scale, step.layer.v_scale)]
            step.arrays(runs)
            limits_of(step)
            for limits in ({{}}, {{"window": 50}}, {{"chunk": 48}}):
                assert call(step, dtype, n_heads, hd, **limits).isfinite().all()
    assert ops.bounds_report() == []

    # ---- a page, a slot, a position outside: recorded by each kernel, and nothing of the cache written ----
    def outside(kind, hd, runs=[(70, 1), (70, 1)], dtype=torch.bfloat16):
        step = Step(runs, 2, hd)
        step.fill()
        limits_of(step)
        pages, slots, per = step.layer.k.shape[0], step.page_table.shape[0], step.page_table.shape[1]
        if kind == "page":
            step.page_table[step.slots[1]] = pages + 3
            bad = ("a page that does not exist", pages + 3, pages)
        elif kind == "slot":
            step.seq_slot[1] = slots + 2
            bad = ("a cache slot that does not exist", slots + 2, slots)
        else:
            step.seq_start[1] += 64 * per
            step.seq_len[1] += 64 * per
            step.max_len += 64 * per
            bad = ("a position beyond a sequence's page table", None, per)
        return step, bad

    def heard(module, bad):
        torch.cuda.synchronize()
        rep = ops.bounds_report()
        assert len(rep) == 1 and rep[0][0] == module and rep[0][1] == bad[0] and rep[0][3] == bad[2] and rep[0][4] >= 1, (rep, bad)
        assert bad[1] is None or rep[0][2] == bad[1], (rep, bad)

    for kind in ("page", "slot", "position"):
        for hd in (64, 128, 24):
            for runs in ([(70, 1), (70, 1)], [(70, 3), (70, 9)]):
                step, bad = outside(kind, hd, runs)
                before = step.host()
                rows = torch.randn(step.n_tokens, 8 * hd).bfloat16()
                step.max_len = min(step.max_len, 100)
                _write(step, rows, n_heads=4, rot=0, style=0)
                heard("quantized_cache", bad)
                after = step.host()
                good = set(int(p) for p in step.table[step.slots[0]])
                for a, b in zip(before, after):
                    same = [torch.equal(a[p].nan_to_num(9.0) if a.is_floating_point() else a[p], b[p].nan_to_num(9.0) if b.is_floating_point() else b[p]) for p in range(a.shape[0])]
                    assert all(s or p in good for p, s in enumerate(same))
                assert not torch.equal(before[0], after[0])                # (the other sequence's tokens are there)
        for hd in (64, 128):
            for dtype in (torch.bfloat16, torch.float32):
                step, bad = outside(kind, hd)
                call(step, dtype, 4, hd)
                heard("attention_quantized", bad)
            step, bad = outside(kind, hd)
            n = step.layer.k.shape[0]
            k, v = (torch.full(step.layer.k.shape, 7.0, device=DEV, dtype=torch.float16) for _ in range(2))
            where = (step.page_table, step.seq_slot, step.seq_start, step.seq_len)
            qc.widen(step.layer, k, v, torch.zeros(2, 2, 2, device=DEV), *where, max_len=step.max_len)
            heard("quantized_cache", bad)
            k, v = k.float().fill_(7.0), v.float().fill_(7.0)
            qc.read(step.layer, k, v, step.page_table, step.seq_slot, torch.zeros_like(step.seq_start), step.seq_len, max_len=step.max_len)
            heard("quantized_cache", bad)
            theirs = [p for p in range(n) if p not in set(int(p) for p in step.table[step.slots[0]])]
            if kind != "position":
                assert (k[theirs] == 7.0).all() and (v[theirs] == 7.0).all()
    print("checked build ok")
""")


def test_silent_on_ordinary_work_and_speaks_on_a_bad_index():
    env = dict(os.environ, RI_B200_CHECK_BOUNDS="1")
    proc = subprocess.run([sys.executable, "-c", SCRIPT.format(root=ROOT, tests=os.path.join(ROOT, "tests"))],
                          env=env, capture_output=True, text=True, timeout=900)
    assert proc.returncode == 0 and "checked build ok" in proc.stdout, proc.stdout[-2000:] + proc.stderr[-3000:]
