"""Tokens drawn on the GPU (tkm_hip_sample, tkm_runtime_sample) against the draw in 64 bits (sample_cases.py): they
have to be the same.  A weight is rounded to a multiple of 2^-45 or finer, so that a border is off by at most
vocab * 2^-46 of the largest weight: under 2^-29 for what is drawn here, where the nearest border of a random u is
further away than that in all but a few of 10^8 draws; such a draw would be named by the assertion."""
import numpy as np
import pytest
import torch

from sample_cases import draw_ref

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def run(gpu, x, u, dtype, **kw):
    from tokamak_amd import runtime
    x = x.to(DT[dtype])
    dev = {k: None if v is None else torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device=gpu) for k, v in kw.items()}
    got = runtime.sample(x.to(gpu), torch.tensor(u, dtype=torch.float32, device=gpu), **dev).tolist()
    for r in range(x.shape[0]):
        one = {k: float(np.float32(v[r])) if k != "top_k" else v[r] for k, v in kw.items() if v is not None}
        ref, near = draw_ref(x[r].double().numpy(), float(np.float32(u[r])), **one)
        assert got[r] == ref, (r, got[r], ref, near, one)


@pytest.mark.parametrize("V", [1, 2, 7, 100, 511, 512, 513, 1000, 8191, 8192, 8193, 32003])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("use", ["", "k", "p", "m", "kp", "kpm"])
def test_draws(gpu, V, dtype, use):
    rng = np.random.default_rng(V + len(use))
    n = 12 if V < 10000 else 4
    x = torch.from_numpy(rng.standard_normal((n, V)) * rng.choice([0.3, 3.0, 8.0], (n, 1)))
    run(gpu, x, rng.random(n).tolist(), dtype, temperature=(0.2 + 1.5 * rng.random(n)).tolist(),
        top_k=rng.integers(1, max(2, V // 2), n).tolist() if "k" in use else None,
        top_p=rng.random(n).tolist() if "p" in use else None, min_p=(0.2 * rng.random(n)).tolist() if "m" in use else None)


@pytest.mark.parametrize("dtype", DT)
def test_large_vocabularies(gpu, dtype):
    rng = np.random.default_rng(5)
    for V in (131072, 524288):
        x = torch.from_numpy(rng.standard_normal((2, V)) * 2)
        run(gpu, x, [0.37, 0.99], dtype, temperature=[1.0, 0.7], top_p=[0.9, 0.6], top_k=[V // 3, 0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("top_k", [1, 3, 40, 5000])
def test_ties(gpu, dtype, top_k):
    """Few distinct logits: borders inside runs of equal ones, and bins with more words than the list holds."""
    rng = np.random.default_rng(top_k)
    n, V = 8, 9001
    x = torch.from_numpy(rng.integers(-2, 3, (n, V)) * np.array([0.0, 0.0, 0.01, 0.5, 0.5, 1, 2, 3.0])[:, None])
    u = rng.random(n).tolist()
    run(gpu, x, u, dtype, top_k=[top_k] * n)
    run(gpu, x, u, dtype, top_p=rng.random(n).tolist(), temperature=[0.5] * n)
    run(gpu, x, u, dtype, top_k=[top_k] * n, top_p=rng.random(n).tolist(), min_p=[0.3] * n)


def test_many_words_in_one_bin(gpu):
    """fp32 logits that differ in their lowest bits alone: the border's bin does not fit the list."""
    rng = np.random.default_rng(0)
    x = torch.from_numpy(1.0 + rng.integers(0, 1 << 18, (4, 20000)) * 2.0 ** -23)
    u = rng.random(4).tolist()
    run(gpu, x, u, "f32", top_k=[1, 700, 15000, 19999])
    run(gpu, x, u, "f32", top_k=[0, 700, 15000, 0], top_p=[0.01, 0.5, 0.9, 0.99])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kw", [{}, dict(top_k=[50] * 8), dict(top_p=[0.9] * 8), dict(min_p=[0.01] * 8), dict(top_k=[9000] * 8, top_p=[0.99] * 8, min_p=[0.001] * 8)])
def test_first_words_unlike_the_rest(gpu, dtype, kw):
    """Rows whose first 8192 words say nothing of the largest: none at all, far lower, many above them, +inf or NaN
    behind; and far higher."""
    rng = np.random.default_rng(11)
    x = torch.from_numpy(rng.standard_normal((8, 20001)))
    x[0, :8192] = float("-inf")
    x[1, :8192] -= 30
    x[2, :8192] -= 3.5
    x[3, 12000:] += 4
    x[4, 19000] = float("inf")
    x[5, 8192:] = float("nan")
    x[6, :8192] += 50
    x[7, 20000] = 9.0
    run(gpu, x, rng.random(8).tolist(), dtype, **kw)
    run(gpu, x, rng.random(8).tolist(), dtype, temperature=[0.05, 2.0, 0.3, 0.3, 1.0, 0.1, 30.0, 0.7], **kw)


@pytest.mark.parametrize("dtype", DT)
def test_odd_logits(gpu, dtype):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(DT[dtype]).min
    V = 700
    g = torch.Generator().manual_seed(1)
    base = torch.randn(V, generator=g, dtype=torch.float64)
    rows = []
    for fill, at in ((-inf, range(0, V, 2)), (low, range(0, V, 3)), (nan, range(1, V, 2)), (inf, (5, 600)), (-inf, range(V)), (nan, range(V)),
                     (low, range(V)), (-inf, range(V - 1)), (-0.0, range(0, V, 2)), (0.0, range(0, V, 2))):
        r = base.clone()
        r[list(at)] = fill
        rows.append(r)
    rows[8][1::2] = 0.0
    x = torch.stack(rows)
    n = len(rows)
    u = [0.03 + 0.09 * i for i in range(n)]
    for kw in ({}, dict(top_k=[7] * n), dict(top_p=[0.8] * n), dict(min_p=[0.5] * n), dict(temperature=[0.0] * n),
               dict(top_k=[600] * n, top_p=[0.999] * n, temperature=[3.0] * n)):
        run(gpu, x, u, dtype, **kw)


def test_settings_at_their_ends(gpu):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(2)
    x = torch.randn(9, 3000, generator=g, dtype=torch.float64) * 3
    u = [0.0, 2.0 ** -30, 0.5, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, nan, 0.999]
    run(gpu, x, u, "f32")
    run(gpu, x, u, "f32", temperature=[0.0, -1.0, nan, inf, 1e-30, 1e30, 1e-40, 100.0, 0.01])
    run(gpu, x, u, "f32", top_k=[0, -5, 1, 2, 2999, 3000, 3001, 2 ** 31 - 1, -2 ** 31])
    run(gpu, x, u, "f32", top_p=[0.0, -1.0, 1.0, 2.0, 1 - 2.0 ** -24, 1e-30, inf, 0.5, 0.25])
    run(gpu, x, u, "f32", min_p=[0.0, -1.0, 1.0, 2.0, 1e-30, 0.5, inf, 0.999, 0.01])


def test_strided_rows_indices_and_what_lies_around(gpu):
    from tokamak_amd import runtime
    wide = torch.full((6, 1031), float("inf"), dtype=torch.bfloat16, device=gpu)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 1000, generator=g).to(torch.bfloat16)
    wide[:, 3:1003] = x.to(gpu)
    idx = [5, 5, 0, -1, 6, 2, 2147483647]
    u = [0.1, 0.9, 0.5, 0.5, 0.5, 0.3, 0.1]
    out = torch.full((9,), 77, dtype=torch.int32, device=gpu)
    runtime.sample(wide[:, 3:1003], torch.tensor(u, device=gpu), row_index=torch.tensor(idx, dtype=torch.int32, device=gpu), out=out[1:8])
    ref = [draw_ref(x[i].double().numpy(), float(np.float32(v)))[0] if 0 <= i < 6 else -1 for i, v in zip(idx, u)]
    assert out.tolist() == [77] + ref + [77]


def test_captured_and_replayed(gpu):
    from tokamak_amd import runtime
    x = torch.randn(5, 32003, device=gpu, dtype=torch.float16) * 3
    u, p = torch.rand(5, device=gpu), torch.full((5,), 0.9, device=gpu)
    out = torch.zeros(5, dtype=torch.int32, device=gpu)
    runtime.sample(x, u, top_p=p, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        runtime.sample(x, u, top_p=p, out=out)
    for i in range(4):
        x.normal_().mul_(3)
        u.uniform_()
        p.fill_(0.2 + 0.2 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.tolist()
        assert got == runtime.sample(x, u, top_p=p).tolist()
        assert got == [draw_ref(x[r].double().cpu().numpy(), float(u[r]), top_p=float(p[r]))[0] for r in range(5)]


def test_runtime_draws_what_its_logits_say(gpu):
    """Runtime.sample: forward, then draws on the device, against draws from forward's own logits."""
    import json
    import os
    from tokamak_amd import runtime as R
    fx = np.load(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "tkm_graphs.npz"))
    raw, js = bytearray(fx["llama_small/graph"].tobytes()), json.loads(bytes(fx["llama_small/json"]).decode())
    for n in js["nodes"]:
        if n["op"] == 59:                # the flow without its loss ends in the logits
            raw[264 * n["id"] + 48:264 * n["id"] + 52] = np.array([1], np.int32).tobytes()
    rt = R.Runtime(R.graph_buffer(bytes(raw)), training=False, token_labels=True)
    rng = np.random.default_rng(4)
    x = rng.standard_normal(rt.input_elements).astype(np.float32)
    logits = rt.forward(x)
    V = [n for n in js["nodes"] if n["op"] in (3, 4, 5)][-1]["C"]
    logits = logits.reshape(-1, V)
    rows = rng.integers(0, logits.shape[0], 9).astype(np.int32)
    rows[4] = -1
    u = rng.random(9).astype(np.float32)
    got = rt.sample(x, u, rows=rows, temperature=0.8, top_k=np.arange(9) * 3, top_p=0.9)
    want = [-1 if r < 0 else draw_ref(logits[r], float(v), float(np.float32(0.8)), 3 * i, float(np.float32(0.9)))[0] for i, (r, v) in enumerate(zip(rows, u))]
    assert got.tolist() == want
    assert rt.sample(x, [0.5, 0.5], temperature=0.0).tolist() == logits[:2].argmax(1).tolist()
    with pytest.raises(RuntimeError):
        rt.sample(x, np.zeros(logits.shape[0] + 1))
    with pytest.raises(ValueError):
        rt.sample(x[:-1], u)
    rt.close()
