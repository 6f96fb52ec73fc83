"""A decoder layer run through the package's entry points from norm to norm:
rms_norm_act -> q/k/v from its planes -> KvCache.write -> KvCache.attend -> o ->
rms_norm_act with the residual -> gate/up + GLU from its planes -> down. Each
step is held to its own definition on the inputs it was given; a captured
decode step replays with the eager step's bits, graphs and streams beside each
other do not disturb each other."""
import os
import subprocess
import sys

import pytest
import torch

from layer_reference import attend64, cache_values, rounding
from swarmllm_amd import GgmlDType, KvCache, QMatMul, QTensor, fill_normal, forward_glu, rms_norm_act

pytestmark = pytest.mark.gpu

HIDDEN, FFN, HEADS, KV, HD, PAGE, EPS = 512, 1024, 8, 2, 64, 16, 1e-5


class Layer:
    def __init__(self, dtype, seed=1):
        def w(n, k, s):
            return QMatMul(QTensor.quantize(fill_normal(n * k, seed=seed + s, std=0.05).reshape(n, k), dtype))
        self.dtype = dtype
        self.q, self.k, self.v = w(HEADS * HD, HIDDEN, 1), w(KV * HD, HIDDEN, 2), w(KV * HD, HIDDEN, 3)
        self.o, self.gate, self.up, self.down = (w(HIDDEN, HEADS * HD, 4), w(FFN, HIDDEN, 5), w(FFN, HIDDEN, 6),
                                                 w(HIDDEN, FFN, 7))
        self.n1, self.n2 = (1.0 + 0.1 * fill_normal(HIDDEN, seed=seed + 8 + i) for i in range(2))

    def __call__(self, x, kv, slots, q_starts, kv_lens, tables, max_q, seen=None):
        """The stream after the layer, and every step's results."""
        n1 = rms_norm_act(x, self.n1, EPS, dtype=self.dtype, y_dtype=torch.float32)
        q, k, v = QMatMul.forward_shared(n1.act, [self.q, self.k, self.v])
        kv.write(k.unflatten(1, (KV, HD)), v.unflatten(1, (KV, HD)), slots)
        a = kv.attend(q.unflatten(1, (HEADS, HD)), q_starts, kv_lens, tables, max_q=max_q)
        o = self.o.forward(a.flatten(1))
        n2 = rms_norm_act(o, self.n2, EPS, residual=n1.h, dtype=self.dtype, y_dtype=torch.float32)
        g = forward_glu(n2.act, self.gate, self.up)
        d = self.down.forward(g)
        if seen is not None:
            seen.update(n1=n1, q=q, k=k, v=v, a=a, o=o, n2=n2, g=g, d=d)
        return n2.h + d


def batch(lens, new, seed):
    """Page tables, and the bounds and slots of sequences of lens[b] positions, the last new[b] of them new."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    per = 8
    tables = torch.randperm(len(lens) * per, generator=g, device="cuda").view(len(lens), per).int()
    starts = torch.tensor([sum(new[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv = KvCache.alloc(len(lens) * per, KV, HD, PAGE)
    slots = torch.cat([kv.slots(tables[b], lens[b] - new[b], new[b]) for b in range(len(lens))])
    return kv, tables, starts, kv_lens, slots


@pytest.mark.parametrize("dtype", [GgmlDType.Q4K, GgmlDType.Q8_0, GgmlDType.Q6K])
def test_layer_steps_hold_their_definitions(dtype):
    layer = Layer(dtype)
    new = [37, 1, 60]
    kv, tables, starts, lens, slots = batch([37, 1, 60], new, 3)
    for step in range(3):  # a ragged prompt, then single tokens
        if step:
            new = [1, 1, 1]
            starts = torch.arange(4, dtype=torch.int32, device="cuda")
            slots = torch.stack([kv.slots(tables[b], int(lens[b]), 1)[0] for b in range(3)])
            lens = lens + 1
        x = fill_normal(sum(new) * HIDDEN, seed=20 + step).reshape(-1, HIDDEN)
        r = {}
        out = layer(x, kv, slots, starts, lens, tables, max(new), r)
        for n, w, h in ((r["n1"], layer.n1, x), (r["n2"], layer.n2, x + r["o"])):
            assert torch.equal(n.h, h)
            y = n.h.double() / (n.h.double().square().mean(1, keepdim=True) + EPS).sqrt() * w.double()
            assert (n.y.double() - y).abs().le(3.001 * 2.0**-24 * y.abs()).all()
        # products of the planes: the bits of the products of the normed values
        for got, w in ((r["q"], layer.q), (r["k"], layer.k), (r["v"], layer.v)):
            assert torch.equal(got, QMatMul.forward_shared(r["n1"].y, [layer.q, layer.k, layer.v])
                               [[layer.q, layer.k, layer.v].index(w)])
        assert torch.equal(r["g"], forward_glu(r["n2"].y, layer.gate, layer.up))
        # the cache holds k and v to half a code (1 / 254 of a block's largest) and the scale's f16 rounding
        for got, val in zip((c[slots] for c in cache_values(kv)), (r["k"], r["v"])):
            val = val.double().unflatten(1, (KV, HD // 32, 32))
            top = val.abs().amax(-1, keepdim=True)
            assert ((got.unflatten(2, (HD // 32, 32)) - val).abs() <= top * (0.5 / 127 * (1 + 2.0**-10) + 2.0**-11) + 2.0**-18).all()
        want, tol = attend64(kv, r["q"].unflatten(1, (HEADS, HD)), starts, lens, tables, HD ** -0.5)
        err = (r["a"].double() - want).abs()
        assert (err <= tol + rounding(r["a"].dtype) * (want.abs() + tol)).all()
        assert torch.equal(out, r["n2"].h + layer.down.forward(r["g"]))


def decode_state(n, seed):
    lens = [30 + 9 * b for b in range(n)]
    kv, tables, starts, kv_lens, slots = batch(lens, [1] * n, seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for i in (0, 2):
        kv.planes[i].copy_(torch.randint(-127, 128, kv.planes[i].shape, generator=g, device="cuda", dtype=torch.int8))
        kv.planes[i + 1].fill_(0.02)
    return kv, tables, starts, kv_lens, slots


def copy_of(kv):
    return KvCache(*(t.clone() for t in kv.planes))


def capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn()
    return g, out


@pytest.mark.parametrize("n", [1, 3])
def test_captured_decode_steps_replay_the_eager_bits(n):
    layer = Layer(GgmlDType.Q4K)
    kv, tables, starts, lens, slots = decode_state(n, 5)
    eager = copy_of(kv)
    x = fill_normal(n * HIDDEN, seed=40).reshape(n, HIDDEN)
    start = [t.clone() for t in kv.planes]
    g, out = capture(lambda: layer(x, kv, slots, starts, lens, tables, 1))
    for t, s in zip(kv.planes, start):
        t.copy_(s)
    for step in range(4):
        x.copy_(fill_normal(n * HIDDEN, seed=50 + step).reshape(n, HIDDEN))
        if step:
            slots.copy_(torch.stack([kv.slots(tables[b], int(lens[b]), 1)[0] for b in range(n)]))
            lens.add_(1)
        out.fill_(float("nan"))
        g.replay()
        want = layer(x.clone(), eager, slots, starts, lens, tables, 1)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(kv.planes, eager.planes):
            assert torch.equal(a, b)


def long_state(new, n, seed, heads=8):
    kv = KvCache.alloc(n // 64 + 2, 1, 128, 64)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for i in (0, 2):
        kv.planes[i].copy_(torch.randint(-127, 128, kv.planes[i].shape, generator=g, device="cuda", dtype=torch.int8))
        kv.planes[i + 1].fill_(0.01)
    q = torch.randn(new, heads, 128, generator=g, device="cuda").half()
    table = torch.arange(kv.pages, device="cuda", dtype=torch.int32).view(1, -1)
    return kv, q, torch.tensor([0, new], dtype=torch.int32, device="cuda"), \
        torch.tensor([n], dtype=torch.int32, device="cuda"), table


def test_captured_graphs_share_no_workspace():
    """Two graphs whose contexts are cut into parts (a workspace each), replayed beside each other on two streams."""
    calls, wants, graphs = [], [], []
    for new, n, seed in ((1, 20000, 1), (70, 9000, 2)):
        kv, q, s, l, t = long_state(new, n, seed)
        calls.append((kv, q, s, l, t, new))
        wants.append(kv.attend(q, s, l, t, max_q=new))
        graphs.append(capture(lambda kv=kv, q=q, s=s, l=l, t=t, new=new: kv.attend(q, s, l, t, max_q=new)))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for _, out in graphs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        for kv, q, s, l, t, new in calls:
            kv.attend(q, s, l, t, max_q=new)
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, wants):
            assert torch.equal(out, want)


def test_calls_on_two_streams_at_once():
    states = [long_state(new, n, seed) + (new,) for new, n, seed in ((1, 20000, 3), (2, 15000, 4), (50, 6000, 5))]
    wants = [kv.attend(q, s, l, t, max_q=new) for kv, q, s, l, t, new in states]
    x = [fill_normal(64 * 4096, seed=i).reshape(64, 4096) for i in range(3)]
    w = torch.ones(4096, device="cuda")
    acts = [rms_norm_act(v, w, EPS).act.dequantize() for v in x]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, (kv, q, s, l, t, new), v in zip(streams, states, x):
            with torch.cuda.stream(st):
                got.append((kv.attend(q, s, l, t, max_q=new), rms_norm_act(v, w, EPS).act.dequantize()))
        torch.cuda.synchronize()
        for (a, b), want, act in zip(got, wants, acts):
            assert torch.equal(a, want) and torch.equal(b, act)


def test_results_do_not_change_from_call_to_call_nor_with_the_batch():
    """No order of any sum depends on timing; a sequence's rows are the same in any batch that plans the same launch."""
    kv, q, s, l, t = long_state(3, 8000, 6)
    first = kv.attend(q, s, l, t, max_q=3)
    for _ in range(5):
        assert torch.equal(kv.attend(q, s, l, t, max_q=3), first)


FIRST_CALLS_CAPTURED = """
import torch
from swarmllm_amd import GgmlDType, KvCache, rms_norm_act
g = torch.Generator(device="cuda")
g.manual_seed(5)
x = torch.randn(600, 8 * 128, generator=g, device="cuda")
w = torch.ones(8 * 128, device="cuda")
kv = KvCache.alloc(60, 2, 128, 64)
tables = torch.randperm(60, generator=g, device="cuda").view(1, 60).int()
slots = kv.slots(tables[0], 3000, 600)
past = torch.randn(3000, 2, 128, generator=g, device="cuda")
starts = torch.tensor([0, 600], device="cuda", dtype=torch.int32)
lens = torch.tensor([3600], device="cuda", dtype=torch.int32)
old = kv.slots(tables[0], 0, 3000)

def step():
    n = rms_norm_act(x, w, 1e-5, dtype=GgmlDType.Q4K, y_dtype=torch.float16)
    q = n.act.dequantize_f16().view(600, 8, 128)
    kv.write(past, past, old)
    kv.write(q[:, :2], q[:, 2:4], slots)
    k, v = kv.read(slots)
    return n.y, q, k, v, kv.attend(q, starts, lens, tables, max_q=600), kv.attend(q[599:], starts // 600, lens, tables, max_q=1)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    first = step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in first]
for a, b in zip(got, step()):
    assert a.dtype == b.dtype and a.isfinite().all() and torch.equal(a, b)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, first))
print("captured first calls equal eager ones")
"""


def test_first_calls_of_a_process_under_capture():
    """Each entry point's first call of a process may be a captured one (no
    qmm_prepare before it): what a first launch sets up, more than 64 KiB of
    LDS for 256 query rows a workgroup among it, is allowed under capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root + (os.pathsep + os.environ["PYTHONPATH"] if os.environ.get("PYTHONPATH") else ""))
    res = subprocess.run([sys.executable, "-u", "-c", FIRST_CALLS_CAPTURED], env=env, cwd=root, capture_output=True,
                         text=True, timeout=100)
    assert res.returncode == 0 and "captured first calls equal" in res.stdout, res.stdout[-2000:] + res.stderr[-2000:]
