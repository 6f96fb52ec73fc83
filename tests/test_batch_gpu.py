"""The batch's steps run together, as a serving loop does: page tables, embedding rows, norm, products with each request's
adapter beside them, cache, attention and sampling, for prompts and decode steps, eager and captured."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, HIDDEN, HEADS, KV, HD, FFN, LAYERS, PAGE, RANK, SLOTS = 1000, 256, 4, 2, 64, 512, 2, 16, 8, 3


class Tiny:
    """A small decoder of Q8_0 weights with adapters at q, k, v and o."""

    def __init__(self, seed=1):
        from swarmllm_amd import Adapters, GgmlDType, QMatMul, QTensor, fill_normal

        seeds, g = iter(range(1000 * seed, 1000 * seed + 1000)), torch.Generator(device=DEV).manual_seed(seed)

        def weight(n, k, std=0.05):
            return QTensor.quantize(fill_normal(n * k, seed=next(seeds), std=std).view(n, k), GgmlDType.Q8_0)

        def adapters(n, k):
            a = fill_normal(SLOTS * RANK * k, seed=next(seeds), std=k ** -0.5).view(SLOTS, RANK, k)
            b = fill_normal(SLOTS * n * RANK, seed=next(seeds), std=0.3).view(SLOTS, n, RANK)
            return Adapters(a.bfloat16(), b.bfloat16(), torch.rand(SLOTS, generator=g, device=DEV) + 0.5)

        self.embed, self.head = weight(VOCAB, HIDDEN, 1.0), QMatMul(weight(VOCAB, HIDDEN, 0.3))
        self.layers = []
        for _ in range(LAYERS):
            sizes = [(HEADS * HD, HIDDEN), (KV * HD, HIDDEN), (KV * HD, HIDDEN), (HIDDEN, HEADS * HD)]
            self.layers.append(([QMatMul(weight(*s)) for s in sizes], [adapters(*s) for s in sizes],
                                [QMatMul(weight(FFN, HIDDEN)) for _ in range(2)] + [QMatMul(weight(HIDDEN, FFN))],
                                [torch.ones(HIDDEN, device=DEV) for _ in range(2)]))
        self.norm = torch.ones(HIDDEN, device=DEV)

    def forward(self, ids, rows, pages, caches, which, max_q):
        from swarmllm_amd import Adapters, GgmlDType, QMatMul, forward_glu, rms_norm_act

        n = ids.numel()
        x, r = self.embed.gather_rows(ids.view(torch.uint32), check_ids=False).dequantize(), None
        for (qkvo, ads, mlp, norms), kv in zip(self.layers, caches):
            a = rms_norm_act(x, norms[0], 1e-5, residual=r, dtype=GgmlDType.Q8_0, y_dtype=torch.float32)
            q, k, v = QMatMul.forward_shared(a.act, qkvo[:3])
            Adapters.add_shared([q, k, v], a.y, ads[:3], which)
            kv.write(k.view(n, KV, HD), v.view(n, KV, HD), rows.slots)
            o = torch.zeros(n, HEADS, HD, device=DEV)  # rows of no sequence: zeros
            kv.attend(q.view(n, HEADS, HD), rows.q_starts, pages.lens, pages.tables, max_q=max_q, out=o)
            o = o.view(n, HEADS * HD)
            y = ads[3].add(qkvo[3].forward(o), o, which)
            m = rms_norm_act(y, norms[1], 1e-5, residual=a.h, dtype=GgmlDType.Q8_0)
            x, r = mlp[2].forward(forward_glu(m.act, mlp[0], mlp[1])), m.h
        last = rms_norm_act(x, self.norm, 1e-5, residual=r, dtype=GgmlDType.Q8_0)
        return self.head.forward(last.act)


class Loop:
    """Requests in the places of a batch: prompts taken in, then a token a step, everything on the device."""

    def __init__(self, model, places, adapter, temperature, top_k, top_p):
        from swarmllm_amd import KvCache, PageTables

        self.model, self.places = model, places
        self.pages = PageTables.alloc(places, 6, 6 * places, page=PAGE)
        self.caches = [KvCache.alloc(6 * places, KV, HD, page=PAGE) for _ in range(LAYERS)]
        self.adapter, self.settings = adapter, (temperature, top_k, top_p)
        self.new = torch.zeros(places, dtype=torch.int32, device=DEV)
        self.keep = torch.full((places,), -1, dtype=torch.int32, device=DEV)
        self.token = torch.zeros(places, dtype=torch.int32, device=DEV)
        self.u = torch.zeros(places, device=DEV)

    def step(self, ids, max_q):
        """One pass over `ids`, one a row (None: each request's last token), and the next tokens."""
        from swarmllm_amd import sample

        n = self.places if ids is None else ids.numel()
        rows = self.pages.step(self.new, n, keep=self.keep)
        of = rows.seq.clamp(min=0).long()
        if ids is None:
            ids = self.token[of]
        which = torch.where(rows.seq >= 0, self.adapter[of], -1)
        logits = self.model.forward(ids, rows, self.pages, self.caches, which, max_q)
        end = (rows.q_starts[1:] - 1).clamp(min=0).long()
        out = sample(logits[end], self.u, *self.settings)
        self.token.copy_(torch.where(rows.taken > 0, out.ids, self.token))
        return out, rows


def requests():
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(VOCAB, (n,), generator=g).to(torch.int32).to(DEV) for n in (5, 1, 30, 12)]
    adapter = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device=DEV)
    temperature = torch.tensor([0.0, 0.8, 1.3, 1.0], device=DEV)
    top_k = torch.tensor([0, 40, 0, 5], dtype=torch.int32, device=DEV)
    top_p = torch.tensor([1.0, 0.9, 0.95, 1.0], device=DEV)
    u = torch.rand(12, 4, generator=g).to(DEV)
    return prompts, adapter, temperature, top_k, top_p, u


def tokens_of(loop, prompts, u, steps, capture=False, like=None):
    """The tokens of each step [steps + 1, places]. The prompts' batch is padded to the rows of the prompts `like`:
    products and attention choose their kernels, and so a row's last bits, by a batch's rows."""
    like = prompts if like is None else like
    ids = torch.cat(prompts)
    ids = torch.nn.functional.pad(ids, (0, sum(len(p) for p in like) - ids.numel()))
    loop.new.copy_(torch.tensor([len(p) for p in prompts]))
    loop.u.copy_(u[0])
    loop.step(ids, max(len(p) for p in like))
    out = [loop.token.clone()]
    loop.new.fill_(1)
    graph = None
    if capture:
        state = [t.clone() for t in (loop.pages.tables, loop.pages.lens, loop.pages.free, loop.pages.free_count, loop.token)]
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            loop.step(None, 1)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            loop.step(None, 1)
        for t, s in zip((loop.pages.tables, loop.pages.lens, loop.pages.free, loop.pages.free_count, loop.token), state):
            t.copy_(s)
    for i in range(steps):
        loop.u.copy_(u[1 + i])
        if graph is not None:
            graph.replay()
        else:
            loop.step(None, 1)
        out.append(loop.token.clone())
    return torch.stack(out)


def test_requests_together_as_alone_and_captured():
    model = Tiny()
    prompts, adapter, temperature, top_k, top_p, u = requests()
    together = tokens_of(Loop(model, 4, adapter, temperature, top_k, top_p), prompts, u, 10)
    assert ((together >= 0) & (together < VOCAB)).all() and len(set(together[:, 1].tolist())) > 3
    captured = tokens_of(Loop(model, 4, adapter, temperature, top_k, top_p), prompts, u, 10, capture=True)
    assert torch.equal(captured, together)
    for b in range(4):
        s = slice(b, b + 1)
        alone = tokens_of(Loop(model, 1, adapter[s], temperature[s], top_k[s], top_p[s]), [prompts[b]], u[:, s].contiguous(), 10,
                          like=prompts)
        assert torch.equal(alone[:, 0], together[:, b]), b


def test_another_adapter_changes_its_own_request_only():
    model = Tiny()
    prompts, adapter, temperature, top_k, top_p, u = requests()
    base = tokens_of(Loop(model, 4, adapter, temperature, top_k, top_p), prompts, u, 6)
    other = adapter.clone()
    other[1] = 0
    changed = tokens_of(Loop(model, 4, other, temperature, top_k, top_p), prompts, u, 6)
    same = [0, 2, 3]
    assert torch.equal(changed[:, same], base[:, same]) and not torch.equal(changed[:, 1], base[:, 1])


def test_a_finished_request_s_pages_serve_the_next_one():
    model = Tiny()
    prompts, adapter, temperature, top_k, top_p, u = requests()
    loop = Loop(model, 4, adapter, temperature, top_k, top_p)
    first = tokens_of(loop, prompts, u, 4)
    # request 2 ends and its place takes request 0's prompt, in one step with the others' next tokens
    loop.keep[2] = 0
    loop.new.copy_(torch.tensor([1, 1, 5, 1]))
    loop.u.copy_(u[0])
    loop.adapter[2], loop.settings[0][2], loop.settings[1][2], loop.settings[2][2] = 0, 0.0, 0, 1.0
    loop.step(torch.cat([loop.token[:2], prompts[0], loop.token[3:]]), 5)
    assert int(loop.token[2]) == int(first[0, 0]) and loop.pages.lens[2] == 5
    loop.keep.fill_(-1)
    loop.new.fill_(1)
    for i in range(4):
        loop.step(None, 1)
        assert int(loop.token[2]) == int(first[1 + i, 0])
    # all end: every page is free again
    loop.pages.step(keep=torch.zeros(4, dtype=torch.int32, device=DEV))
    assert int(loop.pages.free_count) == 24 and sorted(loop.pages.free.tolist()) == list(range(24))


def test_a_batch_without_pages_left_stands_still():
    from swarmllm_amd import PageTables

    pages = PageTables.alloc(3, 4, 3, page=PAGE)
    new = torch.tensor([16, 30, 4], dtype=torch.int32, device=DEV)
    rows = pages.step(new, 50)
    assert rows.taken.tolist() == [16, 30, 0] and (rows.slots[46:] == -1).all()
    # the second fills its pages, then stands still; the third waits
    for taken in (2, 0, 0):
        rows = pages.step(torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV), 6)
        assert rows.taken.tolist() == [0, taken, 0] and pages.lens.tolist() == [16, 32, 0]
    rows = pages.step(torch.tensor([0, 0, 4], dtype=torch.int32, device=DEV), 4,
                      keep=torch.tensor([-1, 10, -1], dtype=torch.int32, device=DEV))
    assert rows.taken.tolist() == [0, 0, 4] and pages.lens.tolist() == [16, 10, 4]


FIRST_UNDER_CAPTURE = """
import sys
sys.path[:0] = ["."]
import torch
from swarmllm_amd import Adapters, PageTables, sample

g = torch.Generator(device="cuda").manual_seed(1)
ad = [Adapters((torch.randn(3, r, k, generator=g, device="cuda") / 64).bfloat16(),
               torch.randn(3, 100, r, generator=g, device="cuda").bfloat16()) for r, k in ((16, 512), (64, 2048))]
xs = [torch.randn(rows, a.k, generator=g, device="cuda") for a, rows in ((ad[0], 9), (ad[1], 30), (ad[1], 1200))]
ids = [(torch.arange(len(x), device="cuda") % 4 - 1).to(torch.int32) for x in xs]
logits, u = 3 * torch.randn(20, 40000, generator=g, device="cuda"), torch.rand(20, generator=g, device="cuda")
k = torch.tensor([0, 0, 50, 3000] * 5, dtype=torch.int32, device="cuda")
p = torch.tensor([0.9, 1.0, 0.8, 1.0, 1.0] * 4, device="cuda")
new = torch.ones(4096, dtype=torch.int32, device="cuda")
new[::2] = 3
pages = [PageTables.alloc(n, 8, 20000, page=16) for n in (5, 4096)]


def steps():
    outs = [s for n, t in ((5, 20), (4096, 9000)) for s in pages[n > 5].step(new[:n], t)]
    outs += [a.add(torch.zeros(len(x), 100, device="cuda"), x, i) for a, x, i in zip((ad[0], ad[1], ad[1]), xs, ids)]
    return outs + [*sample(logits, u), *sample(logits, u, top_k=k, top_p=p)]


torch.cuda.synchronize()
state = [[t.clone() for t in (q.tables, q.lens, q.free, q.free_count)] for q in pages]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = steps()
for turn in range(4):
    graph.replay()
    got = [o.clone() for o in outs] + [t.clone() for q in pages for t in (q.tables, q.lens, q.free_count)]
    after = [[t.clone() for t in (q.tables, q.lens, q.free, q.free_count)] for q in pages]
    for q, s in zip(pages, state):
        for t, v in zip((q.tables, q.lens, q.free, q.free_count), s):
            t.copy_(v)
    want = steps() + [t.clone() for q in pages for t in (q.tables, q.lens, q.free_count)]
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), turn
    for q, s in zip(pages, after):
        for t, v in zip((q.tables, q.lens, q.free, q.free_count), s):
            t.copy_(v)
    state = after
    xs[0].mul_(0.5), xs[2].mul_(-0.5), logits.mul_(0.9)
torch.cuda.synchronize()
print("equal")
"""


def test_first_calls_of_a_process_under_capture():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_UNDER_CAPTURE], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("equal"), r.stdout[-500:] + r.stderr[-2000:]
