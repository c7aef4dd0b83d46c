"""The cache in pages, its attention and the rules on logits as a server uses them: together, in a captured step, on streams and
threads of their own, one workspace for calls of many sizes."""

import threading

import numpy as np
import pytest
import torch

from oracle import pages as oracle
from serving_tools import check_attention
from test_gpu_logits_rules import check as check_rules
from test_gpu_paged_attention import Scene, _rest

pytestmark = pytest.mark.gpu


def _ext():
    from flash_whisper_amd.ext import load_ext

    return load_ext()


class Server:
    """Two prompts with 4 and 3 answers each. A token's key, value and query are rows of tables; its logits a product of the
    attention's output. The first answer of a prompt brings its rows into the cache, the others list its whole pages and copy
    the one that its rows end in."""

    def __init__(self, dev, page=16, heads=4, kv_heads=2, dim=64, vocab=300, prompts=(1200, 37), answers=(4, 3)):
        rng = np.random.default_rng(page)
        self.dev, self.page, self.heads, self.vocab, self.dim = dev, page, heads, vocab, dim
        self.ext, self.n = _ext(), sum(answers)
        half = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).half().to(dev)
        self.eq, self.ek, self.ev, self.w = half(vocab, heads, dim), half(vocab, kv_heads, dim), half(vocab, kv_heads, dim), half(heads * dim, vocab)
        self.width, pages = -(-(max(prompts) + 60) // page), 200
        self.cache = self.ext.kv_pages(pages, kv_heads, page, dim)
        i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=dev)
        self.table = torch.zeros(self.n, self.width, dtype=torch.int32, device=dev)
        self.stack, self.count = torch.randperm(pages, device=dev).int(), i64([pages, 0])
        self.held, self.own = i64([0] * self.n), i64([0] * self.n)
        self.cu_groups, self.shared = i64([0, *np.cumsum(answers)]), i64(prompts)
        first = [int(x) for x in np.r_[0, np.cumsum(answers)][:-1]]
        rows = [0] * self.n
        for f, p in zip(first, prompts):
            rows[f] = p
        self.text = [[] for _ in range(self.n)]
        tokens = [rng.integers(0, vocab, p) for p in prompts]
        packed = i64(np.concatenate(tokens))
        slots = torch.empty(sum(prompts), dtype=torch.int64, device=dev)
        pos = i64([0 if r else -1 for r in rows])
        self.ext.kv_page_map(pos, i64([0, *np.cumsum(rows)]), self.table, self.held, self.stack, self.count, slots, page)
        self.ext.kv_page_append(self.ek[packed], self.ev[packed], slots, self.cache)
        # the answers beside the first
        whole = [p // page for p in prompts]
        for g, f in enumerate(first):
            for s in range(f, f + answers[g]):
                self.text[s] = tokens[g].tolist()
                if s > f:
                    self.table[s, :whole[g]] = self.table[f, :whole[g]]
                    self.held[s] = self.own[s] = whole[g]
        self.pos = i64([p for p, a in zip(prompts, answers) for _ in range(a)])
        self.each = torch.arange(self.n + 1, device=dev)
        back = i64([w * page if s not in first else p for s, (w, p) in enumerate(zip(np.repeat(whole, answers), np.repeat(prompts, answers)))])
        cu = i64([0, *np.cumsum((self.pos - back).tolist())])
        slots = torch.empty(int(cu[-1]), dtype=torch.int64, device=dev)
        self.ext.kv_page_map(back, cu, self.table, self.held, self.stack, self.count, slots, page, self.own)
        for g, f in enumerate(first):
            for s in range(f + 1, f + answers[g]):
                if prompts[g] % page:
                    a, b = self.table[f, whole[g]].long(), self.table[s, whole[g]].long()
                    self.cache.k[b], self.cache.v[b] = self.cache.k[a], self.cache.v[a]
        assert self.count[1] == 0
        self.slots = torch.empty(self.n, dtype=torch.int64, device=dev)
        self.ws = self.ext.decode_attention_paged_workspace(self.n, heads, self.cache, self.width, 2)
        self.token = i64(rng.integers(0, vocab, self.n))
        self.history = torch.zeros(self.n, 80, dtype=torch.int64, device=dev)
        self.steps, self.out = i64([0]), torch.empty(self.n, heads, dim, dtype=torch.float16, device=dev)
        self.logits = torch.empty(self.n, vocab, dtype=torch.float16, device=dev)
        self.ruled = torch.empty_like(self.logits)
        self.rules = dict(cu=self.each * 80, prompt=torch.zeros(self.n, dtype=torch.int64, device=dev),
                          repetition=torch.linspace(1, 1.5, self.n, device=dev), presence=torch.linspace(0, 1, self.n, device=dev),
                          frequency=torch.linspace(0.2, 0, self.n, device=dev), bias_ids=i64([3, 5, 3]), bias=torch.tensor([1.0, -2, 0.5], device=dev),
                          cu_bias=i64([0] * self.n + [3]), masks=torch.randint(-2**31, 2**31, (2, 10), device=dev).int(),
                          mask_of=i64([-1, 0, 1, 0, 1, -1, 1]))

    def step(self):
        """One token of every answer, without the host."""
        self.ext.kv_page_map(self.pos, self.each, self.table, self.held, self.stack, self.count, self.slots, self.page, self.own)
        self.ext.kv_page_append(self.ek[self.token], self.ev[self.token], self.slots, self.cache)
        self.history.scatter_(1, self.steps.expand(self.n, 1), self.token[:, None])
        self.pos += 1
        self.ext.decode_attention_paged(self.eq[self.token], self.cache, self.table, self.pos, self.out, self.ws, self.dim ** -0.5,
                                        self.cu_groups, self.shared)
        torch.mm(self.out.view(self.n, -1), self.w, out=self.logits)
        self.ext.logits_rules(self.logits, self.ruled, tokens=self.history.view(-1), **self.rules)
        self.token.copy_(self.ruled.argmax(1))
        self.steps += 1

    def check(self, before):
        """The step that began with tokens `before`, against the texts so far."""
        ek, ev, eq = (x.double().cpu().numpy() for x in (self.ek, self.ev, self.eq))
        assert self.count[1] == 0 and (self.slots >= 0).all()
        for s in range(self.n):
            self.text[s].append(int(before[s]))
            k, v = ek[self.text[s]], ev[self.text[s]]
            want, spread, size = oracle.serving.attend(eq[int(before[s])][None], k, v, self.dim ** -0.5, False)
            check_attention(self.out[s].double().cpu().numpy()[None], want, spread, size, np.abs(v).max(), len(k), torch.float16)
        rules = {k: v.cpu().numpy() for k, v in {**self.rules, 'tokens': self.history.view(-1)}.items()}
        check_rules(self.ruled, self.logits, rules, torch.float16)
        assert torch.equal(self.token, self.ruled.argmax(1))


@pytest.mark.parametrize('page', [16, 32])
def test_steps(hip_device, page):
    server = Server(hip_device, page)
    for _ in range(40):  # across the ends of pages
        before = server.token.tolist()
        server.step()
        server.check(before)
    # an answer ends: what it owns comes back
    free, held, own = int(server.count[0]), server.held.tolist(), server.own.tolist()
    pos = server.pos.clone()
    pos[1] = 0
    none = torch.zeros(server.n + 1, dtype=torch.int64, device=hip_device)
    _ext().kv_page_map(pos, none, server.table, server.held, server.stack, server.count, server.slots[:0], page, server.own)
    assert server.held.tolist() == [held[0], 0, *held[2:]] and int(server.count[0]) == free + held[1] - own[1]


def test_captured_step(hip_device):
    """A step in a graph, replayed with eager work between; every replay against the oracle."""
    server = Server(hip_device)
    eager = server.token.tolist()
    server.step()  # loads what a first call loads
    server.check(eager)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    state = [server.pos, server.held, server.count, server.token, server.history, server.steps, server.table, server.stack]
    kept = [t.clone() for t in state]
    with torch.cuda.graph(graph, stream=side):
        server.step()
    for t, k in zip(state, kept):
        t.copy_(k)
    for i in range(25):
        before = server.token.tolist()
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
            torch.randn(1000, 1000, device=hip_device).sum().item()
        server.check(before)


def test_two_graphs_share_a_workspace(hip_device):
    """Two captured calls of different sizes with one workspace, replayed in turn on one stream."""
    scenes = [Scene(31, [5], [1500], _rest(1, 5, 0, 90), 32, 2, 3, 64, 'fp16'), Scene(32, [1, 3, 20], [0, 1300, 1111], _rest(2, 24, 0, 1200), 32, 4, 2, 64, 'fp16')]
    from flash_whisper_amd.ext import KvPages

    ext, graphs, outs, ws, keep = _ext(), [], [], None, []
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    for s in reversed(scenes):
        cache, q = KvPages(s.k.to(hip_device), s.v.to(hip_device)), s.q.to(hip_device)
        args = torch.from_numpy(s.table).to(hip_device), i64(s.lens)
        groups, out = (i64(s.cu), i64(s.shared)), torch.zeros_like(q)
        need = ext.decode_attention_paged_workspace(len(s.lens), s.heads, cache, s.table.shape[1], len(s.shared))
        ws = need if ws is None or need.numel() > ws.numel() else ws
        keep.append((cache, q, args, groups, out))
    for cache, q, args, groups, out in keep:
        call = lambda: ext.decode_attention_paged(q, cache, *args, out, ws, 0.125, *groups)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
        outs.append(out)
    for _ in range(4):
        for graph, out, scene in zip(graphs, outs, reversed(scenes)):
            out.fill_(9)
            graph.replay()
            scene.check(out, scale=0.125)
        ws.fill_(float('nan'))  # what a call leaves there means nothing to the next


def test_streams(hip_device):
    """Calls on another stream than the tensors' own, behind the work that makes their inputs."""
    scene = Scene(33, [4, 4], [1200, 90], _rest(3, 8, 0, 500), 16, 2, 2, 128, 'bf16')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(4096, 4096, device=hip_device)
        for _ in range(20):
            x = torch.tanh(x @ x * 1e-3)
        out = scene.run(hip_device)
    torch.cuda.current_stream().wait_stream(side)
    scene.check(out)


def test_two_threads(hip_device):
    """Two threads with a stream, tensors and a workspace each."""
    scenes = [Scene(34 + i, [6], [1300], _rest(i, 6, 0, 300), 32, 2, 2, 64, 'fp16') for i in range(2)]
    outs, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    outs[i] = scenes[i].run(hip_device)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for scene, out in zip(scenes, outs):
        scene.check(out)


def test_without_the_binding(hip_device):
    """The same calls through ctypes."""
    from flash_whisper_amd import ext as module

    ext = _ext()
    bind, ext._bind = ext._bind, None
    try:
        server = Server(hip_device)
        for _ in range(3):
            before = server.token.tolist()
            server.step()
            server.check(before)
        assert module.load_ext() is ext
    finally:
        ext._bind = bind


def test_refused_on_the_gpu(hip_device):
    """What a valid call turns into when an argument does not fit: named errors, nothing launched."""
    ext = _ext()
    cache = ext.kv_pages(8, 2, 16, 64)
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    q, table = torch.zeros(2, 4, 64, dtype=torch.float16, device=hip_device), torch.zeros(2, 4, dtype=torch.int32, device=hip_device)
    ws, lens = ext.decode_attention_paged_workspace(2, 4, cache, 4, 1), i64(3, 5)
    good = dict(q=q, cache=cache, table=table, lens=lens, out=q.clone(), ws=ws, scale=0.125, cu_groups=i64(0, 2), shared=i64(3))
    ext.decode_attention_paged(**good)
    for name, bad in (('q', q.bfloat16()), ('q', q[:, :, :32]), ('q', q[:1]), ('q', q[:, :3]), ('q', q.transpose(1, 2)), ('table', table.long()),
                      ('table', table[:, ::2]), ('table', table[:1]), ('lens', lens.int()), ('lens', lens[:1]), ('out', q[:, :2]),
                      ('out', q[:1].expand(2, 4, 64)), ('ws', ws[:0]), ('ws', ws.half()), ('ws', None), ('cu_groups', None), ('cu_groups', i64(0)),
                      ('shared', None), ('shared', i64(3, 3)), ('scale', float('inf')), ('cache', (cache.k, cache.v.bfloat16())),
                      ('cache', (cache.k[:4], cache.v)), ('cache', (cache.k.transpose(0, 1), cache.v)), ('lens', lens.cpu())):
        with pytest.raises(RuntimeError):
            ext.decode_attention_paged(**{**good, name: bad})
    k = torch.zeros(5, 2, 64, dtype=torch.float16, device=hip_device)
    slots = i64(0, 1, 2, 3, -1)
    ext.kv_page_append(k, k, slots, cache)
    for bad in (dict(k=k.bfloat16()), dict(v=k[:4]), dict(k=k[:, :1]), dict(slots=slots[:4]), dict(slots=slots.int()), dict(cache=(cache.k, cache.v, cache.v))):
        with pytest.raises(RuntimeError):
            ext.kv_page_append(**{**dict(k=k, v=k, slots=slots, cache=cache), **bad})
    good = dict(pos=i64(0, 0), cu=i64(0, 1, 2), table=table, held=i64(0, 0), stack=table[0], count=i64(4, 0), slots=i64(0, 0), page=16)
    ext.kv_page_map(**good)
    for bad in (dict(pos=i64(0)), dict(cu=i64(0, 1)), dict(table=table.long()), dict(table=table[:, :2]), dict(held=i64(0)), dict(stack=i64(1)),
                dict(count=i64(4)), dict(slots=table[0]), dict(page=20), dict(page='x'), dict(own=i64(0)), dict(held_out=i64(0)), dict(count_out=i64(0, 0, 0))):
        with pytest.raises((RuntimeError, ValueError)):
            ext.kv_page_map(**{**good, **bad})
    x = torch.zeros(3, 100, dtype=torch.float16, device=hip_device)
    rep = torch.ones(3, device=hip_device)
    good = dict(logits=x, out=x, tokens=i64(1, 2, 3), cu=i64(0, 1, 2, 3), repetition=rep, bias_ids=i64(1), bias=rep[:1], cu_bias=i64(0, 0, 0, 1),
                masks=torch.zeros(3, 4, dtype=torch.int32, device=hip_device), mask_of=i64(0, 1, 2))
    ext.logits_rules(**good)
    for bad in (dict(out=x[:2]), dict(out=x.float()), dict(out=x[:1].expand(3, 100)), dict(logits=x.t()), dict(logits=x.long()), dict(tokens=None), dict(cu=None),
                dict(cu=i64(0, 1)), dict(tokens=i64(1, 2).int()), dict(repetition=rep[:2]), dict(repetition=rep.half()), dict(bias=None), dict(bias=rep),
                dict(cu_bias=i64(0)), dict(masks=good['masks'][:, :3].contiguous()), dict(masks=good['masks'].long()), dict(mask_of=i64(0)),
                dict(masks=None), dict(masks=good['masks'][:2], mask_of=None)):
        with pytest.raises(RuntimeError):
            ext.logits_rules(**{**good, **bad})
