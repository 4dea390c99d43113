"""The serving operators as a program uses them: a small LLaMA (llama.py's weights and architecture) that reads two
prompts in chunks into a paged cache and goes on token by token, kv_append -> paged_attention in every layer
and sample at the end, against the stock model's full forward over the same tokens."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from autokernel_amd import kernels, llama

pytestmark = pytest.mark.gpu
append, attend, sample = (kernels.get(n) for n in ("kv_append", "paged_attention", "sample"))


def _model(dev, dtype):
    with torch.device(dev):
        m = llama.LlamaModel(vocab_size=1000, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, hidden_dim=512, max_seq_len=128)
    return llama.init_weights(m.to(dtype), std=0.08, seed=3).eval()


class Server:
    def __init__(self, model, pages, page):
        a = model.layers[0].attention
        self.m, self.page = model, page
        shape = (len(model.layers), pages, a.n_kv_heads, page, a.head_dim)
        w = model.output.weight
        self.k, self.v = (torch.full(shape, float("nan"), dtype=w.dtype, device=w.device) for _ in range(2))

    @torch.no_grad()
    def step(self, ids, table, starts, lens):
        """Logits of every row of one step."""
        m, T = self.m, ids.shape[0]
        h = m.tok_embeddings(ids)
        for i, layer in enumerate(m.layers):
            a = layer.attention
            x = layer.attention_norm(h)
            q, k, v = (lin(x).view(T, -1, a.head_dim) for lin in (a.wq, a.wk, a.wv))
            q = append(k, v, self.k[i], self.v[i], table, starts, lens, m.rope_cos.float(), m.rope_sin.float(), q=q)
            h = h + a.wo(attend(q, self.k[i], self.v[i], table, starts, lens).view(T, -1))
            h = h + layer.feed_forward(layer.ffn_norm(h))
        return m.output(m.norm(h))


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_llama_served_from_a_paged_cache(gpu, dtype):
    m = _model(gpu, dtype)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).to(gpu) for n in (37, 90)]
    server = Server(m, pages=20, page=16)
    table = torch.randperm(20, generator=g)[:16].to(torch.int32).view(2, 8).to(gpu)
    seqs = [p.clone() for p in prompts]
    at, served = [0, 0], [[], []]
    # prompts in uneven chunks (one sequence waits while the other is read), then single tokens of both
    for chunks in [(20, 0), (17, 64), (0, 26)] + [(1, 1)] * 12:
        ids = []
        for s, n in enumerate(chunks):
            ids.append(seqs[s][at[s]:at[s] + n])
            at[s] += n
        logits = server.step(torch.cat(ids), table, _i32([0, chunks[0], sum(chunks)], gpu), _i32(at, gpu))
        first = 0
        for s, n in enumerate(chunks):
            served[s].append(logits[first:first + n])
            first += n
        if at[0] >= 37 and at[1] >= 90:  # both prompts read: draw the next token of each
            last = torch.stack([served[0][-1][-1] if chunks[0] else served[0][-2][-1], served[1][-1][-1]])
            u = torch.rand(2, generator=g).to(gpu)
            token = sample(last, u, temperature=0.9, top_k=40, top_p=0.95)
            assert ((token >= 0) & (token < 1000)).all()
            for s in range(2):
                seqs[s] = torch.cat([seqs[s], token[s:s + 1]])
    ref = llama.LlamaModel(vocab_size=1000, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, hidden_dim=512, max_seq_len=128)
    ref.load_state_dict(m.state_dict())
    ref = ref.double().eval()  # (on the CPU, in 64 bits)
    for s in range(2):
        with torch.no_grad():
            want = ref(seqs[s][None, :at[s]].cpu())[0]
            stock = m(seqs[s][None, :at[s]])[0].double().cpu()
        got = torch.cat(served[s]).double().cpu()
        assert got.shape == want.shape
        # As close to 64 bits as the stock modules are on the same weights: they round at the same places, except
        # that the weights of attention are rounded too in f16; twice the stock error allows for that and for
        # another order of sums.
        assert (got - want).abs().max() <= 2 * (stock - want).abs().max(), dtype
        assert (got - want).abs().mean() <= 1.5 * (stock - want).abs().mean(), dtype


def test_decode_step_in_one_graph(gpu):
    """A whole decode step (two layers, sampling, the sampled tokens fed back) captured once; its replays equal eager
    steps bit for bit while the sequences grow past a page's end."""
    m = _model(gpu, torch.float16)
    g = torch.Generator().manual_seed(2)
    page, B = 16, 3
    table = torch.randperm(24, generator=g).to(torch.int32).view(B, 8).to(gpu)
    prompts = torch.randint(0, 1000, (B, 14), generator=g).to(gpu)
    numbers = torch.rand(8, B, generator=g).to(gpu)
    starts = _i32([0, 1, 2, 3], gpu)

    def fresh():
        s = Server(m, pages=24, page=page)
        logits = s.step(prompts.reshape(-1), table, _i32([0, 14, 28, 42], gpu), _i32([14] * B, gpu))
        return s, sample(logits[13::14].contiguous(), numbers[0], top_p=0.9), _i32([15] * B, gpu)

    def step(s, ids, lens, u):
        out = sample(s.step(ids, table, starts, lens), u, top_p=0.9)
        ids.copy_(out)
        lens.add_(1)

    s, ids, lens = fresh()
    eager = []
    for i in range(1, 8):
        step(s, ids, lens, numbers[i])
        eager.append(ids.clone())
    s, ids, lens = fresh()
    u = numbers[1].clone()
    keep = [t.clone() for t in (ids, lens, s.k, s.v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, ids, lens, u)
    torch.cuda.current_stream().wait_stream(side)
    for t, old in zip((ids, lens, s.k, s.v), keep):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s, ids, lens, u)
    for t, old in zip((ids, lens, s.k, s.v), keep):
        t.copy_(old)
    for i in range(1, 8):
        u.copy_(numbers[i])
        graph.replay()
        torch.cuda.synchronize()
        other = sample(torch.randn(4, 500, device=gpu), torch.rand(4, device=gpu))  # eager work in between
        assert other.shape == (4,) and torch.equal(ids, eager[i - 1]), i


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_on_a_device_that_is_not_current(gpu):
    x = torch.randn(3, 900, device="cuda:1")
    assert sample(x, torch.rand(3, device="cuda:1")).device == x.device
