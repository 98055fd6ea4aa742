"""examples/decode_with_drafts.py: the operators together, node by node against exact attention over what was kept, and the bookkeeping."""
import importlib.util
import os

import pytest
import torch

from .conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("decode_with_drafts", os.path.join(ROOT, "examples", "decode_with_drafts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _prompts(lengths):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(512, (n,), generator=g).tolist() for n in lengths]


def _turn(x, positions, freqs):
    angle = positions.double()[:, None] * freqs.double()
    c, s = angle.cos()[:, None].float(), angle.sin()[:, None].float()
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("depth", [0, 1, 5])
def test_every_node_is_attention_over_its_past(depth):
    """The first layer's output for every node against fp32 attention over the bf16 keys and values that were kept, turned to their positions, and its ancestors'.  The cache holds
    them in e4m3: half of the last of four significant bits, 2^-4 of a value at most, about 0.027 of the norm for evenly spread ones; the weights shift by as much again."""
    m = _example()
    model, prompts = m.Model(), _prompts([1, 33, 70])
    seen = []

    def record(q, k, v, o):
        seen.append([t.clone() for t in (q, k, v, o)])

    decoder = m.Decoder(model, prompts, 400, depth)
    # the prompts' keys and values of the first layer, made again
    history = []
    for p in prompts:
        x = model.embedding[torch.tensor(p).cuda()] * 16.0
        norm = x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)
        history.append(list((norm @ model.layers[0][0]).view(len(p), -1, model.d).split([model.h, model.hk, model.hk], dim=1))[1:])
    parents = [-1] + [max(0, 2 * (d - 1) - 1) for d in range(1, depth + 1) for _ in (0, 1)]
    worst, several = [], 0
    for _ in range(40):
        before = decoder.lengths.tolist()
        out, counts = decoder.step(record)
        q, k, v, o = seen.pop()
        tokens_in = [h[0].shape[0] for h in history]
        assert tokens_in == before
        for b in range(len(prompts)):
            kk, vv = history[b]
            for i in range(len(parents)):
                line = [i]
                while parents[line[0]] >= 0:
                    line.insert(0, parents[line[0]])
                ks, vs = torch.cat([kk, k[b, line]]), torch.cat([vv, v[b, line]]).float()
                n = ks.shape[0]
                ks = _turn(ks, torch.arange(n, device="cuda"), model.freqs).repeat_interleave(4, 1)
                qq = _turn(q[b, i:i + 1], torch.tensor([n - 1], device="cuda"), model.freqs)[0]
                p = torch.softmax(torch.einsum("hd,nhd->hn", qq, ks) * 128 ** -0.5, -1)
                want = torch.einsum("hn,nhd->hd", p, vs.repeat_interleave(4, 1))
                worst.append(float((o[b, i].float() - want).norm() / want.norm()))
        # what was kept: by the answers alone, from the drafts as they stood
        for b, n in enumerate(counts.tolist()):
            several += n > 1
            line = [0]
            for d in range(1, n):
                first, second = 2 * d - 1, 2 * d
                line.append(first if torch.equal(k[b, first], _key(model, out[b, d - 1])) else second)
                assert torch.equal(k[b, line[-1]], _key(model, out[b, d - 1]))          # the node is the token that was answered
            history[b] = [torch.cat([h, t[b, line]]) for h, t in zip(history[b], (k, v))]
    assert max(worst) < 0.08, max(worst)                          # the bound of the framework's own e4m3 attention
    assert depth == 0 or several > 10
    m.ops.check_status()


def _key(model, token):
    """A first-layer key by its token."""
    x = model.embedding[token[None, None]] * 16.0
    norm = x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)
    return (norm.expand(3, 1, -1) @ model.layers[0][0]).view(3, -1, model.d)[0, model.h:model.h + model.hk]


def test_graph_equals_eager():
    m = _example()
    model = m.Model()
    eager = m.generate(model, _prompts([5, 40, 64]), 60, 4, graph=False)
    captured = m.generate(model, _prompts([5, 40, 64]), 60, 4)
    assert eager == captured and eager[1] < 60


def test_main_runs(monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["decode_with_drafts.py", "--tokens", "30", "--depth", "3"])
    _example().main()
    assert capsys.readouterr().out.count("a pass and sequence") == 2
