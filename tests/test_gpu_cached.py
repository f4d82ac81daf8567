"""The cached decoder: the operators together, as a serving step uses them.

A prompt run at once, in parts and token by token goes through different
kernels (matrix products of different batch sizes, appends of different
sizes, split and unsplit attention); the answers agree within f32's
accumulation error and the cache's own: codes are e4m3, and a key or value
whose f32 bits differ in the last places may round to the neighbouring code,
2^-3 of itself, for about one in 2^17 of them.  Log probabilities of size up
to 20 are compared to 2e-2, and most of them to 1e-4.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB = 4096


def inputs(rows, seed):
    return torch.randn(rows, 1536, generator=torch.Generator().manual_seed(seed)).to(DEV)


def decoder(ctx, **kw):
    from q4k.cached import CachedDecoder

    return CachedDecoder(ctx, layers=2, seqs=3, positions=512, vocab=VOCAB, **kw)


def near(a, b):
    d = (a - b).abs()
    assert float(d.max()) <= 2e-2
    assert float((d <= 1e-4).float().mean()) >= 0.9


@pytest.mark.parametrize("window", [0, 24])
@pytest.mark.parametrize("page_size", [16, 64])
def test_at_once_in_parts_and_token_by_token(ctx, window, page_size):
    lengths = [40, 17, 33]
    xs = [inputs(n, 10 + i) for i, n in enumerate(lengths)]
    tokens = [torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(i), dtype=torch.int32).to(DEV)
              for i, n in enumerate(lengths)]
    whole = decoder(ctx, window=window, page_size=page_size).step(torch.cat(xs), lengths, torch.cat(tokens), top=5)
    want = whole.logprob.split(lengths)

    parts = decoder(ctx, window=window, page_size=page_size)
    got = [[], [], []]
    for lo, hi in ((0, 16), (16, 17), (17, 29), (29, 40)):
        counts = [max(0, min(hi, n) - min(lo, n)) for n in lengths]
        rows = [slice(min(lo, n), min(hi, n)) for n in lengths]
        a = parts.step(torch.cat([x[r] for x, r in zip(xs, rows)]), counts,
                       torch.cat([t[r] for t, r in zip(tokens, rows)]), top=5)
        for g, p in zip(got, a.logprob.split(counts)):
            g.append(p)
    for g, w in zip(got, want):
        near(torch.cat(g), w)

    single = decoder(ctx, window=window, page_size=page_size)
    got = [[], [], []]
    for i in range(max(lengths)):
        on = [int(i < n) for n in lengths]
        a = single.step(torch.cat([x[i : i + 1] for x, o in zip(xs, on) if o]), on,
                        torch.cat([t[i : i + 1] for t, o in zip(tokens, on) if o]), top=5)
        for g, p in zip(got, a.logprob.split(on)):
            g.append(p)
    ctx.check()
    for g, w in zip(got, want):
        near(torch.cat(g), w)


def test_answers(ctx):
    d = decoder(ctx)
    a = d.step(inputs(9, 3), [4, 0, 5], top=8)
    ctx.check()
    assert torch.isnan(a.logprob).all()  # no token was asked for
    assert torch.isfinite(a.entropy).all() and (a.entropy > 0).all()
    assert (a.top_logprob[:, :-1] >= a.top_logprob[:, 1:]).all()
    b = decoder(ctx).step(inputs(9, 3), [4, 0, 5], a.top_token[:, 0].contiguous(), top=1)
    assert torch.equal(b.logprob, a.top_logprob[:, 0])
    with pytest.raises(ValueError):
        d.step(inputs(2, 1), [1, 1])
    with pytest.raises(ValueError):
        d.step(inputs(513, 1), [513, 0, 0])
