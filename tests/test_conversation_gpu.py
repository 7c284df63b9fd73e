"""The operators of a bounded conversation together, as an engine runs them: pages taken by fork_pages, prompts and tokens written
by norm_rotary_cache_write, attention by forward_window and decode with a window and sinks, sequences that fork, end and go on,
pages given back behind the window and taken by others, compact_pages now and then. After every step the attention is compared
with float64 over each sequence's own rows, kept aside as they were written, and the pages with the tables' counts.
"""
import random

import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs,layout,window,sinks,hq,hkv", [(16, "HND", 40, 5, 12, 2), (48, "NHD", 33, 1, 24, 4), (8, "HND", 70, 20, 6, 6)])
def test_steps(bs, layout, window, sinks, hq, hkv):
    rng, g = random.Random(bs), torch.Generator().manual_seed(bs)
    layers, pages, cols, scale = 2, 420 // bs + 40, 300 // bs + 2, 1 / 16
    caches = [kvc.allocate_cache(pages, bs, hkv, layout, "cuda") for _ in range(layers)]
    for c in caches:
        c.kv.copy_(torch.randint(-128, 128, c.kv.shape, dtype=torch.int8, generator=g))  # (pages never written hold noise)
    table = rotary.rotary_table(64, 400, 1e4).cuda()
    weights = [[(torch.rand(256, generator=g) + 0.5).half().cuda() for _ in range(2)] for _ in range(layers)]
    rows = 4
    bt = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    needed = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = [[[] for _ in range(rows)] for _ in range(layers)]  # per layer and row: (K, V) [Hkv, 256] of each key, dequantised

    def attention(layer, out, q, starts, host_lens):
        worst = 0.0
        for b, (q0, q1) in enumerate(zip(starts, starts[1:])):
            if q1 == q0 or host_lens[b] == 0:
                continue
            k, v = (torch.stack([x[i] for x in kept[layer][b]]).double() for i in range(2))  # [n, Hkv, 256]
            key = torch.arange(host_lens[b])
            for i in range(q0, q1):
                p = host_lens[b] - (q1 - i)
                see = (key <= p) & ((p - key < window) | (key < sinks))
                for h in range(hq):
                    x = torch.mv(k[see][:, h // (hq // hkv)], q[i, h].double()) * scale
                    ref = torch.softmax(x, 0) @ v[see][:, h // (hq // hkv)]
                    worst = max(worst, kvc.fp16_output_errors(out[i, h].double().numpy(), ref.numpy())[2])
        assert worst <= 0, worst

    def step(parents, news):
        """Tables for news[i] more keys of row i, which goes on from parents[i]; the tokens through both layers."""
        nonlocal bt, lens, refs, kept
        grow = max(news)
        par = None if parents is None else torch.tensor(parents, dtype=torch.int32, device="cuda")
        n = bt.shape[0] if parents is None else len(parents)
        new_bt, new_lens, new_refs = torch.empty((n, cols), dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"), \
            torch.empty_like(refs)
        free = int((refs == 0).sum())
        pth_dec.fork_pages(caches, refs, bt, lens, par, new_refs, new_bt, new_lens, needed, grow=grow, window=window, sinks=sinks)
        assert int(needed) <= free
        bt, lens, refs = new_bt, new_lens, new_refs
        kept = [[list(layer[p]) if p >= 0 else [] for p in (range(n) if parents is None else parents)] for layer in kept]
        before = lens.tolist()
        assert before == [len(x) for x in kept[0]]
        live = [parents is None or p >= 0 for p in (parents or range(n))]
        news = [x if a else 0 for x, a in zip(news, live)]
        starts = [0]
        for x in news:
            starts.append(starts[-1] + x)
        row = torch.tensor([b for b, x in enumerate(news) for _ in range(x)])
        pos = torch.tensor([before[b] + i for b, x in enumerate(news) for i in range(x)])
        page = bt.cpu()[row, pos // bs].long()
        assert bool((page >= 0).all())
        slots = (page * bs + pos % bs).cuda()
        lens = lens + torch.tensor(news, dtype=torch.int32, device="cuda")
        host_lens = lens.tolist()
        qsl = torch.tensor(starts, dtype=torch.int32, device="cuda")
        T = starts[-1]
        for layer, c in enumerate(caches):
            qkv = torch.randn((T, hq + 2 * hkv, 256), generator=g).half().cuda()
            q = torch.empty((T, hq, 256), dtype=torch.float16, device="cuda")
            pth_dec.norm_rotary_cache_write(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], *weights[layer], pos.cuda(), table,
                                            c.key_cache, c.value_cache, c.k_scale, c.v_scale, slots, query_out=q)
            out = torch.full_like(q, 7.0)
            if max(news) > 4:
                pth_dec.forward_window(q, c.key_cache, c.value_cache, bt, lens, scale, qsl, out, window, sinks=sinks)
            else:
                bufs = kvc.partial_buffers(T, hq, 16, "cuda")
                pth_dec.decode(q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, bt, lens, qsl, out, scale, *bufs, n, max(news),
                               rng.choice([1, 4, 16]), window=window, sinks=sinks)
            k = c.key_cache[page, pos % bs, :, :256].float() * c.k_scale[page, pos % bs][..., None]
            v = c.value_cache[page, pos % bs, :, :256].float() * c.v_scale[page, pos % bs][..., None]
            for i in range(T):
                kept[layer][int(row[i])].append((k[i].cpu(), v[i].cpu()))
            attention(layer, out.cpu(), q.cpu(), starts, host_lens)
        counts = torch.zeros(pages + 1, dtype=torch.int32)
        counts.index_add_(0, torch.where(bt.cpu() < 0, pages, bt.cpu()).view(-1).long(), torch.ones(bt.numel(), dtype=torch.int32))
        assert torch.equal(counts[:pages], refs.cpu())

    def compact():
        nonlocal bt, refs
        places, used = torch.empty_like(refs), torch.empty(1, dtype=torch.int32, device="cuda")
        count = int((refs > 0).sum())
        pth_dec.compact_pages(caches, refs, bt, refs, bt, places, used)
        assert int(used) == count and bool((refs[:count] > 0).all()) and not bool(refs[count:].any()) and int(bt.max()) < count

    step(None, [50, 7, 90, 33])
    for i in range(14):
        if i == 3:
            step([2, 0, 2, 2, -1, 1], [1, 2, 1, 3, 1, 1])     # three go on from row 2, row 3 ends, an empty row
        elif i == 7:
            compact()
            step([5, 0, 1, 4, 3], [30, 5, 12, 60, 1])         # another turn's tokens, the empty row's first ones
        elif i == 11:
            step([3, 3, 0], [1, 1, 1])
            compact()
        else:
            step(None, [rng.choice([1, 1, 2, 4]) for _ in range(bt.shape[0])])
    assert int((refs > 0).sum()) < pages
