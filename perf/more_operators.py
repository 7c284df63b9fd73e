"""Long conversations in a bounded int8 paged KV cache, as measurable cases.

  decode   a decode step whose rows see their last `window` keys and the first `sinks` ones
           (decode(.., window=, sinks=)).
  prefill  the same attention for chunks of new tokens, several sequences in one call (forward_window).
  write    RMS norms of the query and key heads, rotary positions, the keys and values quantised into the
           cache rows, in one pass (norm_rotary_cache_write).
  fork     a serving step's block tables: every new row goes on from a parent row, full pages are shared, a
           part-filled one is copied where others go on from it too, pages that the window has left are
           dropped, room for the next tokens is taken from the free pages (fork_pages).
  compact  the used pages moved into the lowest numbers, tables and reference counts with them
           (compact_pages).

Sizes are those of this repository's benchmark and tests: 24 q / 4 kv heads (the whole model on one
GPU) and 12 / 2 (one of two tensor-parallel ranks), head size 256, block sizes 16 to 1,584, contexts
of up to 61,440 keys, windows of 1,000 to 8,192 keys, 1 to 8 query tokens per decoded sequence.

`own` False computes the operators from elementary torch operations, True calls the package.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DIM, _HALF, _ROW = 256, 260, 520
_SCALE = 1.0 / math.sqrt(_DIM)
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_POSITIONS = 65536  # rows of the rotary table
_BASE = 1e6
_EPS = 1e-6
_SEGMENTS = 64      # of the decode's partial buffers


def _package():
    name = "mi50_vllm_lab_amd"
    if name not in sys.modules:
        d = os.path.join(_ROOT, "mi50-vllm-lab_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        sys.modules[name] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _case(kind, name, **kw):
    c = {"name": name, "kind": kind, "heads_q": 24, "heads_kv": 4, "block_size": 16, "layout": "HND"}
    c.update(kw)
    return c


def listed():
    return [
        # one user's next token in a long conversation: launches and latency are what is left
        _case("decode", "decode_1x1_2k", seqs=1, qlen=1, ctx_lo=30000, ctx_hi=30000, window=2048, sinks=4, causal=True),
        # a full batch of conversations, some of them still shorter than the window
        _case("decode", "decode_96x1_4k", seqs=96, qlen=1, ctx_lo=200, ctx_hi=61440, window=4096, sinks=4, causal=True),
        # odd sizes: a drafter's non-causal rows on one rank's heads, the reference's block size, more sinks than a tile holds
        _case("decode", "decode_5x3_odd_rank", seqs=5, qlen=3, ctx_lo=700, ctx_hi=20000, window=1000, sinks=37, causal=False,
              heads_q=12, heads_kv=2, block_size=1584, layout="NHD"),
        # a short turn of a long conversation
        _case("prefill", "prefill_64_2k", seqs=1, new_lo=64, new_hi=64, ctx_lo=30000, ctx_hi=30000, window=2048, sinks=4),
        # a ragged batch of turns on one rank's heads, sizes that no tile divides
        _case("prefill", "prefill_7x_odd_rank", seqs=7, new_lo=33, new_hi=1100, ctx_lo=100, ctx_hi=9000, window=1000, sinks=37,
              heads_q=12, heads_kv=2, block_size=1584),
        # the largest: a fresh prompt in one chunk
        _case("prefill", "prefill_8k_4k", seqs=1, new_lo=8192, new_hi=8192, ctx_lo=0, ctx_hi=0, window=4096, sinks=4),
        # a decode batch of a bf16 model, a quarter of the head rotated, queries handed on in the decode operator's fp16
        _case("write", "write_33_bf16_part", tokens=33, dtype="bf16", rotary_dim=64, interleaved=False, prompt=False, out="fp16"),
        # a long prompt on one rank's heads, adjacent pairs
        _case("write", "write_16k_pairs_rank", tokens=16384, dtype="fp16", rotary_dim=256, interleaved=True, prompt=True, out="same",
              heads_q=12, heads_kv=2, block_size=1584),
        # a decode step's pages: every sequence goes on, a few need a page, a few lose one behind the window
        _case("fork", "fork_step_48", seqs=48, children=48, layers=4, ctx_lo=200, ctx_hi=30000, window=2048, sinks=4, grow=1,
              spare=64, step=True),
        # sixteen of 64 rows go on in 64 new ones (samples, beams): full pages shared, part-filled ones copied
        _case("fork", "fork_64_of_64", seqs=64, children=64, layers=16, ctx_lo=300, ctx_hi=2000, window=0, sinks=0, grow=4,
              spare=160, step=False),
        # a pool after many sequences have come and gone
        _case("compact", "compact_6k_pages", pages=6144, used=0.55, seqs=48, layers=8),
        # few large pages, tokens-major, one rank's heads
        _case("compact", "compact_large_pages_rank", pages=150, used=0.7, seqs=5, layers=2, heads_q=12, heads_kv=2, block_size=1584,
              layout="NHD"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; none costs more than prefill_8k_4k."""
    hq, hkv = rng.choice([(24, 4), (24, 4), (12, 2)])
    common = {"heads_q": hq, "heads_kv": hkv, "block_size": rng.choice([16, 16, 32, 48, 1584]),
              "layout": rng.choice(["HND", "HND", "NHD"])}
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "write", "fork", "compact"])
    window, sinks = _log_int(rng, 1000, 8192), rng.choice([0, 1, 4, 16, 37, 128])
    if kind == "decode":
        seqs, hi = _log_int(rng, 1, 128), _log_int(rng, 300, 61440)
        window = min(window, 400000 // seqs)
        c = _case(kind, "", seqs=seqs, qlen=rng.choice([1, 1, 2, 4, 8]), ctx_lo=max(1, hi // rng.choice([1, 8, 64])), ctx_hi=hi,
                  window=window, sinks=sinks, causal=rng.random() < 0.8, **common)
    elif kind == "prefill":
        seqs, window = rng.choice([1, 1, 2, 5, 16]), min(window, 4096)
        new, hi = _log_int(rng, 16, 8192 // seqs), rng.choice([0, _log_int(rng, 10, 61440)])
        c = _case(kind, "", seqs=seqs, new_lo=max(1, new // rng.choice([1, 3, 20])), new_hi=new, ctx_lo=hi // rng.choice([1, 8]), ctx_hi=hi,
                  window=window, sinks=sinks, **common)
    elif kind == "write":
        c = _case(kind, "", tokens=_log_int(rng, 1, 16384), dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]),
                  rotary_dim=rng.choice([256, 128, 64, 64, 96, 200]), interleaved=rng.random() < 0.4, prompt=rng.random() < 0.5,
                  out=rng.choice(["inplace", "same", "fp16"]), **common)
    elif kind == "fork":
        seqs, step = _log_int(rng, 1, 96), rng.random() < 0.4
        children = seqs if step else _log_int(rng, 1, 96)
        grow, keys = rng.choice([0, 1, 4, 100]), 40000 if common["block_size"] <= 48 else 200000
        hi = _log_int(rng, 20, max(40, keys // max(seqs, children)))
        c = _case(kind, "", seqs=seqs, children=children, layers=rng.choice([1, 4, 8]), ctx_lo=max(1, hi // rng.choice([1, 8])), ctx_hi=hi,
                  window=rng.choice([0, min(window, max(1, hi // 2))]), sinks=sinks, grow=grow,
                  spare=children * (1 + -(-grow // common["block_size"])) + rng.choice([0, 7, 300 if common["block_size"] <= 48 else 20]),
                  step=step, **common)
    else:
        large = common["block_size"] > 48
        pages = _log_int(rng, 10, 150) if large else _log_int(rng, 50, 6144)
        c = _case(kind, "", pages=pages, used=rng.choice([0.05, 0.4, 0.7, 0.95]), seqs=_log_int(rng, 1, max(2, min(64, pages // 8))),
                  layers=rng.choice([1, 2] if large else [1, 4, 8]), **common)
    del c["name"]
    return c


# ---- inputs, from the seed alone ----

def _lengths(n, lo, hi, what):
    """A length for each sequence, evenly spread over their logarithm, in an order fixed by the case."""
    if lo <= 0:
        return [0] * n
    a, b = math.log(lo), math.log(hi)
    out = [int(round(math.exp(a + (b - a) * i / (n - 1)))) for i in range(n)] if n > 1 else [hi]
    random.Random("%s %d %d" % (what, n, hi)).shuffle(out)
    return out


def _batch(case):
    """(query tokens, keys with them) of each sequence."""
    n = case["seqs"]
    new = [case["qlen"]] * n if case["kind"] == "decode" else _lengths(n, case["new_lo"], case["new_hi"], "new")
    return [(t, c + t) for t, c in zip(new, _lengths(n, case["ctx_lo"], case["ctx_hi"], "ctx"))]


def _first_seen(case, new, length):
    """The first key that the window of a sequence's first row holds."""
    return max(0, length - new - case["window"] + 1)


def _rand_rows(gen, rows):
    """int8 cache rows [rows, 520] of K, V ~ N(0, 1)."""
    kv = torch.empty((rows, _ROW), dtype=torch.int8, device="cuda")
    step = 1 << 18
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = torch.randn((n, 2, _DIM), device="cuda", generator=gen)
        s = x.abs().amax(-1, keepdim=True) / 127.0
        kv[r:r + n].view(n, 2, _HALF)[:, :, :_DIM] = (x / s).round_().clamp_(-127, 127).to(torch.int8)
        kv[r:r + n].view(n, 2, _HALF)[:, :, _DIM:] = s.view(torch.int8).view(n, 2, 4)
    return kv


def _blocks(case, pages, rows):
    """Raw cache [blocks, Hkv, block_size, 520] in the case's order."""
    if case["layout"] == "HND":
        return rows.view(pages, case["heads_kv"], case["block_size"], _ROW)
    return rows.view(pages, case["block_size"], case["heads_kv"], _ROW).transpose(1, 2)


def _views(kv):
    """The operators' views of a raw cache: int8 [blocks, block_size, Hkv, 260] for K and V, fp32 [blocks, block_size, Hkv] for
    their scales; and all int8 values and scales as [blocks, Hkv, block_size, 2, ..]."""
    f32 = torch.tensor([], dtype=torch.float32, device="cuda").set_(kv.untyped_storage())
    nblk, hkv, bs, _ = kv.shape
    st = [x // 4 for x in kv.stride()]
    key, value = kv.transpose(1, 2).split(_HALF, dim=-1)
    ks, vs = (torch.as_strided(f32, (nblk, bs, hkv), (st[0], st[2], st[1]), o) for o in (_DIM // 4, (_HALF + _DIM) // 4))
    rows = torch.as_strided(kv, (nblk, hkv, bs, 2, _DIM), (*kv.stride()[:3], _HALF, 1))
    scales = torch.as_strided(f32, (nblk, hkv, bs, 2, 1), (*st[:3], _HALF // 4, 1), _DIM // 4)
    return {"kv": kv, "key_cache": key, "value_cache": value, "k_scale": ks, "v_scale": vs, "rows": rows, "scales": scales}


def _prepare_attention(case, gen, host):
    hq, hkv, bs = case["heads_q"], case["heads_kv"], case["block_size"]
    batch = _batch(case)
    n, tokens = len(batch), sum(t for t, _ in batch)
    bt = torch.full((n, max(-(-x // bs) for _, x in batch)), -1, dtype=torch.int32)
    held = []  # pages with a key that some row sees: the others have been given back
    for b, (new, length) in enumerate(batch):
        lo = _first_seen(case, new, length) // bs
        first = min(-(-case["sinks"] // bs), lo)
        held += [(b, c) for c in range(-(-length // bs)) if c < first or c >= lo]
    perm = torch.randperm(len(held) + 2, generator=host).to(torch.int32)
    at = torch.tensor(held)
    bt[at[:, 0], at[:, 1]] = perm[:len(held)]
    s = _views(_blocks(case, len(held) + 2, _rand_rows(gen, (len(held) + 2) * bs * hkv)))
    s["q"] = torch.randn((tokens, hq, _DIM), device="cuda", generator=gen).half()
    s["out"] = torch.zeros_like(s["q"])
    starts = [0]
    for t, _ in batch:
        starts.append(starts[-1] + t)
    s["block_table"], s["query_start_loc"] = bt.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["lens_host"] = torch.tensor([x for _, x in batch], dtype=torch.int32)
    s["seq_lens"] = s["lens_host"].cuda()
    s["batch"], s["starts"] = batch, starts
    if case["kind"] == "decode":
        s["seg"] = [torch.empty((tokens, hq, _SEGMENTS) + d, device="cuda") for d in ((_DIM,), (), ())]
        s["tok"] = torch.arange(case["qlen"], device="cuda")
        # the places of a row of keys in the plain form: the sinks, then the window of the first row up to the last key
        s["place"] = torch.arange(case["sinks"] + case["window"] + case["qlen"] - 1, device="cuda")
        if own:  # the engine's split count for such a batch
            shim = _package().vllm_shim
            plan = (_SEGMENTS, case["window"] + case["sinks"], hkv, n, s["q"].device, s["lens_host"], case["qlen"], hq)
            s["nsplit"] = shim.launched_splits(shim.decode_splits(*plan), *plan)
    return s


def _prepare_write(case, gen, host):
    hq, hkv, bs, t, dt, rd = (case[k] for k in ("heads_q", "heads_kv", "block_size", "tokens", "dtype", "rotary_dim"))
    dt = _DTYPES[dt]
    qkv = torch.randn((t, (hq + 2 * hkv) * _DIM), device="cuda", generator=gen).mul_(3.0).to(dt)
    heads = qkv.view(t, hq + 2 * hkv, _DIM)
    s = {"query": heads[:, :hq], "key": heads[:, hq:hq + hkv], "value": heads[:, hq + hkv:]}
    s["query_weight"], s["key_weight"] = (torch.rand(_DIM, device="cuda", generator=gen).add_(0.5).to(dt) for _ in range(2))
    angle = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * \
        _BASE ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)[None, :]
    s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float()
    first = int(torch.randint(0, _POSITIONS - t, (1,), generator=host))
    s["positions"] = torch.arange(first, first + t, device="cuda") if case["prompt"] else \
        torch.randint(0, _POSITIONS, (t,), generator=host).cuda()
    pages = -(-t // bs)
    slots = (torch.randperm(pages, generator=host)[:, None] * bs + torch.arange(bs)[None, :]).reshape(-1)[:t]
    s["slots"] = slots.cuda()
    s.update(_views(_blocks(case, pages, torch.zeros((pages * bs * hkv, _ROW), dtype=torch.int8, device="cuda"))))
    # in place the query's values would be normed again in every pass: a program's are fresh ones each time
    out = {"inplace": None, "same": dt, "fp16": torch.float16}[case["out"]]
    s["query_out"] = None if out is None else torch.empty((t, hq, _DIM), dtype=out, device="cuda")
    return s


def _prepare_pages(case, gen, host):
    bs, n = case["block_size"], case["seqs"]
    rng = random.Random("pages %d %d" % (n, case["layers"]) + str(int(torch.randint(0, 1 << 30, (1,), generator=host))))
    if case["kind"] == "fork":
        lens = _lengths(n, case["ctx_lo"], case["ctx_hi"], "ctx")
        cols = max(-(-(x + case["grow"]) // bs) for x in lens)
        holes = [max(0, x - case["window"]) // bs if case["window"] else 0 for x in lens]  # what earlier steps gave back
        first = -(-case["sinks"] // bs)
        held = [(b, c) for b, x in enumerate(lens) for c in range(-(-x // bs)) if c < first or c >= holes[b]]
        pages = len(held) + case["spare"]
        s = {"seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "parents": None}
        if not case["step"]:  # the better rows have more children, some have none, a few new rows are empty
            best = rng.sample(range(n), max(1, n // 4))
            s["parents"] = torch.tensor([-1 if rng.random() < 0.03 else rng.choice(best) for _ in range(case["children"])],
                                        dtype=torch.int32, device="cuda")
        s["needed"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        pages = case["pages"]
        live = max(1, int(pages * case["used"]))
        cols = -(-live // n) + 3
        held = [(i % n, i // n) for i in range(live)]
        s = {"used": torch.zeros(1, dtype=torch.int32, device="cuda"), "places": torch.zeros(pages, dtype=torch.int32, device="cuda")}
    perm = torch.randperm(pages, generator=host).to(torch.int32)
    bt = torch.full((n, cols), -1, dtype=torch.int32)
    at = torch.tensor(held)
    bt[at[:, 0], at[:, 1]] = perm[:len(held)]
    if n > 1:  # a prompt's first page that two rows share
        a, b = sorted(rng.sample(range(n), 2))
        if case["kind"] == "compact" or min(lens[a], lens[b]) >= bs:
            bt[b, 0] = bt[a, 0]
    refs = torch.zeros(pages + 1, dtype=torch.int32)
    refs.index_add_(0, torch.where(bt < 0, pages, bt).view(-1).long(), torch.ones(bt.numel(), dtype=torch.int32))
    s["refs"], s["block_table"] = refs[:pages].cuda(), bt.cuda()
    rows = s["block_table"].shape[0] if case["kind"] == "compact" or case["step"] else case["children"]
    s["new_block_table"] = torch.zeros((rows, cols), dtype=torch.int32, device="cuda")
    s["new_seq_lens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s["new_refs"] = torch.zeros_like(s["refs"])
    # (their bytes are moved, not read)
    s["caches"] = [_blocks(case, pages, torch.randint(-128, 128, (pages * bs * case["heads_kv"], _ROW), dtype=torch.int8, device="cuda",
                                                      generator=gen)) for _ in range(case["layers"])]
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    make = {"decode": _prepare_attention, "prefill": _prepare_attention, "write": _prepare_write}.get(case["kind"], _prepare_pages)
    return {"case": case, **make(case, gen, host)}


# ---- the operators ----

def _gather(s, page, at):
    """K and V of the keys at (page, at) [..] in 32 bits: [.., Hkv, 256] each."""
    k = s["key_cache"][page, at, :, :_DIM].float() * s["k_scale"][page, at][..., None]
    return k, s["value_cache"][page, at, :, :_DIM].float() * s["v_scale"][page, at][..., None]


def _plain_decode(s):
    """The visible keys of each sequence side by side (padded to sinks + window + qlen - 1), masked row by row."""
    case = s["case"]
    n, new, hq, hkv, bs, window, sinks = (case[k] for k in ("seqs", "qlen", "heads_q", "heads_kv", "block_size", "window", "sinks"))
    g = hq // hkv
    lens = s["seq_lens"].long()[:, None]
    lo = (lens - new - window + 1).clamp(min=0)
    place = s["place"][None, :]
    key = torch.where(place < sinks, place, lo + place - sinks)                       # [n, K]
    live = (key < lens) & ((place < sinks) | (key >= sinks))                          # (a sink inside the window counts once)
    # (a sink that the sequence does not have, or a place past its end: read its last key)
    safe = torch.where(live, key, lens - 1)
    k, v = _gather(s, torch.gather(s["block_table"].long(), 1, safe // bs), safe % bs)  # [n, K, Hkv, 256]
    q = s["q"].float().view(n, new, hkv, g, _DIM).mul(_SCALE).transpose(1, 2).reshape(n, hkv, new * g, _DIM)
    x = (q @ k.permute(0, 2, 3, 1).contiguous()).view(n, hkv, new, g, -1)
    at = lens - new + s["tok"][None, :]                                               # [n, new]
    seen = live[:, None, :] & ((at[:, :, None] - key[:, None, :] < window) | (key[:, None, :] < sinks))
    if case["causal"]:
        seen = seen & (key[:, None, :] <= at[:, :, None])
    x = x.masked_fill(~seen[:, None, :, None, :], -math.inf).view(n, hkv, new * g, -1)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    o = (x @ v.transpose(1, 2).contiguous()) / x.sum(-1, keepdim=True)
    s["out"].copy_(o.view(n, hkv, new, g, _DIM).transpose(1, 2).reshape(n * new, hq, _DIM))


def _plain_prefill(s):
    """Runs of up to 1,024 tokens of a sequence against the keys that any of them sees, masked."""
    case = s["case"]
    hq, hkv, bs, window, sinks = (case[k] for k in ("heads_q", "heads_kv", "block_size", "window", "sinks"))
    g = hq // hkv
    for b, (new, length) in enumerate(s["batch"]):
        table = s["block_table"][b].long()
        for t0 in range(0, new, 1024):
            t = min(1024, new - t0)
            p0 = length - new + t0
            lo = max(0, p0 - window + 1)
            key = torch.cat([torch.arange(min(sinks, lo), device="cuda"), torch.arange(lo, p0 + t, device="cuda")])
            k, v = _gather(s, table[key // bs], key % bs)                             # [K, Hkv, 256]
            rows = s["q"][s["starts"][b] + t0:s["starts"][b] + t0 + t]
            q = rows.float().mul(_SCALE).view(t, hkv, g, _DIM).transpose(0, 1).reshape(hkv, t * g, _DIM)
            x = (q @ k.permute(1, 2, 0).contiguous()).view(hkv, t, g, -1)
            at = p0 + torch.arange(t, device="cuda")[:, None]
            seen = (key <= at) & ((at - key < window) | (key < sinks))
            x = x.masked_fill_(~seen[None, :, None, :], -math.inf).view(hkv, t * g, -1)
            x = x.sub_(x.amax(-1, keepdim=True)).exp_()
            o = (x @ v.transpose(0, 1).contiguous()) / x.sum(-1, keepdim=True)
            s["out"][s["starts"][b] + t0:s["starts"][b] + t0 + t] = o.view(hkv, t, g, _DIM).transpose(0, 1).reshape(t, hq, _DIM).half()


def _plain_head(case, x, weight, cos_sin):
    """x [T, H, 256] in 32 bits: over its root mean square, times the weight, its first rotary_dim values rotated pair by pair."""
    x = x.float()
    x = x * (x.square().mean(-1, keepdim=True) + _EPS).rsqrt() * weight.float()
    rd = case["rotary_dim"]
    c, sn = cos_sin[:, None, :rd // 2], cos_sin[:, None, rd // 2:]
    if case["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([turned, x[..., rd:]], -1)


def _plain_quantise(x):
    """x [T, H, 256] as int8 and scale = largest magnitude / 127 per (token, head)."""
    most = x.abs().amax(-1, keepdim=True)
    scale = most / torch.full_like(most, 127.0)
    return (x / torch.where(scale > 0, scale, 1.0)).round().clamp(-127, 127).to(torch.int8), scale[..., 0]


def _plain_write(s, query, query_out):
    case, bs = s["case"], s["case"]["block_size"]
    cos_sin = s["cos_sin"][s["positions"]]
    query_out.copy_(_plain_head(case, query, s["query_weight"], cos_sin))
    page, at = s["slots"] // bs, s["slots"] % bs
    s["key_cache"][page, at, :, :_DIM], s["k_scale"][page, at] = _plain_quantise(_plain_head(case, s["key"], s["key_weight"], cos_sin))
    s["value_cache"][page, at, :, :_DIM], s["v_scale"][page, at] = _plain_quantise(s["value"].float())


def _count(pages, entries):
    """How many of the entries name each page (those below 0 none)."""
    named = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    named.index_add_(0, torch.where(entries < 0, pages, entries).reshape(-1).long(),
                     torch.ones(entries.numel(), dtype=torch.int32, device="cuda"))
    return named[:pages]


def _plain_fork(s):
    case, refs, old = s["case"], s["refs"], s["block_table"]
    bs, window, sinks, grow, pages = case["block_size"], case["window"], case["sinks"], case["grow"], refs.numel()
    parents = s["parents"].long() if s["parents"] is not None else torch.arange(old.shape[0], device="cuda")
    live = parents >= 0
    p = parents.clamp(min=0)
    child = torch.arange(p.numel(), device="cuda")
    eldest = torch.full((old.shape[0] + 1,), p.numel(), device="cuda").scatter_reduce_(
        0, torch.where(live, p, old.shape[0]), child, "amin")
    heir = (live & (eldest[p] == child))[:, None]
    n = torch.where(live, s["seq_lens"].long()[p], 0)[:, None]
    src = torch.where(live[:, None], old[p], -1)
    start = torch.arange(old.shape[1], device="cuda")[None, :] * bs
    keep = start < torch.where(live[:, None], n + grow, 0)
    if window > 0:  # every key of the page lies between the sinks and what the next token sees
        keep = keep & ~((start >= sinks) & (start + bs <= n + 1 - window))
    full = start + bs <= n
    alone = (src >= 0) & (refs[src.clamp(min=0).long()] == 1)
    takes = keep & ~full & heir & alone
    fresh = keep & ~full & ~takes
    rank = fresh.view(-1).cumsum(0).view(fresh.shape) - 1
    free = torch.where(refs <= 0, torch.arange(pages, device="cuda"), pages).sort()[0]
    free = torch.cat([free, torch.full((1,), pages, device="cuda")])
    new = torch.where(keep & full | takes, src, -1)
    taken = free[rank.clamp(min=0, max=pages)]
    new = torch.where(fresh, torch.where(taken < pages, taken, -1).int(), new)
    s["needed"].copy_(fresh.sum())
    s["new_block_table"].copy_(new)
    s["new_seq_lens"].copy_(n[:, 0])
    s["new_refs"].copy_(refs - _count(pages, old) + _count(pages, new))
    moved = fresh & (start < n) & (src >= 0) & (new >= 0)
    a, b = src[moved].long(), new[moved].long()
    filled = (torch.arange(bs, device="cuda")[None, :] < (n - start)[moved][:, None])[:, None, :, None]
    for kv in s["caches"]:
        kv[b] = torch.where(filled, kv[a], kv[b])


def _plain_compact(s):
    refs, old = s["refs"], s["block_table"]
    pages = refs.numel()
    number = torch.arange(pages, device="cuda")
    live = refs > 0
    used = live.sum()
    moves = live & (number >= used)
    holes = torch.where(~live & (number < used), number, pages).sort()[0]
    to = torch.where(moves, holes[(moves.cumsum(0) - 1).clamp(min=0)], number)
    s["places"].copy_(torch.where(live, to, -1))
    s["used"].copy_(used)
    s["new_block_table"].copy_(torch.where(old >= 0, s["places"][old.clamp(min=0).long()], -1))
    s["new_refs"].copy_(torch.zeros_like(refs).scatter_reduce_(0, to, torch.where(live, refs, 0), "amax"))
    a = number[moves]
    b = to[moves]
    for kv in s["caches"]:
        kv[b] = kv[a]


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "decode":
        if own:
            _package().decode(s["q"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
                              s["query_start_loc"], s["out"], _SCALE, *s["seg"], case["seqs"], case["qlen"], s["nsplit"],
                              window=case["window"], causal=case["causal"], sinks=case["sinks"])
        else:
            _plain_decode(s)
        return {"out": s["out"]}
    if kind == "prefill":
        if own:
            _package().forward_window(s["q"], s["key_cache"], s["value_cache"], s["block_table"], s["seq_lens"], _SCALE,
                                      s["query_start_loc"], s["out"], case["window"], sinks=case["sinks"])
        else:
            _plain_prefill(s)
        return {"out": s["out"]}
    if kind == "write":
        query = s["query"]
        out = s["query_out"]
        if out is None:  # (a fresh projection's query, which the call may write over)
            query = out = query.clone()
        if own:
            _package().norm_rotary_cache_write(query, s["key"], s["value"], s["query_weight"], s["key_weight"], s["positions"],
                                               s["cos_sin"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"], s["slots"],
                                               eps=_EPS, interleaved=case["interleaved"], query_out=out)
        else:
            _plain_write(s, query, out)
        return {"query": out, "cache": s["rows"] * s["scales"]}
    if kind == "fork":
        if own:
            _package().fork_pages(s["caches"], s["refs"], s["block_table"], s["seq_lens"], s["parents"], s["new_refs"],
                                  s["new_block_table"], s["new_seq_lens"], s["needed"], grow=case["grow"], window=case["window"],
                                  sinks=case["sinks"])
        else:
            _plain_fork(s)
        return {"table": s["new_block_table"], "lens": s["new_seq_lens"], "refs": s["new_refs"], "needed": s["needed"],
                "caches": s["caches"]}
    if own:
        _package().compact_pages(s["caches"], s["refs"], s["block_table"], s["new_refs"], s["new_block_table"], s["places"], s["used"])
    else:
        _plain_compact(s)
    return {"table": s["new_block_table"], "refs": s["new_refs"], "places": s["places"], "used": s["used"], "caches": s["caches"]}


# ---- what a pass cannot do without ----

def _fork_counts(case):
    """Table entries that a batch's pages need, and part-filled pages that are copied at the least (half of each, on average)."""
    bs, n = case["block_size"], case["seqs"]
    lens = _lengths(n, case["ctx_lo"], case["ctx_hi"], "ctx")
    entries = sum(-(-(x + case["grow"]) // bs) for x in lens)
    copies = 0 if case["step"] else max(0, case["children"] - max(1, n // 4))
    return entries, copies


def work(case):
    hq, hkv, bs = case["heads_q"], case["heads_kv"], case["block_size"]
    page = bs * hkv * _ROW
    if case["kind"] in ("decode", "prefill"):
        window, sinks = case["window"], case["sinks"]
        keys = pairs = entries = tokens = 0
        for new, length in _batch(case):
            lo = _first_seen(case, new, length)
            seen = length - lo + min(sinks, lo)
            keys += seen
            entries += -(-length // bs) - lo // bs + min(-(-sinks // bs), lo // bs)
            tokens += new
            for i in range(new):  # keys of a row: its window's, and the sinks before it
                p = length - new + i
                first = max(0, p - window + 1)
                last = p if case.get("causal", True) else length - 1
                pairs += last - first + 1 + min(sinks, first)
        return {"bytes": keys * hkv * _ROW + 4 * tokens * hq * _DIM + 4 * entries + 8 * case["seqs"], "flops": 4 * _DIM * hq * pairs}
    if case["kind"] == "write":
        t, rd, size = case["tokens"], case["rotary_dim"], 4 if case["dtype"] == "fp32" else 2
        out = size + (2 if case["out"] == "fp16" else size)
        return {"bytes": t * (hq * _DIM * out + hkv * (2 * _DIM * size + _ROW) + 4 * rd + 16) + 2 * _DIM * size,
                "flops": t * (hq + hkv) * (3 * rd + 4 * _DIM)}
    if case["kind"] == "fork":
        entries, copies = _fork_counts(case)
        rows = case["children"]
        return {"bytes": 8 * entries + 8 * rows + copies * case["layers"] * page, "flops": entries}
    live = max(1, int(case["pages"] * case["used"]))
    moves = live * (case["pages"] - live) // case["pages"]  # of pages in no order
    return {"bytes": 2 * moves * case["layers"] * page + 12 * case["pages"] + 8 * live, "flops": 2 * case["pages"]}


# ---- from the definitions, in 64 bits ----

def _exact_attention(case, s):
    hq, hkv, bs, window, sinks = (case[k] for k in ("heads_q", "heads_kv", "block_size", "window", "sinks"))
    g = hq // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    half = lambda rows, j: rows[:, j, :_DIM].double() * rows[:, j, _DIM:].contiguous().view(torch.float32).double()  # noqa: E731
    for b, (new, length) in enumerate(s["batch"]):
        key = torch.arange(length, device="cuda")
        key = key[(key < sinks) | (key >= _first_seen(case, new, length))]
        page = s["block_table"][b].long()[key // bs]
        for h in range(hkv):
            rows = s["kv"][page, h, key % bs].view(-1, 2, _HALF)
            k, v = half(rows, 0).t().contiguous(), half(rows, 1)
            step = max(1, (1 << 26) // (g * key.numel()))
            for t0 in range(0, new, step):
                t = torch.arange(t0, min(new, t0 + step), device="cuda")
                behind = (length - new + t)[:, None] - key[None, :]
                hidden = (behind >= window) & (key[None, :] >= sinks)
                if case.get("causal", True):
                    hidden |= behind < 0
                x = s["q"][s["starts"][b] + t, h * g:(h + 1) * g].double() @ k * _SCALE   # [t, g, K]
                x[hidden[:, None, :].expand_as(x)] = -math.inf
                out[s["starts"][b] + t, h * g:(h + 1) * g] = torch.softmax(x, -1) @ v
    return {"out": out}


def _exact_fork(case, s):
    refs, old, lens = s["refs"].tolist(), s["block_table"].tolist(), s["seq_lens"].tolist()
    bs, window, sinks = case["block_size"], case["window"], case["sinks"]
    parents = s["parents"].tolist() if s["parents"] is not None else list(range(len(old)))
    free = [i for i, r in enumerate(refs) if r <= 0]
    count, caches, met, wanted = list(refs), [kv.clone() for kv in s["caches"]], set(), 0
    for row in old:
        for e in row:
            count[e] -= e >= 0
    table, sizes = [], []
    for p in parents:
        row, n = [-1] * len(old[0]), 0
        if p >= 0:
            n = lens[p]
            for c in range(min(len(row), -(-(n + case["grow"]) // bs))):
                e, end = old[p][c], (c + 1) * bs
                if window > 0 and c * bs >= sinks and end <= n + 1 - window:
                    continue
                if end <= n:
                    row[c] = e
                elif e >= 0 and refs[e] == 1 and p not in met:
                    row[c] = e
                else:
                    row[c] = free[wanted] if wanted < len(free) else -1
                    wanted += 1
                    if e >= 0 and row[c] >= 0 and c * bs < n:
                        for kv in caches:
                            kv[row[c], :, :n - c * bs] = kv[e, :, :n - c * bs]
            met.add(p)
        for e in row:
            count[e] += e >= 0
        table.append(row)
        sizes.append(n)
    whole = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return {"table": whole(table), "lens": whole(sizes), "refs": whole(count), "needed": whole([wanted]), "caches": caches}


def _exact_compact(case, s):
    refs, caches = s["refs"].tolist(), [kv.clone() for kv in s["caches"]]
    live = [i for i, r in enumerate(refs) if r > 0]
    places = [-1] * len(refs)
    holes = iter([i for i in range(len(live)) if refs[i] <= 0])
    for i in live:
        places[i] = i if i < len(live) else next(holes)
        if places[i] != i:
            for kv in caches:
                kv[places[i]] = kv[i]
    counts = [0] * len(refs)
    for i in live:
        counts[places[i]] = refs[i]
    table = [[places[e] if e >= 0 else -1 for e in row] for row in s["block_table"].tolist()]
    whole = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return {"table": whole(table), "refs": whole(counts), "places": whole(places), "used": whole([len(live)]), "caches": caches}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("decode", "prefill"):
        return _exact_attention(case, s)
    if case["kind"] == "fork":
        return _exact_fork(case, s)
    if case["kind"] == "compact":
        return _exact_compact(case, s)
    rd = case["rotary_dim"]
    # pair j of the head is (x, y); (x + iy) times (cos + i sin)
    first = torch.arange(rd // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else rd // 2)
    turn = torch.complex(*s["cos_sin"].double()[s["positions"]].view(-1, 1, 2, rd // 2).unbind(2))
    q = s["query"].double()
    q = q / ((q ** 2).sum(-1, keepdim=True) / _DIM + _EPS).sqrt() * s["query_weight"].double()
    z = torch.complex(q[..., first], q[..., second]) * turn
    q[..., first], q[..., second] = z.real, z.imag
    return {"query": q, "cache": None}  # the cache's bytes come of a rounding to whole steps
