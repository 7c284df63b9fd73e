"""The operators around one decode or prefill step over the int8 paged KV cache, as measurable cases.

  shared   decode attention of a batch whose sequences share a long prefix: the prefix keys are read
           once for the whole batch, each sequence's own keys once for it, and the two softmax parts
           are joined (decode_shared).
  write    rotary positions on the query and key heads of the new tokens, the rotated keys and the
           values quantised into the cache rows (rotary_cache_write).
  weights  the softmax weight that a decode step's rows gave each cached key, added to the running sums
           of the sequence and kv head (key_weights).
  evict    per sequence and kv head the recent keys and those with the largest sums are kept, their rows
           copied into other blocks (evict).

Sizes are those of this repository's benchmark and tests: 24 q / 4 kv heads (the whole model on one
GPU) and 12 / 2 (one of two tensor-parallel ranks), head size 256, block sizes 16 to 1,584, contexts
of up to 61,440 keys, 1 to 8 query tokens per decoded sequence, prompts of up to 32,768 tokens.

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


def _package():
    name = "mi50_vllm_lab_amd"
    if name not in sys.modules:
        d = os.path.join(_ROOT, "mi50-vllm-lab_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        sys.modules[name] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _shared(name, **kw):
    c = {"name": name, "kind": "shared", "heads_q": 24, "heads_kv": 4, "block_size": 16, "layout": "HND", "outliers": 0.0}
    c.update(kw)
    return c


def _rotary(name, **kw):
    c = {"name": name, "kind": "write", "heads_q": 24, "heads_kv": 4, "block_size": 16, "layout": "HND", "dtype": "fp16",
         "rotary_dim": 256, "interleaved": False, "prompt": True}
    c.update(kw)
    return c


def _weights(name, **kw):
    c = {"name": name, "kind": "weights", "heads_q": 24, "heads_kv": 4, "block_size": 16, "layout": "HND"}
    c.update(kw)
    return c


def _evict(name, **kw):
    c = {"name": name, "kind": "evict", "heads_q": 24, "heads_kv": 4, "block_size": 16, "layout": "HND"}
    c.update(kw)
    return c


def listed():
    return [
        # a few samples of one short prompt: launches and latency are what is left
        _shared("shared_4x1_2k", seqs=4, qlen=1, prefix=2048, own_lo=16, own_hi=300),
        # a chat service's system prompt and examples, conversations of different lengths
        _shared("shared_32x1_8k", seqs=32, qlen=1, prefix=8192, own_lo=100, own_hi=2000),
        # multi-token verification on one rank's heads, the reference's block size
        _shared("shared_16x4_15k_rank", seqs=16, qlen=4, prefix=15840, own_lo=200, own_hi=4000, heads_q=12, heads_kv=2,
                block_size=1584),
        # odd sizes: three tokens each, a prefix that ends inside a block, short own parts, tokens-major blocks, outliers
        _shared("shared_7x3_odd", seqs=7, qlen=3, prefix=1111, own_lo=3, own_hi=500, layout="NHD", outliers=0.01),
        # the largest: a full batch of questions about one document of the benchmark's context
        _shared("shared_128x1_61k", seqs=128, qlen=1, prefix=61440, own_lo=64, own_hi=2048),
        # one user's decode step, a quarter of the head rotated: launch latency
        _rotary("write_1tok_part", tokens=1, rotary_dim=64, prompt=False, out="inplace"),
        # a decode batch of a bf16 model, queries handed on in the decode operator's fp16
        _rotary("write_batch129_bf16", tokens=129, dtype="bf16", prompt=False, out="fp16"),
        # a long prompt on one rank's heads, adjacent pairs, the reference's block size
        _rotary("write_32k_pairs_rank", tokens=32768, interleaved=True, heads_q=12, heads_kv=2, block_size=1584, out="same"),
        # a decode batch that keeps its sums from step to step
        _weights("weights_16x1_8k", seqs=16, qlen=1, ctx_lo=500, ctx_hi=8192),
        # multi-token verification over the benchmark's context
        _weights("weights_1x4_61k", seqs=1, qlen=4, ctx_lo=61440, ctx_hi=61440),
        # a batch held to a budget of 2,048 keys each; one sequence is still below it
        _evict("evict_8_to_2k", seqs=8, ctx_lo=1000, ctx_hi=6000, keep=2048, recent=128),
        # a long prompt's keys cut down to an eighth, on one rank's heads
        _evict("evict_61k_to_8k_rank", seqs=1, ctx_lo=61440, ctx_hi=61440, keep=8000, recent=500, heads_q=12, heads_kv=2,
               block_size=1584, layout="NHD"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges; none costs more than shared_128x1_61k."""
    hq, hkv = rng.choice([(24, 4), (24, 4), (12, 2)])
    common = {"heads_q": hq, "heads_kv": hkv, "block_size": rng.choice([16, 16, 32, 1584]),
              "layout": rng.choice(["HND", "HND", "NHD"])}
    kind = rng.choice(["shared", "shared", "shared", "write", "write", "weights", "evict"])
    if kind == "shared":
        seqs = _log_int(rng, 2, 128)
        qlen = rng.choice([1, 1, 2, 4, 8])
        prefix = _log_int(rng, 64, min(61440, 100 * 61440 // (seqs * qlen)))
        if rng.random() < 0.7:  # blocks are shared whole, as an engine shares them
            prefix = max(common["block_size"], prefix // common["block_size"] * common["block_size"])
        hi = _log_int(rng, 8, min(8192, 200000 // seqs))
        c = _shared("", seqs=seqs, qlen=qlen, prefix=prefix, own_lo=max(1, hi // rng.choice([1, 8, 64])), own_hi=hi,
                    outliers=rng.choice([0.0, 0.0, 0.01]), **common)
    elif kind == "write":
        c = _rotary("", tokens=_log_int(rng, 1, 32768), dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]),
                    rotary_dim=rng.choice([256, 256, 128, 64, 32, 96, 200]), interleaved=rng.random() < 0.4,
                    prompt=rng.random() < 0.5, out=rng.choice(["inplace", "same", "fp16"]), **common)
    elif kind == "weights":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 20, min(61440, 131072 // seqs))
        c = _weights("", seqs=seqs, qlen=rng.choice([1, 1, 2, 4, 8]), ctx_lo=max(1, hi // rng.choice([1, 8, 64])), ctx_hi=hi,
                     **common)
    else:
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 100, min(61440, 131072 // seqs))
        keep = max(8, int(hi * rng.choice([0.1, 0.3, 0.6, 0.97])))
        c = _evict("", seqs=seqs, ctx_lo=max(1, hi // rng.choice([1, 2, 16])), ctx_hi=hi, keep=keep,
                   recent=rng.choice([0, 1, keep // 8, keep // 2]), **common)
    del c["name"]
    return c


# ---- inputs, from the seed alone ----

def _lengths(case, lo, hi):
    """A length for each sequence, evenly spread over their logarithm, in an order fixed by the case."""
    n = case["seqs"]
    a, b = math.log(lo), math.log(hi)
    out = [int(round(math.exp(a + (b - a) * i / (n - 1)))) for i in range(n)] if n > 1 else [hi]
    random.Random("lengths %d %d" % (n, hi)).shuffle(out)
    return out


def _own_lengths(case):
    """Keys of each sequence behind the prefix and before its query tokens."""
    return _lengths(case, case["own_lo"], case["own_hi"])


def _rand_rows(gen, rows, outliers):
    """int8 cache rows [rows, 520] of K, V ~ N(0, 1) (a share `outliers` of them times 50)."""
    kv = torch.empty((rows, _ROW), dtype=torch.int8, device="cuda")
    step = 1 << 18
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = torch.randn((n, 2, _DIM), device="cuda", generator=gen)
        if outliers:
            x *= torch.where(torch.rand((n, 2, 1), device="cuda", generator=gen) < outliers, 50.0, 1.0)
        s = x.abs().amax(-1, keepdim=True) / 127.0
        kv[r:r + n].view(n, 2, _HALF)[:, :, :_DIM] = (x / s).round_().clamp_(-127, 127).to(torch.int8)
        kv[r:r + n].view(n, 2, _HALF)[:, :, _DIM:] = s.view(torch.int8).view(n, 2, 4)
    return kv


def _cache(case, kv):
    """The operators' views of a raw cache [blocks, Hkv, block_size, 520]: int8 [blocks, block_size, Hkv, 260] for K and
    V, fp32 [blocks, block_size, Hkv] for their scales; and all int8 values and scales as [blocks, Hkv, block_size, 2, ..]."""
    f32 = torch.tensor([], dtype=torch.float32, device="cuda").set_(kv.untyped_storage())
    nblk, hkv, bs, _ = kv.shape
    st = [x // 4 for x in kv.stride()]
    key, value = kv.transpose(1, 2).split(_HALF, dim=-1)
    ks, vs = (torch.as_strided(f32, (nblk, bs, hkv), (st[0], st[2], st[1]), o) for o in (_DIM // 4, (_HALF + _DIM) // 4))
    rows = torch.as_strided(kv, (nblk, hkv, bs, 2, _DIM), (*kv.stride()[:3], _HALF, 1))
    scales = torch.as_strided(f32, (nblk, hkv, bs, 2, 1), (*st[:3], _HALF // 4, 1), _DIM // 4)
    return {"kv": kv, "key_cache": key, "value_cache": value, "k_scale": ks, "v_scale": vs, "rows": rows, "scales": scales}


def _blocks(case, pages, rows):
    shape = (pages, case["heads_kv"], case["block_size"], _ROW) if case["layout"] == "HND" else \
        (pages, case["block_size"], case["heads_kv"], _ROW)
    kv = rows.view(shape)
    return kv if case["layout"] == "HND" else kv.transpose(1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    hq, hkv, bs = case["heads_q"], case["heads_kv"], case["block_size"]
    s = {"case": case}
    if case["kind"] == "shared":
        n, p, new = case["seqs"], case["prefix"], case["qlen"]
        lens = [p + c + new for c in _own_lengths(case)]
        whole = p // bs                      # blocks that every table names
        per = [-(-x // bs) - whole for x in lens]
        pages = whole + sum(per) + 2
        perm = torch.randperm(pages, generator=host).to(torch.int32)
        bt = torch.zeros((n, whole + max(per)), dtype=torch.int32)
        bt[:, :whole] = perm[:whole]
        at = whole
        for b, m in enumerate(per):
            bt[b, whole:whole + m] = perm[at:at + m]
            at += m
        kv = _blocks(case, pages, _rand_rows(gen, pages * bs * hkv, case["outliers"]))
        for b in range(1, n):  # a block that the prefix ends in: the sequences' own copies agree on its keys
            if p % bs:
                kv[int(bt[b, whole]), :, :p % bs] = kv[int(bt[0, whole]), :, :p % bs]
        s.update(_cache(case, kv))
        s["q"] = torch.randn((n * new, hq, _DIM), device="cuda", generator=gen).half()
        s["out"] = torch.zeros_like(s["q"])
        s["block_table"], s["seq_lens"] = bt.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["query_start_loc"] = torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda")
        s["seg"] = [torch.empty((n * new, hq, 64) + d, device="cuda") for d in ((_DIM,), (), ())]
        # what the plain form counts by: the prefix's positions, the longest own part's, and each query token's place
        s["prefix_pos"] = torch.arange(p, device="cuda")
        s["own_pos"] = torch.arange(p, max(lens), device="cuda")
        s["tok"] = torch.arange(new, device="cuda")
        return s
    if case["kind"] == "write":
        t, dt, rd = case["tokens"], _DTYPES[case["dtype"]], case["rotary_dim"]
        qkv = torch.randn((t, (hq + 2 * hkv) * _DIM), device="cuda", generator=gen).to(dt)
        heads = qkv.view(t, hq + 2 * hkv, _DIM)
        s["query"], s["key"], s["value"] = heads[:, :hq], heads[:, hq:hq + hkv], heads[:, hq + hkv:]
        angle = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * \
            _BASE ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)[None, :]
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float()
        first = int(torch.randint(0, _POSITIONS - t, (1,), generator=host))
        s["positions"] = torch.arange(first, first + t, device="cuda") if case["prompt"] else \
            torch.randint(0, _POSITIONS, (t,), generator=host).cuda()
        pages = -(-t // bs) + 1
        slots = (torch.randperm(pages, generator=host)[:, None] * bs + torch.arange(bs)[None, :]).reshape(-1)[:t]
        s["slots"] = slots.cuda()
        s.update(_cache(case, _blocks(case, pages, torch.zeros((pages * bs * hkv, _ROW), dtype=torch.int8, device="cuda"))))
        out = {"inplace": None, "same": dt, "fp16": torch.float16}[case["out"]]
        s["query_out"] = s["query"] if out is None else torch.empty((t, hq, _DIM), dtype=out, device="cuda")
        return s
    n, new = case["seqs"], case.get("qlen", 0)
    lens = [c + new for c in _lengths(case, case["ctx_lo"], case["ctx_hi"])]
    per = [-(-x // bs) for x in lens]
    keep = case.get("keep", 0)
    fresh = n * -(-keep // bs)  # blocks that the kept rows go to, behind the others
    pages = sum(per) + 2
    perm = torch.randperm(pages, generator=host).to(torch.int32)
    bt = torch.zeros((n, max(per)), dtype=torch.int32)
    at = 0
    for b, m in enumerate(per):
        bt[b, :m] = perm[at:at + m]
        at += m
    s.update(_cache(case, _blocks(case, pages + fresh + 1, _rand_rows(gen, (pages + fresh + 1) * bs * hkv, 0.0))))
    s["block_table"], s["seq_lens"] = bt.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["pos"] = torch.arange(max(lens), device="cuda")
    if case["kind"] == "weights":
        s["q"] = torch.randn((n * new, hq, _DIM), device="cuda", generator=gen).half()
        s["query_start_loc"] = torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda")
        s["tok"] = torch.arange(new, device="cuda")
        s["lse"] = torch.cat([_row_sums(s, b, length).log().float() for b, length in enumerate(lens)])
        s["weights"] = torch.rand((n, hkv, max(lens)), device="cuda", generator=gen).pow_(8)
    else:
        # sums as they grow over many steps: a few large ones, a long tail, a part that no row has seen yet
        w = torch.randn((n, hkv, max(lens)), device="cuda", generator=gen).mul_(2).exp_()
        s["weights"] = torch.where(torch.rand(w.shape, device="cuda", generator=gen) < 0.2, 0.0, w)
        to = (torch.randperm(fresh, generator=host) + pages).to(torch.int32)
        s["new_block_table"] = to.view(n, -1).cuda()
        s["new_seq_lens"] = torch.zeros_like(s["seq_lens"])
        s["new_weights"] = torch.zeros((n, hkv, keep), device="cuda")
        s["kept"] = torch.zeros((n, hkv, keep), dtype=torch.int32, device="cuda")
        s["dump"] = pages + fresh  # where the plain form puts what a short sequence does not have
        s["kv"][s["dump"] - fresh:].zero_()
        s["new_rows"] = s["kv"][pages:pages + fresh]
        s["heads"], s["place"] = torch.arange(hkv, device="cuda"), torch.arange(keep, device="cuda")
    return s


def _row_sums(s, b, length):
    """The softmax sums of one sequence's rows [new, Hq], in 64 bits (an engine has their logarithms from its decode)."""
    case = s["case"]
    new, hkv, bs = case["qlen"], case["heads_kv"], case["block_size"]
    pos = torch.arange(length, device="cuda")
    page, at = s["block_table"][b].long()[pos // bs], pos % bs
    k = s["key_cache"][page, at, :, :_DIM].double() * s["k_scale"][page, at].double()[..., None]   # [S, Hkv, 256]
    q = s["q"][b * new:(b + 1) * new].double().view(new, hkv, -1, _DIM).transpose(0, 1).reshape(hkv, -1, _DIM)
    x = (q @ k.permute(1, 2, 0).contiguous()).mul_(_SCALE).exp_().view(hkv, new, -1, length)
    seen = pos[None, :] <= (length - new + s["tok"])[:, None]
    return (x * seen[None, :, None, :]).sum(-1).transpose(0, 1).reshape(new, -1)


# ---- the operators ----

def _plain_shared(s):
    """Scores of all query tokens against the prefix as one product per kv head, against the own keys as one per
    sequence (padded to the longest, masked behind each token's position), the two parts joined by their row
    maxima and sums."""
    case = s["case"]
    n, new, hq, hkv, bs, p = (case[k] for k in ("seqs", "qlen", "heads_q", "heads_kv", "block_size", "prefix"))
    g = hq // hkv
    keys = lambda cache, scale, page, at: cache[page, at, :, :_DIM].float() * scale[page, at][..., None]  # noqa: E731
    q = s["q"].float().view(n, new, hkv, g, _DIM) * _SCALE
    page, at = s["block_table"][0].long()[s["prefix_pos"] // bs], s["prefix_pos"] % bs
    k = keys(s["key_cache"], s["k_scale"], page, at).permute(1, 2, 0).contiguous()         # [Hkv, 256, P]
    v = keys(s["value_cache"], s["v_scale"], page, at).transpose(0, 1).contiguous()        # [Hkv, P, 256]
    x = q.permute(2, 0, 1, 3, 4).reshape(hkv, n * new * g, _DIM) @ k
    m1 = x.amax(-1, keepdim=True)
    x = (x - m1).exp_()
    l1, o1 = x.sum(-1, keepdim=True), x @ v
    m1, l1, o1 = (y.view(hkv, n, new * g, -1).transpose(0, 1) for y in (m1, l1, o1))         # [n, Hkv, new G, ..]
    live = s["own_pos"][None, :] < s["seq_lens"][:, None]
    last = torch.where(live, s["own_pos"][None, :], s["seq_lens"][:, None] - 1)              # a key of the sequence's own
    page = torch.gather(s["block_table"].long(), 1, last // bs)
    k = keys(s["key_cache"], s["k_scale"], page, last % bs).permute(0, 2, 3, 1).contiguous()
    v = keys(s["value_cache"], s["v_scale"], page, last % bs).transpose(1, 2).contiguous()   # [n, Hkv, S, 256]
    x = q.permute(0, 2, 1, 3, 4).reshape(n, hkv, new * g, _DIM) @ k
    seen = s["own_pos"][None, None, :] <= (s["seq_lens"][:, None] - new + s["tok"][None, :])[:, :, None]  # [n, new, S]
    x = x.view(n, hkv, new, g, -1).masked_fill(~seen[:, None, :, None, :], -math.inf).view(n, hkv, new * g, -1)
    m = torch.maximum(x.amax(-1, keepdim=True), m1)
    x = (x - m).exp_()
    w = (m1 - m).exp()
    o = (x @ v + w * o1) / (x.sum(-1, keepdim=True) + w * l1)
    return o.view(n, hkv, new, g, _DIM).transpose(1, 2).reshape(n * new, hq, _DIM).half()


def _plain_rotate(case, x, cos_sin):
    """x [T, H, 256] in 32 bits with its first rotary_dim values rotated by the tokens' angles, pair by pair."""
    rd = case["rotary_dim"]
    c, sn = cos_sin[:, None, :rd // 2], cos_sin[:, None, rd // 2:]
    x = x.float()
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


def _plain_write(s):
    case, bs = s["case"], s["case"]["block_size"]
    cos_sin = s["cos_sin"][s["positions"]]
    s["query_out"].copy_(_plain_rotate(case, s["query"], cos_sin))
    page, at = s["slots"] // bs, s["slots"] % bs
    s["key_cache"][page, at, :, :_DIM], s["k_scale"][page, at] = _plain_quantise(_plain_rotate(case, s["key"], cos_sin))
    s["value_cache"][page, at, :, :_DIM], s["v_scale"][page, at] = _plain_quantise(s["value"].float())


def _plain_weights(s):
    """Scores of each sequence's rows against its keys (padded to the longest), e to the score less the row's
    logarithm, summed over the rows of the kv head."""
    case = s["case"]
    n, new, hq, hkv, bs = (case[k] for k in ("seqs", "qlen", "heads_q", "heads_kv", "block_size"))
    g = hq // hkv
    last = torch.minimum(s["pos"][None, :], s["seq_lens"][:, None] - 1).long()
    page = torch.gather(s["block_table"].long(), 1, last // bs)
    k = s["key_cache"][page, last % bs, :, :_DIM].float() * s["k_scale"][page, last % bs][..., None]
    q = s["q"].float().view(n, new, hkv, g, _DIM).mul(_SCALE).transpose(1, 2).reshape(n, hkv, new * g, _DIM)
    x = (q @ k.permute(0, 2, 3, 1).contiguous()).view(n, hkv, new, g, -1)
    x = (x - s["lse"].view(n, new, hkv, g, 1).transpose(1, 2)).exp_()
    seen = s["pos"][None, None, :] <= (s["seq_lens"][:, None] - new + s["tok"][None, :])[:, :, None]  # [n, new, S]
    s["weights"].add_(x.mul_(seen[:, None, :, None, :]).sum((2, 3)))


def _plain_evict(s):
    """The keys in the order of their sums, the recent ones first and those behind the end last; the first `keep` of
    them in the order of their positions."""
    case, bs = s["case"], s["case"]["block_size"]
    keep, recent = case["keep"], case["recent"]
    lens = s["seq_lens"][:, None, None]
    w = torch.where(s["pos"] >= lens - recent, math.inf, s["weights"])
    w = torch.where(s["pos"] >= lens, -math.inf, w)
    first = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep]
    pad = max(0, keep - first.shape[-1])
    first = torch.nn.functional.pad(first, (0, pad), value=1 << 30)
    kept = torch.where(first < lens, first, 1 << 30).sort(-1)[0]
    live = kept < lens
    s["kept"].copy_(torch.where(live, kept, -1))
    src = torch.where(live, kept, 0)
    s["new_weights"].copy_(torch.where(live, torch.gather(s["weights"], -1, src), 0.0))
    s["new_seq_lens"].copy_(s["seq_lens"].clamp(max=keep))
    table = s["block_table"].long()[:, None, :].expand(-1, kept.shape[1], -1)
    head = s["heads"][None, :, None]
    to = torch.where(live, s["new_block_table"].long()[:, s["place"] // bs][:, None, :], s["dump"])
    s["kv"][to, head, s["place"] % bs] = s["kv"][torch.gather(table, -1, src // bs), head, src % bs]


def run(state):
    s, case = state, state["case"]
    if case["kind"] == "shared":
        if not own:
            return {"out": _plain_shared(s)}
        _package().decode_shared(s["q"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                 s["seq_lens"], s["query_start_loc"], s["out"], _SCALE, *s["seg"], case["seqs"], case["qlen"],
                                 case["prefix"])
        return {"out": s["out"]}
    if case["kind"] == "write":
        if own:
            _package().rotary_cache_write(s["query"], s["key"], s["value"], s["positions"], s["cos_sin"], s["key_cache"],
                                          s["value_cache"], s["k_scale"], s["v_scale"], s["slots"],
                                          interleaved=case["interleaved"], query_out=s["query_out"])
        else:
            _plain_write(s)
        return {"query": s["query_out"], "cache": s["rows"] * s["scales"]}
    if case["kind"] == "weights":
        if own:
            _package().key_weights(s["q"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                   s["seq_lens"], s["query_start_loc"], s["lse"], s["weights"], _SCALE, case["seqs"],
                                   case["qlen"])
        else:
            _plain_weights(s)
        return {"weights": s["weights"]}
    if own:
        _package().evict(s["weights"], s["key_cache"], s["value_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                         s["seq_lens"], s["new_block_table"], s["new_seq_lens"], s["new_weights"], s["kept"], case["seqs"],
                         case["keep"], case["recent"])
    else:
        _plain_evict(s)
    # (the rows are moved, not computed: their bytes come back as they are)
    return {"kept": s["kept"], "lens": s["new_seq_lens"], "weights": s["new_weights"], "cache": s["new_rows"]}


def work(case):
    hq, hkv, bs = case["heads_q"], case["heads_kv"], case["block_size"]
    if case["kind"] == "shared":
        n, new, p = case["seqs"], case["qlen"], case["prefix"]
        mine = _own_lengths(case)
        keys = p + sum(mine) + n * new
        pairs = sum(new * (p + c) + new * (new + 1) // 2 for c in mine)
        table = 4 * (-(-p // bs) + sum(-(-(p + c + new) // bs) - p // bs for c in mine))
        return {"bytes": keys * hkv * _ROW + 4 * n * new * hq * _DIM + table + 8 * n, "flops": 4 * _DIM * hq * pairs}
    if case["kind"] == "write":
        t, rd, size = case["tokens"], case["rotary_dim"], 4 if case["dtype"] == "fp32" else 2
        out = 2 * rd * size if case["out"] == "inplace" else _DIM * (size + (2 if case["out"] == "fp16" else size))
        return {"bytes": t * (hq * out + hkv * (2 * _DIM * size + _ROW) + 4 * rd + 16), "flops": 3 * t * (hq + hkv) * rd}
    n, new = case["seqs"], case.get("qlen", 0)
    lens = [c + new for c in _lengths(case, case["ctx_lo"], case["ctx_hi"])]
    table = 4 * sum(-(-x // bs) for x in lens) + 8 * n
    if case["kind"] == "weights":  # a key's half of the row, its sum read and written
        pairs = sum(new * (x - new) + new * (new + 1) // 2 for x in lens)
        return {"bytes": sum(lens) * hkv * (_HALF + 8) + n * new * hq * (2 * _DIM + 4) + table, "flops": 2 * _DIM * hq * pairs}
    rows = hkv * sum(min(x, case["keep"]) for x in lens)
    return {"bytes": 4 * hkv * sum(lens) + rows * (2 * _ROW + 8) + table, "flops": hkv * sum(lens)}


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, bs = case["heads_q"], case["heads_kv"], case["block_size"]
    g, new = hq // hkv, case.get("qlen", 0)
    value = lambda rows, j: rows[:, j, :_DIM].double() * rows[:, j, _DIM:].contiguous().view(torch.float32).double()  # noqa: E731
    if case["kind"] in ("shared", "weights"):
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        sums = s["weights"].double() if case["kind"] == "weights" else None
        for h in range(hkv):
            for b, length in enumerate(s["seq_lens"].tolist()):
                pos = torch.arange(length, device="cuda")
                rows = s["kv"][s["block_table"][b].long()[pos // bs], h, pos % bs].view(length, 2, _HALF)
                k, v = value(rows, 0), value(rows, 1) if sums is None else None
                for i in range(new):
                    see = length - new + i + 1
                    x = s["q"][b * new + i, h * g:(h + 1) * g].double() @ k[:see].t().contiguous() * _SCALE
                    if sums is None:
                        out[b * new + i, h * g:(h + 1) * g] = torch.softmax(x, -1) @ v[:see]
                    else:
                        sums[b, h, :see] += (x - s["lse"][b * new + i, h * g:(h + 1) * g].double()[:, None]).exp().sum(0)
        return {"out": out} if sums is None else {"weights": sums}
    if case["kind"] == "write":
        rd = case["rotary_dim"]
        # pair j of the head is (x, y); (x + iy) times (cos + i sin)
        first = torch.arange(rd // 2, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else rd // 2)
        turn = torch.complex(*s["cos_sin"].double()[s["positions"]].view(-1, 1, 2, rd // 2).unbind(2))
        q = s["query"].double()
        z = torch.complex(q[..., first], q[..., second]) * turn
        q[..., first], q[..., second] = z.real, z.imag
        return {"query": q, "cache": None}  # the cache's bytes come of a rounding to whole steps
    kept, weights = s["kept"].cpu().fill_(-1), torch.zeros(s["new_weights"].shape, dtype=torch.float64)
    w = s["weights"].double().cpu()
    for b, length in enumerate(s["seq_lens"].tolist()):
        for h in range(hkv):
            old = max(0, length - case["recent"])
            if length <= case["keep"]:
                chosen = list(range(length))
            else:
                mine = w[b, h, :old].tolist()
                order = sorted(range(old), key=lambda t: (-mine[t], t))
                chosen = sorted(order[:case["keep"] - (length - old)] + list(range(old, length)))
            kept[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            weights[b, h, :len(chosen)] = w[b, h, chosen]
    return {"kept": kept, "lens": None, "weights": weights, "cache": None}
