"""The serving step's operators over the paged cache, as they are measured: page and row maps built
on the GPU from request lengths, attention of a chunk of new tokens over the paged cache, and
products with 4-bit weights at few rows.

``own`` false computes each in its plain form (elementary torch operations in 32 bits); ``own`` true
makes the framework's calls.  Shapes are those of the Qwen3-ASR 0.6B and 1.7B text decoders (16 query
heads over 8 kv heads of 128 dims, pages of 64 positions) and generic ones next to them.
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

PAGE = 64
DIM = 128
DEV = "cuda"


# ---------------------------------------------------------------------------------------- cases
def _attn(name, **kw):
    c = dict(op="attention", n=1, singles=0, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=0, nq=16, nkv=8, layers=1,
             layer=0, pad=0, dtype="f16", mix=1)
    c.update(kw)
    return dict(c, name=name) if name else c


def _w4(name, **kw):
    c = dict(op="w4", n_out=2048, k=2048, group=128, zeros=False, rows=1, dtype="f16", pad=0)
    c.update(kw)
    return dict(c, name=name) if name else c


def _plan(name, **kw):
    c = dict(op="plan", release=False, n=1, slots=1, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=0, mix=1)
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode step of 32 slots: one new position each, a page turned over now and then
        _plan("plan decode 32", n=32, slots=32, ctx_lo=100, ctx_hi=1500),
        # 512 requests admitted at once, whole prompts in front of them: a million row map entries
        _plan("plan admit 512", n=512, slots=512, new_lo=256, new_hi=4096, mix=2),
        # a batch of 300 finished requests gives its pages back
        _plan("release 300", release=True, n=300, slots=512, ctx_lo=100, ctx_hi=4096, mix=3),
        # one speaker, one token: latency alone
        _attn("attn 1 token", ctx_lo=224, ctx_hi=224),
        # the decode step of 32 slots with ragged caches
        _attn("attn decode 32", n=32, ctx_lo=100, ctx_hi=1499, mix=4),
        # a large decode step, half a thousand slots: the cache streams once
        _attn("attn decode 512", n=512, ctx_lo=256, ctx_hi=4095, mix=5),
        # streaming: every live stream appends the 13 tokens of one audio chunk
        _attn("attn append 13", n=64, new_lo=13, new_hi=13, ctx_lo=100, ctx_hi=1500, layers=2, layer=1, mix=6),
        # a mixed step: 24 slots decode while 8 requests are prefilled in chunks, bf16
        _attn("attn mixed bf16", n=32, singles=24, new_lo=200, new_hi=777, ctx_lo=0, ctx_hi=1500, dtype="bf16", mix=7),
        # one long recording's prompt in one piece
        _attn("attn prompt 8192", new_lo=8192, new_hi=8192, mix=8),
        # 0.6B o_proj at one row: the smallest product of a step
        _w4("w4 1024x2048 r1 g32", n_out=1024, k=2048, group=32, rows=1),
        # 1.7B down_proj with zero points for 16 slots, bf16
        _w4("w4 2048x6144 r16", n_out=2048, k=6144, group=64, zeros=True, rows=16, dtype="bf16"),
        # the vocabulary's table as a 4-bit head at one row: bandwidth alone
        _w4("w4 151936x2048 r1", n_out=151936, k=2048, group=128, rows=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "attention", "attention", "w4", "w4"])
    if op == "plan":
        n = _log(rng, 1, 512)
        slots = n + rng.randrange(0, 40)
        if rng.random() < 0.3:
            return _plan(None, release=True, n=n, slots=slots, ctx_lo=rng.randrange(0, 200), ctx_hi=_log(rng, 200, 4096),
                         mix=rng.randrange(1 << 30))
        hi = _log(rng, 1, 2000)
        return _plan(None, n=n, slots=slots, new_lo=rng.randrange(0, hi + 1), new_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 1, 2000),
                     mix=rng.randrange(1 << 30))
    if op == "w4":
        return _w4(None, n_out=_log(rng, 300, 60000), k=128 * _log(rng, 4, 64), group=rng.choice([32, 64, 128]),
                   zeros=rng.random() < 0.5, rows=_log(rng, 1, 32), dtype=rng.choice(["f16", "bf16"]),
                   pad=8 * rng.randrange(0, 3))
    nq, nkv = rng.choice([(16, 8), (16, 8), (16, 8), (16, 2), (8, 8), (12, 4), (20, 4)])
    kind = rng.choice(["decode", "chunk", "mixed"])
    hi = 1 if kind == "decode" else _log(rng, 2, 1500)
    ctx = _log(rng, 16, 4096)
    n = _log(rng, 1, max(2, min(256, int(4e8 / (nq * hi * (hi + ctx))))))
    return _attn(None, n=n, singles=n // 2 if kind == "mixed" else 0, new_lo=max(1, hi // 3), new_hi=hi, ctx_lo=ctx // 4,
                 ctx_hi=ctx, nq=nq, nkv=nkv, layers=rng.choice([1, 2]), layer=0, pad=8 * rng.randrange(0, 3),
                 dtype=rng.choice(["f16", "bf16"]), mix=rng.randrange(1 << 30))


def _lens(case):
    """(positions cached before, new positions) of each request; they are the case's, not the seed's."""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["n"]):
        new = 1 if i < case.get("singles", 0) else rng.randint(case["new_lo"], case["new_hi"])
        got.append((rng.randint(case["ctx_lo"], case["ctx_hi"]), new))
    return got


def _pages(n):
    return -(-n // PAGE)


# ---------------------------------------------------------------------------------------- inputs
def _package():
    if "qasr_b200" in sys.modules:
        return sys.modules["qasr_b200"]
    at = Path(__file__).resolve().parents[1] / "qwen3-asr-wgpu_b200"
    spec = importlib.util.spec_from_file_location("qasr_b200", at / "__init__.py", submodule_search_locations=[str(at)])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["qasr_b200"] = mod
    spec.loader.exec_module(mod)
    return mod


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 13)
    return {"plan": _prepare_plan, "attention": _prepare_attention, "w4": _prepare_w4}[case["op"]](case, seed, g)


def _prepare_plan(case, seed, g):
    lens = _lens(case)
    n, slots, release = case["n"], case["slots"], case["release"]
    max_pages = max(1, max(_pages(a + (0 if release else b)) for a, b in lens))
    held = [_pages(a) for a, _ in lens]
    need = [0 if release else _pages(a + b) - _pages(a) for a, b in lens]
    pool_pages = sum(held) + sum(need) + 17
    # an allocator in the middle of its life: pages handed out in no particular order
    order = torch.randperm(pool_pages, generator=g, device=DEV, dtype=torch.int32)
    slot = torch.randperm(slots, generator=g, device=DEV)[:n].to(torch.int32)
    table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=DEV)
    held_t = torch.tensor(held, device=DEV)
    i = torch.repeat_interleave(torch.arange(n, device=DEV), held_t)
    j = torch.arange(sum(held), device=DEV) - (held_t.cumsum(0) - held_t)[i]
    table[slot.long()[i], j] = order[: sum(held)]
    free = torch.zeros(pool_pages, dtype=torch.int32, device=DEV)
    count = pool_pages - sum(held)
    free[:count] = order[sum(held):]
    rows = 0 if release else sum(b for _, b in lens)
    e = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(case=case, slot=slot, kv_len=_ints([a for a, _ in lens]), new_len=_ints([b for _, b in lens]), table=table,
                free=free, count=_ints([count]), rows=rows, max_pages=max_pages, pool_pages=pool_pages, slots=slots, n=n,
                kv_len_out=e(n), count_out=e(1), cu=e(n + 1), row_slot=e(max(1, rows)), row_pos=e(max(1, rows)), status=e(2))


def _prepare_attention(case, seed, g):
    lens, t = _lens(case), _type(case)
    n, nq, nkv, layers = case["n"], case["nq"], case["nkv"], case["layers"]
    total = [a + b for a, b in lens]
    max_pages = max(_pages(x) for x in total)
    pool_pages = sum(_pages(x) for x in total) + 3
    # scores of a q-normed, k-normed decoder: unit spread and somewhat above
    pool = torch.empty((pool_pages, layers, 2, nkv, PAGE, DIM), dtype=t, device=DEV)
    for part in pool.split(max(1, (1 << 27) // pool[0].numel())):
        part.normal_(generator=g)
    slot = torch.randperm(n + 2, generator=g, device=DEV)[:n].to(torch.int32)
    order = torch.randperm(pool_pages, generator=g, device=DEV, dtype=torch.int32)
    table = torch.full((n + 2, max_pages), pool_pages, dtype=torch.int32, device=DEV)
    counts = torch.tensor([_pages(x) for x in total], device=DEV)
    i = torch.repeat_interleave(torch.arange(n, device=DEV), counts)
    table[slot.long()[i], torch.arange(int(counts.sum()), device=DEV) - (counts.cumsum(0) - counts)[i]] = order[: int(counts.sum())]
    rows = sum(b for _, b in lens)
    ld = nq * DIM + case["pad"]
    q = torch.empty((rows, ld), dtype=t, device=DEV).normal_(0.0, 1.5, generator=g)
    cu = [0]
    for _, b in lens:
        cu.append(cu[-1] + b)
    s = dict(case=case, q=q, ld=ld, rows=rows, pool=pool, pool_pages=pool_pages, table=table, slots=n + 2, max_pages=max_pages,
             slot=slot, cu=_ints(cu), kv_len=_ints(total), n=n, max_new=max(b for _, b in lens), max_kv=max(total),
             out=torch.zeros((rows, nq * DIM), dtype=t, device=DEV), type=t)
    if own:  # the workspace that a program keeps for its stream
        q_ = _package()
        s["ws_bytes"] = q_.kernel_attention_chunk_workspace(0)
        s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device=DEV)
    return s


def _prepare_w4(case, seed, g):
    n_out, k, group, rows, t = case["n_out"], case["k"], case["group"], case["rows"], _type(case)
    codes = torch.randint(0, 256, (n_out, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    scale = (torch.rand((n_out, k // group), device=DEV, generator=g) * 0.006 + 0.002).to(torch.float16)
    zero = torch.randint(4, 12, (n_out, k // group), dtype=torch.uint8, device=DEV, generator=g) if case["zeros"] else None
    ldx = k + case["pad"]
    x = torch.empty((rows, ldx), dtype=t, device=DEV).normal_(generator=g)
    s = dict(case=case, codes=codes, scale=scale, zero=zero, x=x, ldx=ldx, out=torch.zeros((rows, n_out), dtype=t, device=DEV),
             type=t)
    if own:  # the weights laid out once, as a program keeps them
        q_ = _package()
        s["packed"] = torch.empty(q_.kernel_w4_packed_bytes(n_out, k, group, zero is not None), dtype=torch.uint8, device=DEV)
        q_.kernel_pack_w4(0, torch.cuda.current_stream().cuda_stream, codes.data_ptr(), scale.data_ptr(),
                          zero.data_ptr() if zero is not None else None, n_out, k, group, s["packed"].data_ptr())
    return s


# ---------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "attention": _own_attention, "w4": _own_w4}[op](state)
    return {"plan": _plain_plan, "attention": _plain_attention, "w4": _plain_w4}[op](state)


def _own_plan(s):
    q, st = _package(), torch.cuda.current_stream().cuda_stream
    if s["case"]["release"]:
        q.kernel_kv_release(0, st, s["slot"].data_ptr(), s["kv_len"].data_ptr(), s["n"], s["slots"], s["table"].data_ptr(),
                            s["max_pages"], s["free"].data_ptr(), s["pool_pages"], s["count"].data_ptr(),
                            s["kv_len_out"].data_ptr(), s["count_out"].data_ptr(), s["status"].data_ptr())
        return s["free"], s["kv_len_out"], s["count_out"], s["status"]
    q.kernel_kv_plan(0, st, s["slot"].data_ptr(), s["kv_len"].data_ptr(), s["new_len"].data_ptr(), s["n"], s["slots"],
                     s["table"].data_ptr(), s["max_pages"], s["free"].data_ptr(), s["pool_pages"], s["count"].data_ptr(),
                     s["kv_len_out"].data_ptr(), s["count_out"].data_ptr(), s["cu"].data_ptr(), s["row_slot"].data_ptr(),
                     s["row_pos"].data_ptr(), s["rows"], s["status"].data_ptr())
    return s["table"], s["kv_len_out"], s["count_out"], s["cu"], s["row_slot"], s["row_pos"], s["status"]


def _own_attention(s):
    q, st, c = _package(), torch.cuda.current_stream().cuda_stream, s["case"]
    q.kernel_attention_chunk(0, st, q.TYPE_BF16 if s["type"] is torch.bfloat16 else q.TYPE_F16, s["q"].data_ptr(), s["ld"],
                             s["out"].data_ptr(), c["nq"] * DIM, s["rows"], s["pool"].data_ptr(), s["pool_pages"],
                             s["table"].data_ptr(), s["slots"], s["max_pages"], c["layers"], c["nq"], c["nkv"], c["layer"],
                             s["slot"].data_ptr(), s["cu"].data_ptr(), s["kv_len"].data_ptr(), s["n"], s["ws"].data_ptr(),
                             s["ws_bytes"])
    return s["out"]


def _own_w4(s):
    q, st, c = _package(), torch.cuda.current_stream().cuda_stream, s["case"]
    q.kernel_gemv_w4(0, st, q.TYPE_BF16 if s["type"] is torch.bfloat16 else q.TYPE_F16, s["packed"].data_ptr(), c["zeros"],
                     c["n_out"], c["k"], c["group"], s["x"].data_ptr(), s["ldx"], c["rows"], s["out"].data_ptr(), c["n_out"])
    return s["out"]


def _plain_plan(s):
    n, dev = s["n"], s["slot"].device
    a, slot = s["kv_len"].long(), s["slot"].long()
    have = (a + PAGE - 1) // PAGE
    seq = torch.arange(n, device=dev)
    status = torch.zeros(2, dtype=torch.int32, device=dev)
    if s["case"]["release"]:
        total = int(have.sum())
        i = torch.repeat_interleave(seq, have, output_size=total)
        j = torch.arange(total, device=dev)
        first = have.cumsum(0) - have
        s["free"][s["count"].long() + j] = s["table"][slot[i], j - first[i]]
        return s["free"], torch.zeros_like(s["kv_len"]), (s["count"] + total).to(torch.int32), status
    new = s["new_len"].long()
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), new.cumsum(0)])
    i = torch.repeat_interleave(seq, new, output_size=s["rows"])
    row_slot = s["slot"][i]
    row_pos = a[i] + torch.arange(s["rows"], device=dev) - cu[i]
    need = (a + new + PAGE - 1) // PAGE - have
    total = int(need.sum())
    p = torch.repeat_interleave(seq, need, output_size=total)
    j = torch.arange(total, device=dev)
    first = need.cumsum(0) - need
    s["table"][slot[p], have[p] + j - first[p]] = s["free"][s["count"].long() - 1 - j]
    if not s["rows"]:
        row_slot, row_pos = s["row_slot"], s["row_pos"]
    return (s["table"], (a + new).to(torch.int32), (s["count"] - total).to(torch.int32), cu.to(torch.int32), row_slot,
            row_pos.to(torch.int32), status)


def _columns(dev):
    """Where dim d of position p of a page stands in its row: 16-byte chunks permuted by the position's low 3 bits."""
    p, d = torch.arange(PAGE, device=dev)[:, None], torch.arange(DIM, device=dev)[None, :]
    return (((d >> 3) ^ (p & 7)) << 3) | (d & 7)


def _plain_attention(s):
    c, dev = s["case"], s["q"].device
    n, nq, nkv, S, T = s["n"], c["nq"], c["nkv"], s["max_new"], s["max_kv"]
    pages = s["table"][s["slot"].long()][:, : _pages(T)].long().clamp(0, s["pool_pages"] - 1)
    kv = s["pool"][pages, c["layer"]].float()  # [n, pages, 2, nkv, 64, 128]
    kv = torch.gather(kv, 5, _columns(dev).expand(kv.shape))
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, n, nkv, -1, DIM)[:, :, :, :T]
    cu, L = s["cu"].long(), s["kv_len"].long()
    new = cu[1:] - cu[:-1]
    j = torch.arange(S, device=dev)
    row = (cu[:-1, None] + j).clamp(max=s["rows"] - 1)  # [n, S]
    q = s["q"][:, : nq * DIM].float()[row].view(n, S, nkv, nq // nkv, DIM).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, DIM)
    score = (q @ kv[0].transpose(2, 3)) * (1.0 / math.sqrt(DIM))
    pos = (L - new)[:, None] + j  # [n, S]
    hidden = torch.arange(T, device=dev) > pos[:, :, None]  # [n, S, T]
    score = score.view(n, nkv, nq // nkv, S, T).masked_fill_(hidden[:, None, None], -math.inf)
    score = (score - score.amax(-1, keepdim=True)).exp_()
    kv[1].masked_fill_((torch.arange(T, device=dev) >= L[:, None])[:, None, :, None], 0.0)
    o = (score.view(n, nkv, -1, T) @ kv[1]) / score.sum(-1).view(n, nkv, -1, 1)
    o = o.view(n, nq, S, DIM).transpose(1, 2).reshape(n * S, nq * DIM)
    i = torch.repeat_interleave(torch.arange(n, device=dev), new, output_size=s["rows"])
    return o[i * S + torch.arange(s["rows"], device=dev) - cu[i]].to(s["type"])


def _plain_w4(s):
    c = s["case"]
    n_out, k, group = c["n_out"], c["k"], c["group"]
    u = torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).view(n_out, k // group, group).float()
    z = s["zero"].float()[:, :, None] if s["zero"] is not None else 8.0
    w = ((u - z) * s["scale"].float()[:, :, None]).view(n_out, k)
    return (s["x"][:, :k].float() @ w.t()).to(s["type"])


# ---------------------------------------------------------------------------------------- floors and 64 bits
def work(case):
    lens = _lens(case) if case["op"] != "w4" else []
    if case["op"] == "plan":
        n, rows = case["n"], sum(b for _, b in lens)
        if case["release"]:
            pages = sum(_pages(a) for a, _ in lens)
            return {"bytes": 4 * (2 * n + 2 * pages + n + 4), "flops": 0}
        pages = sum(_pages(a + b) - _pages(a) for a, b in lens)
        return {"bytes": 4 * (3 * n + 2 * pages + n + n + 1 + 2 * rows + 4), "flops": 0}
    if case["op"] == "w4":
        n_out, k, g, r = case["n_out"], case["k"], case["group"], case["rows"]
        return {"bytes": n_out * k // 2 + n_out * (k // g) * (3 if case["zeros"] else 2) + 2 * r * (k + n_out),
                "flops": 2 * r * n_out * k}
    nq, nkv, rows = case["nq"], case["nkv"], sum(b for _, b in lens)
    kv = sum(a + b for a, b in lens)
    seen = sum(b * a + b * (b + 1) // 2 for a, b in lens)
    return {"bytes": 2 * 2 * rows * nq * DIM + 2 * 2 * kv * nkv * DIM + 4 * (sum(_pages(a + b) for a, b in lens) + 3 * len(lens)),
            "flops": 4 * DIM * nq * seen}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "w4":
        n_out, k, group = case["n_out"], case["k"], case["group"]
        x = s["x"][:, :k].double()
        out = torch.empty((case["rows"], n_out), dtype=torch.float64, device=DEV)
        for m in range(0, n_out, 8192):
            b = s["codes"][m : m + 8192].to(torch.int64)
            u = torch.empty((b.shape[0], k), dtype=torch.float64, device=DEV)
            u[:, 0::2], u[:, 1::2] = (b % 16).double(), (b // 16).double()
            sc = s["scale"][m : m + 8192].double().repeat_interleave(group, 1)
            z = s["zero"][m : m + 8192].double().repeat_interleave(group, 1) if s["zero"] is not None else torch.full_like(u, 8.0)
            out[:, m : m + 8192] = x @ (sc * (u - z)).t()
        return out
    nq, nkv = case["nq"], case["nkv"]
    out = torch.zeros((s["rows"], nq * DIM), dtype=torch.float64, device=DEV)
    first = 0
    for i, (a, b) in enumerate(_lens(case)):
        pages = s["table"][int(s["slot"][i]), : _pages(a + b)].long()
        got = s["pool"][pages, case["layer"]]  # [pages, 2, nkv, 64, 128]
        flat = torch.empty((2, nkv, (a + b), DIM), dtype=torch.float64, device=DEV)
        pos = torch.arange(a + b, device=DEV)
        for chunk in range(DIM // 8):
            at = ((chunk ^ (pos % 8)) * 8)[:, None] + torch.arange(8, device=DEV)  # [positions, 8]
            part = got[pos // PAGE, :, :, pos % PAGE]  # [positions, 2, nkv, 128]
            part = part.gather(3, at[:, None, None, :].expand(-1, 2, nkv, -1))
            flat[..., chunk * 8 : chunk * 8 + 8] = part.permute(1, 2, 0, 3).double()
        for h in range(nq):
            k, v = flat[0, h // (nq // nkv)], flat[1, h // (nq // nkv)]
            for r in range(0, b, 2048):
                m = min(2048, b - r)
                q = s["q"][first + r : first + r + m, h * DIM : (h + 1) * DIM].double()
                w = q @ k.t() / math.sqrt(DIM)
                w[pos[None, :] > (a + r + torch.arange(m, device=DEV))[:, None]] = -math.inf
                out[first + r : first + r + m, h * DIM : (h + 1) * DIM] = torch.softmax(w, -1) @ v
        first += b
    return out
