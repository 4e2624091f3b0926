"""Cases of the drafted-token tree operators over the paged KV cache.

Three operators of the kernel-level interface (include/tvara_kernels.h), in the
order in which a speculative step uses them:

* ``plan``   tvara_tree_plan: block tables, slot maps, positions and ancestor
  masks on the GPU from request lengths;
* ``attend`` tvara_tree_attention: attention of every drafted token to its
  sequence's cached positions and to its ancestors in the tree;
* ``commit`` tvara_tree_commit: the walk down each tree along the model's own
  choices, and the accepted tokens' K/V rows moved to where the sequence
  continues.

``run`` computes them in plain torch operations (F32, rounded once), or through
the library where ``own`` is true.  What a case's requests look like (lengths,
tree shapes) follows from the case alone, so that its work is known; every value
follows from the seed.
"""

import math
import random

import torch

own = False

KV = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "i8": (2, torch.int8, 1)}
NO_TOKEN = -1  # 0xFFFFFFFF in the 32-bit token arrays


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a single user decoding greedily: one token behind a short prompt, the reference's F32 cache
        {"name": "attend_one_token_f32", "op": "attend", "kv": "f32", "n_seq": 1, "context_lo": 130, "context_hi": 130,
         "nodes_lo": 1, "nodes_hi": 1, "heads": 9, "kv_heads": 3, "head_dim": 64, "block_tokens": 16, "pattern": 1},
        # a single user with a small static tree over a conversation
        {"name": "attend_single_user_f16", "op": "attend", "kv": "f16", "n_seq": 1, "context_lo": 1900, "context_hi": 1900,
         "nodes_lo": 26, "nodes_hi": 26, "heads": 32, "kv_heads": 8, "head_dim": 128, "block_tokens": 16, "pattern": 2},
        # a serving batch: ragged contexts, trees of up to 64 nodes
        {"name": "attend_batch_f16", "op": "attend", "kv": "f16", "n_seq": 64, "context_lo": 200, "context_hi": 4000,
         "nodes_lo": 1, "nodes_hi": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "block_tokens": 16, "pattern": 3},
        # the same heads over the int8 cache, longer contexts, small trees
        {"name": "attend_batch_i8", "op": "attend", "kv": "i8", "n_seq": 24, "context_lo": 1000, "context_hi": 12000,
         "nodes_lo": 4, "nodes_hi": 29, "heads": 32, "kv_heads": 8, "head_dim": 128, "block_tokens": 32, "pattern": 4},
        # the small model's heads (three query heads to a KV head) over the F32 cache
        {"name": "attend_small_heads_f32", "op": "attend", "kv": "f32", "n_seq": 31, "context_lo": 64, "context_hi": 6000,
         "nodes_lo": 5, "nodes_hi": 33, "heads": 9, "kv_heads": 3, "head_dim": 64, "block_tokens": 16, "pattern": 5},
        # few long documents, large trees
        {"name": "attend_large_trees_f16", "op": "attend", "kv": "f16", "n_seq": 4, "context_lo": 8000, "context_hi": 30000,
         "nodes_lo": 129, "nodes_hi": 255, "heads": 32, "kv_heads": 8, "head_dim": 128, "block_tokens": 64, "pattern": 6},
        # bookkeeping of one user's step
        {"name": "plan_single_user", "op": "plan", "n_seq": 1, "context_lo": 1900, "context_hi": 1900, "nodes_lo": 26, "nodes_hi": 26,
         "tree": True, "block_tokens": 16, "pattern": 7},
        # bookkeeping of a serving batch of trees
        {"name": "plan_batch_trees", "op": "plan", "n_seq": 500, "context_lo": 1, "context_hi": 8000, "nodes_lo": 1, "nodes_hi": 63,
         "tree": True, "block_tokens": 16, "pattern": 8},
        # prompts of a batch of requests entering the cache: no trees, many tokens each
        {"name": "plan_prompts", "op": "plan", "n_seq": 511, "context_lo": 0, "context_hi": 3000, "nodes_lo": 1, "nodes_hi": 2047,
         "tree": False, "block_tokens": 16, "pattern": 9},
        # one user's tree over the small model's F32 cache
        {"name": "commit_single_user_f32", "op": "commit", "kv": "f32", "n_seq": 1, "nodes_lo": 26, "nodes_hi": 26, "layers": 30,
         "kv_heads": 3, "head_dim": 64, "block_tokens": 16, "pattern": 10},
        # a serving batch, 32 layers
        {"name": "commit_batch_f16", "op": "commit", "kv": "f16", "n_seq": 48, "nodes_lo": 8, "nodes_hi": 64, "layers": 32,
         "kv_heads": 8, "head_dim": 128, "block_tokens": 16, "pattern": 11},
        # the same over the int8 cache (codes and row scales move together)
        {"name": "commit_batch_i8", "op": "commit", "kv": "i8", "n_seq": 33, "nodes_lo": 1, "nodes_hi": 63, "layers": 32,
         "kv_heads": 8, "head_dim": 128, "block_tokens": 32, "pattern": 12},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, name, lo, hi):
    a, b = sorted((_spread(rng, lo, hi), _spread(rng, lo, hi)))
    return {name + "_lo": a, name + "_hi": b}


def draw(rng):
    op = rng.choice(["attend", "attend", "plan", "commit"])
    case = {"op": op, "block_tokens": rng.choice([8, 16, 16, 24, 32, 64]), "pattern": rng.randrange(1 << 30)}
    if op == "plan":
        tree = rng.random() < 0.6
        case.update(n_seq=_spread(rng, 1, 500), context_lo=0, context_hi=_spread(rng, 1, 8000), tree=tree,
                    **_range(rng, "nodes", 1, 255 if tree else 2047))
        return case
    heads, kv_heads, head_dim = rng.choice([(9, 3, 64), (32, 8, 128), (32, 8, 128), (8, 2, 32), (16, 16, 64), (28, 4, 128)])
    case.update(kv=rng.choice(["f32", "f16", "f16", "i8"]), kv_heads=kv_heads, head_dim=head_dim)
    if op == "commit":
        case.update(n_seq=_spread(rng, 1, 48), layers=rng.randint(1, 32), **_range(rng, "nodes", 1, 64))
        return case
    positions = 100000 if case["kv"] != "f32" else 60000  # of all sequences together
    n_seq = _spread(rng, 1, 64)
    longest = max(2, min(30000, positions // n_seq))
    case.update(heads=heads, n_seq=n_seq, **_range(rng, "nodes", 1, 255 if n_seq <= 4 else 64),
                **_range(rng, "context", 1, longest))
    return case


def _requests(case):
    """Context length, node count and tree (parents within the sequence, -1 for
    children of the context) of every request of a case."""
    rng = random.Random(case["pattern"])
    out = []
    for _ in range(case["n_seq"]):
        n = rng.randint(case["nodes_lo"], case["nodes_hi"])
        context = rng.randint(case.get("context_lo", 100), case.get("context_hi", 100))
        parents, depth = [], []
        if case.get("tree", True):
            for i in range(n):  # bushy near the root, thin below, as drafted by top-k proposals
                p = -1 if i == 0 else rng.randrange(-1, i) if rng.random() < 0.3 else max(0, i - rng.randint(1, 1 + i // 2))
                parents.append(p)
                depth.append(0 if p < 0 else depth[p] + 1)
        out.append((context, n, parents, depth))
    return out


def _accepted(case):
    """The path of accepted nodes of each request: from a root down, mostly to a leaf."""
    rng = random.Random(case["pattern"] + 1)
    paths = []
    for _, n, parents, _ in _requests(case):
        path, at = [], -1
        while True:
            children = [c for c in range(n) if parents[c] == at]
            if not children or rng.random() < 0.15:
                break
            at = rng.choice(children)
            path.append(at)
        paths.append(path)
    return paths


# ------------------------------------------------------------------- the work
def work(case):
    reqs = _requests(case)
    if case["op"] == "attend":
        size, d, hq, hkv = KV[case["kv"]][2], case["head_dim"], case["heads"], case["kv_heads"]
        row = d * size + (4 if case["kv"] == "i8" else 0)
        b = f = 0
        for context, n, _, depth in reqs:
            b += (context + n) * 2 * hkv * row        # K and V, once
            b += 2 * n * hq * d * 4                   # queries and outputs
            b += 4 * -(-context // case["block_tokens"]) + 16 * n + 12
            f += sum(context + 1 + e for e in depth) * hq * d * 4
        return {"bytes": b, "flops": f}
    if case["op"] == "plan":
        b = 0
        for context, n, _, _ in reqs:
            new = _new_blocks(case, context, n)
            b += 16 + 12 * n + 8 * new + (4 * n + 8 * n * _words(case) if case["tree"] else 0)
        return {"bytes": b, "flops": 0}
    row = case["head_dim"] * KV[case["kv"]][2] + (4 if case["kv"] == "i8" else 0)
    moved = sum(len(p) for p in _accepted(case))
    nodes = sum(r[1] for r in reqs)
    return {"bytes": moved * 2 * case["layers"] * case["kv_heads"] * row * 2 + moved * 20 + nodes * 16
            + case["n_seq"] * 24, "flops": 0}


def _words(case):
    return -(-case["nodes_hi"] // 64)


def _new_blocks(case, context, n):
    bt = case["block_tokens"]
    return -(-(context + n) // bt) - -(-context // bt)


# ----------------------------------------------------------------- the inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    reqs = _requests(case)
    s = dict(case)
    counts = [r[1] for r in reqs]
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    s.update(total=cu[-1], most=max(counts), longest=max(r[0] for r in reqs), cu=_ints(cu),
             lengths=_ints([r[0] for r in reqs]))
    s["parents"] = _ints([p for r in reqs for p in r[2]]) if case.get("tree", True) else None
    {"attend": _prepare_attend, "plan": _prepare_plan, "commit": _prepare_commit}[case["op"]](s, case, reqs, gen)
    if own:
        _arguments(s)
    return s


def _pool(case, blocks, layers, gen):
    """A cache in use: every row holds some token's values."""
    shape = (blocks, layers, 2, case["kv_heads"], case["block_tokens"], case["head_dim"])
    _, dtype, _ = KV[case["kv"]]
    if case["kv"] == "i8":
        pool = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
        return pool, (torch.rand(shape[:-1], generator=gen, device="cuda") + 0.5) * (2.5 / 127)
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype), None


def _prepare_attend(s, case, reqs, gen):
    bt = case["block_tokens"]
    need = [-(-(r[0] + r[1]) // bt) for r in reqs]
    s["layers"], s["layer"] = 2, 1
    s["blocks"] = sum(need) + 3
    s["pool"], s["scales"] = _pool(case, s["blocks"], s["layers"], gen)
    order = torch.randperm(s["blocks"], generator=gen, device="cuda").to(torch.int32)
    s["table_stride"] = max(need)
    table = torch.zeros(len(reqs), max(need), dtype=torch.int32, device="cuda")
    slots = torch.empty(s["total"], dtype=torch.int64, device="cuda")
    at = row = 0
    for i, (context, n, _, _) in enumerate(reqs):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        p = torch.arange(context, context + n, device="cuda")
        slots[row:row + n] = table[i].long()[p // bt] * bt + p % bt
        row += n
    width = case["heads"] * case["head_dim"]
    s["q"] = torch.randn(s["total"], width, generator=gen, device="cuda") * 1.5
    s["out"] = torch.zeros_like(s["q"])
    s["tables"], s["slots"], s["words"] = table, slots, _words(case)
    s["ancestors"] = _ancestor_words(s)


def _prepare_plan(s, case, reqs, gen):
    bt = case["block_tokens"]
    held = [-(-r[0] // bt) for r in reqs]
    need = [-(-(r[0] + r[1]) // bt) for r in reqs]
    s["blocks"] = sum(need) + 5
    order = torch.randperm(s["blocks"], generator=gen, device="cuda").to(torch.int32)
    s["table_stride"], s["words"] = max(need) + 1, _words(case)
    table = torch.zeros(len(reqs), s["table_stride"], dtype=torch.int32, device="cuda")
    j = torch.arange(s["table_stride"], device="cuda")
    h = _ints(held, torch.int64)
    first = torch.cumsum(h, 0) - h
    mine = j[None] < h[:, None]
    table[mine] = order[(first[:, None] + j[None])[mine]]
    s["tables"], s["held"] = table, _ints(held)
    s["free"] = order[sum(held):].contiguous()
    s["free_count"] = _ints([s["blocks"] - sum(held)])
    n = s["total"]
    s["slots"] = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    s["positions"] = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    s["ancestors"] = torch.zeros(n, s["words"], dtype=torch.int64, device="cuda") if case["tree"] else None
    s["held_out"], s["free_left"] = torch.zeros_like(s["held"]), torch.zeros_like(s["free_count"])


def _prepare_commit(s, case, reqs, gen):
    """Drafted rows lie in blocks of their own; accepted ones move to the
    sequences' blocks."""
    bt, n = case["block_tokens"], s["total"]
    per = [-(-r[1] // bt) for r in reqs]
    s["blocks"] = 2 * sum(per) + len(reqs) + 2
    s["pool"], s["scales"] = _pool(case, s["blocks"], case["layers"], gen)
    order = torch.randperm(s["blocks"], generator=gen, device="cuda").tolist()
    rng = random.Random(case["pattern"] + 2)
    slots, dest, at = [], [], 0
    for r, blocks in zip(reqs, per):
        slots += [order[at + i // bt] * bt + i % bt for i in range(r[1])]
        at += blocks
        off = rng.randrange(bt)  # the sequence's next position lies inside its last block
        dest += [order[at + (off + i) // bt] * bt + (off + i) % bt for i in range(r[1])]
        at += blocks + 1
    s["slots"], s["dest"] = _ints(slots, torch.int64), _ints(dest, torch.int64)
    # token ids and the model's choices: siblings differ, choices follow the accepted path and then leave the tree
    vocab = 49152
    tokens = torch.randint(0, vocab // 2, (n,), generator=gen, device="cuda", dtype=torch.int32)
    tokens = tokens * 2
    index = torch.arange(n, device="cuda", dtype=torch.int32) - torch.repeat_interleave(s["cu"][:-1], s["cu"].diff())
    tokens = (tokens - tokens % 1024 + 2 * (index % 512)).to(torch.int32)
    choices = torch.randint(0, vocab // 2, (n,), generator=gen, device="cuda", dtype=torch.int32) * 2 + 1
    first = torch.randint(0, vocab // 2, (len(reqs),), generator=gen, device="cuda", dtype=torch.int32) * 2 + 1
    cu = s["cu"].tolist()
    link_from, link_to, roots, root_seq = [], [], [], []
    for i, path in enumerate(_accepted(case)):
        if path:
            roots.append(cu[i] + path[0])
            root_seq.append(i)
        for a, b in zip(path, path[1:]):
            link_from.append(cu[i] + a)
            link_to.append(cu[i] + b)
    if link_from:
        choices[_ints(link_from, torch.int64)] = tokens[_ints(link_to, torch.int64)]
    if roots:
        first[_ints(root_seq, torch.int64)] = tokens[_ints(roots, torch.int64)]
    s["tokens"], s["choices"], s["first"] = tokens, choices, first
    s["path"] = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    s["accepted"], s["next"] = torch.zeros_like(first), torch.zeros_like(first)
    s["lengths_out"] = torch.zeros_like(s["lengths"])


# ------------------------------------------------------------ the plain forms
def _padded(s):
    """Rows of the flat token arrays as [n_seq, most], and which of them exist."""
    i = torch.arange(s["most"], device="cuda")
    cu = s["cu"].long()
    rows = cu[:-1, None] + i[None]
    there = rows < cu[1:, None]
    return torch.where(there, rows, 0), there


def _closure(s, rows, there):
    """[n_seq, most, most]: node j is node i itself or an ancestor of it."""
    n = s["most"]
    parent = torch.where(there, s["parents"].long()[rows], -1)
    reach = (parent[:, :, None] == torch.arange(n, device="cuda")[None, None]).float()
    reach = reach + torch.eye(n, device="cuda")
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    return (reach > 0) & there[:, :, None] & there[:, None, :]


def _to_words(mask, words):
    """The last axis of truth values as 64-bit words, least significant bit first."""
    pad = words * 64 - mask.shape[-1]
    bits = torch.nn.functional.pad(mask, (0, pad)).reshape(*mask.shape[:-1], words, 64).long()
    return (bits << torch.arange(64, device="cuda")).sum(-1)


def _ancestor_words(s):
    rows, there = _padded(s)
    words = _to_words(_closure(s, rows, there), s["words"])
    return words[there]


def _plain_plan(s):
    bt, stride = s["block_tokens"], s["table_stride"]
    lengths, cu, held = s["lengths"].long(), s["cu"].long(), s["held"].long()
    counts = cu[1:] - cu[:-1]
    new = torch.clamp((lengths + counts + bt - 1) // bt - held, min=0)
    first = torch.cumsum(new, 0) - new
    j = torch.arange(stride, device="cuda")[None]
    fresh = (j >= held[:, None]) & (j < (held + new)[:, None])
    take = s["free_count"].long() - 1 - (first[:, None] + j - held[:, None])
    tables = torch.where(fresh, s["free"].long()[torch.where(fresh, take, 0)], s["tables"].long())
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    place = lengths[seq] + row - cu[seq]
    slots = tables[seq, place // bt] * bt + place % bt
    out = {"tables": tables.int(), "slots": slots, "held": (held + new).int(),
           "free_left": (s["free_count"].long() - new.sum()).int()}
    if s["parents"] is None:
        out["positions"] = place.int()
        return out
    rows, there = _padded(s)
    closure = _closure(s, rows, there)
    out["ancestors"] = _to_words(closure, s["words"])[there]
    depth = closure.sum(-1)[there] - 1
    out["positions"] = (lengths[seq] + depth).int()
    return out


def _plain_attend(s):
    bt, d, hkv = s["block_tokens"], s["head_dim"], s["kv_heads"]
    group = s["heads"] // hkv
    rows, there = _padded(s)
    context = s["lengths"].long()
    j = torch.arange(s["longest"], device="cuda")
    cached = j[None] < context[:, None]
    slot = torch.where(cached, s["tables"].long()[:, j // bt] * bt + j % bt, 0)
    slot = torch.cat([slot, torch.where(there, s["slots"][rows], 0)], 1)
    valid = torch.cat([cached, there], 1)
    block, off = slot // bt, slot % bt

    def side(kind):  # [n_seq, kv_heads, positions, d]
        x = s["pool"][block, s["layer"], kind, :, off].float()
        if s["scales"] is not None:
            x = x * s["scales"][block, s["layer"], kind, :, off][..., None]
        return torch.where(valid[:, :, None, None], x, 0.0).permute(0, 2, 1, 3)

    k = side(0)
    n_seq, most = rows.shape
    q = s["q"][rows].reshape(n_seq, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(n_seq, hkv, most * group, d)
    scores = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    del k
    words = s["ancestors"][rows]
    i = torch.arange(s["most"], device="cuda")
    mine = ((words[:, :, i // 64] >> (i % 64)) & 1).bool() & there[:, None, :]
    seen = torch.cat([cached[:, None, :].expand(-1, most, -1), mine], 2)
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    del scores
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, side(1)) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n_seq, hkv, most, group, d).permute(0, 2, 1, 3, 4).reshape(n_seq, most, -1)
    return {"out": out[there]}


def _plain_commit(s):
    bt = s["block_tokens"]
    rows, there = _padded(s)
    parent = torch.where(there, s["parents"].long()[rows], -2)
    tokens = s["tokens"][rows]
    wanted = torch.where(parent >= 0, s["choices"][rows].gather(1, parent.clamp(min=0)), s["first"][:, None])
    twin = (parent[:, :, None] == parent[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :])
    earlier = torch.ones(s["most"], s["most"], dtype=torch.bool, device="cuda").tril(-1)
    good = there & (tokens == wanted) & ~(twin & earlier).any(-1)
    closure = _closure(s, rows, there)
    kept = there & ~(closure & ~good[:, None, :]).any(-1)
    accepted = kept.sum(1)
    order = torch.where(kept, torch.cumsum(kept, 1) - 1, s["most"])
    path = torch.full((s["n_seq"], s["most"] + 1), -1, dtype=torch.int64, device="cuda")
    path.scatter_(1, order, torch.arange(s["most"], device="cuda")[None].expand_as(order))
    path = torch.where(torch.arange(s["most"], device="cuda")[None] < accepted[:, None], path[:, :-1], -1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])[:, 0]
    follow = torch.where(accepted > 0, s["choices"][rows].gather(1, last.clamp(min=0)[:, None])[:, 0], s["first"])
    pool, scales = s["pool"], s["scales"]
    moved = path >= 0
    src = s["slots"][rows.gather(1, path.clamp(min=0))[moved]]
    dst = s["dest"][rows[moved]]
    pool[dst // bt, :, :, :, dst % bt] = pool[src // bt, :, :, :, src % bt]
    out = {"path": path[there].int(), "accepted": accepted.int(), "next": follow,
           "lengths": (s["lengths"] + accepted).int(), "pool": pool}
    if scales is not None:
        scales[dst // bt, :, :, :, dst % bt] = scales[src // bt, :, :, :, src % bt]
        out["scales"] = scales
    return out


def run(s):
    if own:
        return _own(s)
    return {"attend": _plain_attend, "plan": _plain_plan, "commit": _plain_commit}[s["op"]](s)


# ---------------------------------------------------------- through the library
def _arguments(s):
    """The argument structure and workspace that a program keeps from call to call."""
    import ctypes as C

    from tvara_b200 import _bindings as B
    from tvara_b200 import load_library

    lib = load_library()
    name = {"attend": "TreeAttentionArgs", "plan": "TreePlanArgs", "commit": "TreeCommitArgs"}[s["op"]]
    a = getattr(B, name)()
    a.struct_size = C.sizeof(a)

    def give(**fields):
        for key, value in fields.items():
            setattr(a, key, value.data_ptr() if isinstance(value, torch.Tensor) else value)

    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    give(block_tokens=s["block_tokens"], n_seq=s["n_seq"], capacity=s["total"], max_blocks=s["blocks"],
         max_nodes=s["most"] if s["op"] == "commit" else s["nodes_hi"], cu_nodes=s["cu"], lengths=s["lengths"],
         status=s["status"])
    if s["op"] == "plan":
        give(table_stride=s["table_stride"], held=s["held"], free_blocks=s["free"], free_capacity=s["free"].numel(),
             free_count=s["free_count"], tables=s["tables"], slots=s["slots"], positions=s["positions"],
             held_out=s["held_out"], free_left=s["free_left"])
        if s["parents"] is not None:
            give(parents=s["parents"], ancestors=s["ancestors"])
        s["call"] = lib.tvara_tree_plan
    elif s["op"] == "attend":
        width = s["heads"] * s["head_dim"]
        give(kv_dtype=KV[s["kv"]][0], heads=s["heads"], kv_heads=s["kv_heads"], head_dim=s["head_dim"],
             layers=s["layers"], layer=s["layer"], table_stride=s["table_stride"], q_stride=width, out_stride=width,
             q=s["q"], out=s["out"], pool=s["pool"], tables=s["tables"], slots=s["slots"], ancestors=s["ancestors"])
        if s["scales"] is not None:
            give(kv_scales=s["scales"])
        size = lib.tvara_tree_attention_workspace(C.byref(a))
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        s["workspace_args"] = (C.c_void_p(s["workspace"].data_ptr()), size)
        s["call"] = lib.tvara_tree_attention
    else:
        give(kv_dtype=KV[s["kv"]][0], kv_heads=s["kv_heads"], head_dim=s["head_dim"], layers=s["layers"],
             parents=s["parents"], tokens=s["tokens"], choices=s["choices"], first=s["first"], slots=s["slots"],
             dest=s["dest"], pool=s["pool"], path=s["path"], accepted=s["accepted"], next=s["next"],
             lengths_out=s["lengths_out"])
        if s["scales"] is not None:
            give(kv_scales=s["scales"])
        s["call"] = lib.tvara_tree_commit
    s["args"], s["by"], s["lib"] = a, C.byref(a), lib


def _own(s):
    stream = torch.cuda.current_stream().cuda_stream
    if s["call"](s["by"], *s.get("workspace_args", ()), stream):
        raise RuntimeError(s["lib"].tvara_last_error().decode())
    if s["op"] == "attend":
        return {"out": s["out"]}
    if s["op"] == "plan":
        out = {"tables": s["tables"], "slots": s["slots"], "held": s["held_out"], "free_left": s["free_left"],
               "positions": s["positions"]}
        if s["parents"] is not None:
            out["ancestors"] = s["ancestors"]
        return out
    out = {"path": s["path"], "accepted": s["accepted"], "next": s["next"], "lengths": s["lengths_out"],
           "pool": s["pool"]}
    if s["scales"] is not None:
        out["scales"] = s["scales"]
    return out


# -------------------------------------------------------------- the definition
def exact(case, seed):
    """Attention in 64 bits, one sequence and node at a time in the masks: every
    drafted token attends to its sequence's cached positions and to the nodes on
    its way up the tree.  The other operators' outputs are whole numbers and
    moved values."""
    if case["op"] != "attend":
        return None
    s = prepare(case, seed)
    bt, d, hkv = s["block_tokens"], s["head_dim"], s["kv_heads"]
    group = s["heads"] // hkv
    out = torch.empty(s["total"], s["heads"], d, dtype=torch.float64, device="cuda")
    row = 0
    for i, (context, n, parents, _) in enumerate(_requests(case)):
        at = torch.arange(context, device="cuda")
        table = s["tables"][i].long()
        where = torch.cat([table[at // bt] * bt + at % bt, s["slots"][row:row + n]])
        kv = []
        for kind in (0, 1):
            x = s["pool"][where // bt, s["layer"], kind, :, where % bt].double()
            if s["scales"] is not None:
                x = x * s["scales"][where // bt, s["layer"], kind, :, where % bt].double()[..., None]
            kv.append(x)
        seen = torch.zeros(n, context + n, dtype=torch.bool)
        seen[:, :context] = True
        for node in range(n):
            up = node
            while up >= 0:
                seen[node, context + up] = True
                up = parents[up]
        seen = seen.cuda()
        for h in range(s["heads"]):
            q = s["q"][row:row + n, h * d:(h + 1) * d].double()
            scores = (q @ kv[0][:, h // group].T) / math.sqrt(d)
            p = torch.softmax(scores.masked_fill(~seen, -math.inf), 1)
            out[row:row + n, h] = p @ kv[1][:, h // group]
        row += n
    return {"out": out.reshape(s["total"], -1)}
