"""Plain 64-bit forms of the drafted-token tree operators
(include/tvara_kernels.h tvara_tree_*) and the inputs their tests share."""

import ctypes as C

import numpy as np

from tvara_b200 import _bindings as B

KV = {"f32": (0, np.float32), "f16": (1, np.float16), "i8": (2, np.int8)}
NONE = 0xFFFFFFFF


def random_tree(rng, n, chain=False):
    """Parents of n nodes: -1 for children of the context, else a smaller index."""
    if chain:
        return np.arange(-1, n - 1, dtype=np.int32)
    return np.array([rng.integers(-1, i) if rng.random() < 0.4 else max(-1, i - int(rng.integers(1, 4)))
                     for i in range(n)], dtype=np.int32)


def ancestors(parents):
    """[n, n] truth values: j is i or one of its ancestors."""
    n = len(parents)
    out = np.zeros((n, n), bool)
    for i in range(n):
        if parents[i] >= 0:
            out[i] = out[parents[i]]
        out[i, i] = True
    return out


def mask_words(mask, words):
    """Truth values [n, m] as [n, words] 64-bit words."""
    n, m = mask.shape
    bits = np.zeros((n, words * 64), np.uint8)
    bits[:, :m] = mask
    return np.ascontiguousarray(np.packbits(bits, axis=1, bitorder="little")).view(np.uint64)


def plan(lengths, held, cu, parents, tables, free, free_count, bt):
    """The plan's outputs as the header defines them; None when blocks run out."""
    tables, n_seq = tables.copy(), len(lengths)
    held_out = held.copy()
    top = int(free_count)
    slots = np.full(cu[-1], -1, np.int64)
    positions = np.full(cu[-1], -1, np.int32)
    masks = []
    for s in range(n_seq):
        n = int(cu[s + 1] - cu[s])
        need = max(0, -(-(int(lengths[s]) + n) // bt) - int(held[s]))
        for e in range(need):
            if top == 0:
                return None
            top -= 1
            tables[s, held[s] + e] = free[top]
        held_out[s] += need
        p = int(lengths[s]) + np.arange(n)
        slots[cu[s]:cu[s + 1]] = tables[s][p // bt].astype(np.int64) * bt + p % bt
        if parents is None:
            positions[cu[s]:cu[s + 1]] = p
        else:
            a = ancestors(parents[cu[s]:cu[s + 1]])
            positions[cu[s]:cu[s + 1]] = lengths[s] + a.sum(1) - 1
            masks.append(a)
    return dict(tables=tables, held=held_out, free_left=top, slots=slots, positions=positions, masks=masks)


def walk(parents, tokens, choices, first):
    """Accepted nodes of one sequence and the choice the walk ends with; first
    None: node 0 is accepted as it is."""
    n, path = len(parents), []
    want, at = first, -1
    if first is None:
        want = NONE
        if n and parents[0] == -1:
            path, at, want = [0], 0, int(choices[0])
    while want != NONE:
        hit = [c for c in range(at + 1, n) if parents[c] == at and int(tokens[c]) == want]
        if not hit:
            break
        at = hit[0]
        path.append(at)
        want = int(choices[at])
    return path, want


def attention(q, k, v, mask, group, split=False):
    """Softmax attention in 64 bits: q [n, heads, d], k and v [kv_heads, m, d],
    mask [n, m].  Returns the rows and a bound on the rounding of an F32
    evaluation.  The bound: a score is 2 d/16 + 1 truncating F32 additions of
    products that carry q to 22 bits, so it is off by at most (2 d/16 + 1)
    2^-23 of its sum of |q k|; a weight by twice that (numerator and sum) and
    2^-22 of the exponential; the weighted sum adds 24 additions' 2^-23; and a
    weight carries an absolute 2^-24 of the row's largest, of either sign,
    which over m terms adds up like a random walk (six deviations of
    sqrt(m) 2^-25).

    split: K and V are F32 and enter as two F16 parts, hi a multiple of 16 and
    lo at most 8 for a row whose largest value lies in [2^14, 2^15).  lo rounds
    by at most 2^-9, so an element is off by 2^-23 of its row's largest: a
    score by 2^-23 kmax sum|q|, an output by 2^-23 of the weighted row maxima.
    The lo x lo products are left out: q_lo k_lo is the product of two values
    uniform within 2^-11 of the rows' largest, over d terms six deviations are
    6 sqrt(d) (2^-11)^2 / 3; p_lo v_lo likewise with p_lo within 2^-12 of the
    row's largest weight: 6 sqrt(m) 2^-12 2^-11 / 3."""
    n, heads, d = q.shape
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    out = np.zeros((n, heads, d))
    tol = np.zeros((n, heads, d))
    for h in range(heads):
        kh, vh = k[h // group], v[h // group]
        for i in range(n):
            seen = mask[i]
            if not seen.any():
                continue
            ks, vs = kh[seen], vh[seen]
            s = ks @ q[i, h] / np.sqrt(d)
            size = np.abs(ks) @ np.abs(q[i, h]) / np.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vs
            e = (2 * -(-d // 16) + 1) * 2.0 ** -23 * size.max()
            if split:
                kmax, qmax = np.abs(ks).max(), np.abs(q[i, h]).max()
                e += (2.0 ** -23 * kmax * np.abs(q[i, h]).sum() + 2 * np.sqrt(d) * 2.0 ** -22 * qmax * kmax) / np.sqrt(d)
            tol[i, h] = (w @ np.abs(vs)) * (2 * e + 2.0 ** -22 + 24 * 2.0 ** -23) \
                + 6 * np.sqrt(len(vs)) * 2.0 ** -25 * np.abs(vs).max(0) + 1e-30
            if split:
                row = np.abs(vs).max(1)
                tol[i, h] += 2.0 ** -23 * (w @ row) + 2 * np.sqrt(len(vs)) * 2.0 ** -23 * row.max()
    return out, tol


class Dev:
    """Device arrays by name, kept alive beside an argument structure."""

    def __init__(self, struct, **sizes):
        self.a = struct()
        self.a.struct_size = C.sizeof(struct)
        self.keep = {}
        self.set(**sizes)

    def set(self, **fields):
        import torch
        for name, value in fields.items():
            if isinstance(value, np.ndarray):
                view = {np.dtype(np.uint32): np.int32, np.dtype(np.uint64): np.int64}.get(value.dtype)
                value = torch.from_numpy(np.ascontiguousarray(value.view(view) if view else value)).cuda()
            if hasattr(value, "data_ptr"):
                self.keep[name] = value
                value = value.data_ptr()
            setattr(self.a, name, value)
        return self

    def get(self, name):
        return self.keep[name].cpu().numpy()

    @property
    def by(self):
        return C.byref(self.a)


class AttentionCase:
    """One attention call: sequences with `lengths` cached positions and
    `nodes` drafts in a shuffled pool whose unused slots hold NaN (f32, f16) or
    extreme codes with NaN scales (int8)."""

    def __init__(self, rng, kv, lengths, nodes, heads, kv_heads, d, bt=16, layers=2, layer=1, masks="tree",
                 spare_rows=3, pad=0, max_nodes=None, q_scale=1.5):
        self.kv, self.lengths, self.nodes, self.heads, self.kv_heads, self.d, self.bt = kv, lengths, nodes, heads, \
            kv_heads, d, bt
        n_seq = len(lengths)
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        self.total = total = int(self.cu[-1])
        self.max_nodes = max_nodes or max(1, max(nodes))
        words = -(-self.max_nodes // 64)
        per = [-(-(a + b) // bt) for a, b in zip(lengths, nodes)]
        blocks = sum(per) + 4
        ids = rng.permutation(blocks)
        self.stride = max(1, max(per)) + 1
        self.tables = np.full((n_seq, self.stride), -7, np.int32)
        shape = (blocks, layers, 2, kv_heads, bt, d)
        _, dtype = KV[kv]
        self.scales = None
        if kv == "i8":
            self.pool = np.full(shape, -127, np.int8)
            self.scales = np.full(shape[:-1], np.nan, np.float32)
        else:
            self.pool = np.full(shape, np.nan, dtype)
        self.slots = np.full(total + spare_rows, -1, np.int64)
        self.k, self.v, self.mask = [], [], []
        at = 0
        for s, (length, n) in enumerate(zip(lengths, nodes)):
            mine = ids[at:at + per[s]]
            at += per[s]
            self.tables[s, :per[s]] = mine
            p = np.arange(length + n)
            slot = mine[p // bt].astype(np.int64) * bt + p % bt if len(p) else np.zeros(0, np.int64)
            if n:  # nodes in any order within their blocks: the slot map alone says where
                slot[length:] = rng.permutation(slot[length:])
            self.slots[self.cu[s]:self.cu[s + 1]] = slot[length:]
            b, o = slot // bt, slot % bt
            for kind, to in ((0, self.k), (1, self.v)):
                if kv == "i8":
                    codes = rng.integers(-127, 128, (length + n, kv_heads, d)).astype(np.int8)
                    sc = (rng.random((length + n, kv_heads)) * 0.03 + 0.001).astype(np.float32)
                    self.pool[b, layer, kind, :, o] = codes
                    self.scales[b, layer, kind, :, o] = sc
                    x = codes.astype(np.float64) * sc[..., None].astype(np.float64)
                else:
                    x = rng.standard_normal((length + n, kv_heads, d)).astype(dtype)
                    self.pool[b, layer, kind, :, o] = x
                to.append(np.moveaxis(x.astype(np.float64), 1, 0))
            if masks == "chain":
                m = np.tril(np.ones((n, n), bool))
            elif masks == "any":  # not a tree, some rows empty
                m = rng.random((n, n)) < 0.4
                m[rng.random(n) < 0.3] = False
            else:
                m = ancestors(random_tree(rng, n))
            self.mask.append(np.concatenate([np.ones((n, length), bool), m], 1))
        self.words = np.zeros((total + spare_rows, words), np.uint64)
        for s in range(n_seq):
            if nodes[s]:
                self.words[self.cu[s]:self.cu[s + 1]] = mask_words(self.mask[s][:, lengths[s]:], words)
        width = heads * d
        self.q = (rng.standard_normal((total + spare_rows, width + pad)) * q_scale).astype(np.float32)
        self.out = np.full((total + spare_rows, width + 2 * pad), 123.0, np.float32)
        self.dev = Dev(B.TreeAttentionArgs, kv_dtype=KV[kv][0], heads=heads, kv_heads=kv_heads, head_dim=d,
                       block_tokens=bt, layers=layers, layer=layer, n_seq=n_seq, capacity=total + spare_rows,
                       max_nodes=self.max_nodes, max_blocks=blocks, table_stride=self.stride, q_stride=width + pad,
                       out_stride=width + 2 * pad)
        self.chain = masks == "chain"

    def upload(self):
        self.dev.set(q=self.q, out=self.out, pool=self.pool, tables=self.tables,
                     lengths=np.asarray(self.lengths, np.int32), cu_nodes=self.cu, slots=self.slots,
                     status=np.zeros(1, np.int32))
        if self.scales is not None:
            self.dev.set(kv_scales=self.scales)
        if not self.chain:
            self.dev.set(ancestors=self.words)
        return self

    def run(self, lib, stream=None):
        import torch
        size = lib.tvara_tree_attention_workspace(self.dev.by)
        assert size, lib.tvara_last_error()
        self.workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert lib.tvara_tree_attention(self.dev.by, self.workspace.data_ptr(), size, stream) == 0, \
            lib.tvara_last_error()
        return self

    def want(self):
        out = self.out.astype(np.float64).copy()
        tol = np.zeros_like(out)
        width = self.heads * self.d
        for s, n in enumerate(self.nodes):
            if not n:
                continue
            r = slice(self.cu[s], self.cu[s + 1])
            q = self.q[r, :width].reshape(n, self.heads, self.d)
            o, t = attention(q, self.k[s], self.v[s], self.mask[s], self.heads // self.kv_heads,
                             self.kv == "f32")
            out[r, :width], tol[r, :width] = o.reshape(n, width), t.reshape(n, width)
        return out, tol

    def check(self):
        got = self.dev.get("out").astype(np.float64)
        want, tol = self.want()
        assert np.isfinite(got).all()
        worst = np.max(np.abs(got - want) - tol)
        assert worst <= 0, (worst, np.max(np.abs(got - want)), tol.max())
        assert self.dev.get("status")[0] == 0
