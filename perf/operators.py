"""Cases, inputs and plain forms of the operators on 4-bit rows and on pages of rows.

Rows of embeddings (or of a weight matrix) are held in 4 bits with a scale, and
where wanted a zero point, for every group of 32, 64 or 128 values.  A store keeps
rows in pages that sequences (collections) of rows own or share.

    products  y[b, i] = sum_g s[i, g] * sum_{j in g} (c[i, j] - z[i, g]) * x[b, j]
    search    the k nearest rows by squared L2 distance, or the k largest products
    append    rows are quantised into the pages of sequences, and read back as the
              values that they then stand for
    copy      pages of the pools onto others
    fork      children share their parents' full pages and copy the last, part-filled one
    compact   the kept rows of a sequence go, in order, into fresh pages

Without zero points z is 8 and s the largest magnitude of the group over 7; with
them s is the group's range (zero within it) over 15.  s is rounded to 32 and then
to 16 bits, a code to the nearest, ties to even.  Fresh pages are the lowest-numbered
free ones.  What changes a store begins its pass by freeing what the pass before
made, as a step of a service does, so that a pass finds the state as the first did.
"""
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OPERATORS = ("products", "search", "append", "copy", "fork", "compact")


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one vector against ten thousand rows of an odd width, with zero points: a
        # small collection, or one linear layer for one token; latency counts
        {"name": "products one", "op": "products", "n": 10000, "dim": 1000, "batch": 1, "group": 32,
         "x": "f32", "out": "f32", "zeros": True, "page_rows": 0},
        # 16 queries against a million passages of 1024 values, in pages
        {"name": "products many", "op": "products", "n": 1000000, "dim": 1024, "batch": 16, "group": 64,
         "x": "f16", "out": "f32", "zeros": False, "page_rows": 128},
        # the 10 nearest passages of one query, in an eighth of the million
        {"name": "search one", "op": "search", "n": 125000, "dim": 1024, "batch": 1, "group": 64,
         "x": "f32", "zeros": False, "page_rows": 0, "k": 10, "metric": "l2"},
        # 16 queries, 100 candidates each for a later stage, from pages
        {"name": "search many", "op": "search", "n": 1000000, "dim": 1024, "batch": 16, "group": 128,
         "x": "bf16", "zeros": True, "page_rows": 128, "k": 100, "metric": "ip"},
        # one new row for one collection
        {"name": "append one", "op": "append", "seqs": 1, "count": 1, "dim": 128, "group": 32,
         "x": "f32", "zeros": True, "page_rows": 64},
        # a load of passages for 8 collections of different sizes
        {"name": "append many", "op": "append", "seqs": 8, "count": 12500, "dim": 1024, "group": 64,
         "x": "f16", "zeros": False, "page_rows": 128},
        # a handful of small pages
        {"name": "copy few", "op": "copy", "pages": 3, "dim": 128, "page_rows": 16},
        # an eighth of a million fp16 rows
        {"name": "copy many", "op": "copy", "pages": 1953, "dim": 1024, "page_rows": 64},
        # one snapshot of a short sequence
        {"name": "fork one", "op": "fork", "parents": 1, "children": 1, "count": 1000, "dim": 128, "page_rows": 64},
        # 64 samples of 4 long sequences
        {"name": "fork many", "op": "fork", "parents": 4, "children": 64, "count": 20000, "dim": 1024, "page_rows": 16},
        # a tenth of a short sequence is dropped
        {"name": "compact one", "op": "compact", "seqs": 1, "count": 1000, "keep": 0.9, "dim": 128, "page_rows": 16},
        # a third of 8 collections is dropped
        {"name": "compact many", "op": "compact", "seqs": 8, "count": 25000, "keep": 0.67, "dim": 1024, "page_rows": 64},
    ]


def draw(rng):
    def spread(low, high):
        return int(round(low * (high / low) ** rng.random()))

    def width(high):
        d = spread(64, high)
        return d if rng.random() < 0.5 else -(-d // 32) * 32

    op = rng.choice(OPERATORS)
    page_rows = rng.choice((16, 48, 64, 100, 128, 256))
    if op in ("products", "search"):
        dim, batch = width(4096), rng.choice((1, 1, 2, 3, 5, 8, 11, 16))
        n = min(spread(100, 1000000), (1 << 30) // dim, (1 << 34) // (dim * batch))
        case = {"op": op, "n": n, "dim": dim, "batch": batch, "group": rng.choice((32, 64, 128)),
                "x": rng.choice(("f32", "f16", "bf16")), "zeros": rng.random() < 0.5,
                "page_rows": page_rows if rng.random() < 0.5 else 0}
        if op == "products":
            case["out"] = rng.choice(("f32", case["x"]))
        else:
            case["k"] = spread(1, 128)
            case["metric"] = rng.choice(("l2", "ip"))
        return case
    if op == "append":
        dim, seqs = width(4096), rng.choice((1, 2, 5, 8, 32))
        count = min(spread(1, 100000), max(1, (1 << 27) // (dim * seqs)))
        return {"op": op, "seqs": seqs, "count": count, "dim": dim, "group": rng.choice((32, 64, 128)),
                "x": rng.choice(("f32", "f16", "bf16")), "zeros": rng.random() < 0.5, "page_rows": page_rows}
    dim = rng.choice((width(2048), 128, 1024))
    if op == "copy":
        pages = min(spread(1, 4096), max(1, (1 << 28) // (2 * dim * page_rows)))
        return {"op": op, "pages": pages, "dim": dim, "page_rows": page_rows}
    if op == "fork":
        parents = rng.choice((1, 2, 4, 8))
        count = min(spread(10, 50000), (1 << 27) // (dim * parents))
        return {"op": op, "parents": parents, "children": parents * rng.choice((1, 2, 4, 8, 16)), "count": count,
                "dim": dim, "page_rows": page_rows}
    seqs = rng.choice((1, 2, 5, 8))
    count = min(spread(10, 100000), (1 << 27) // (dim * seqs))
    return {"op": op, "seqs": seqs, "count": count, "keep": round(rng.uniform(0.1, 0.95), 2), "dim": dim,
            "page_rows": page_rows}


def _ceil(a, b):
    return -(-a // b)


def _ragged(count, n):
    """Lengths of n sequences, the longest of `count` rows and the shortest of half of them."""
    return [count - (i * 7919) % (count // 2 + 1) for i in range(n)]


def work(case):
    op, dim = case["op"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if op in ("products", "search"):
        n, b, groups = case["n"], case["batch"], _ceil(dim, case["group"])
        held = n * (dim / 2 + groups * (3 if case["zeros"] else 2)) + b * dim * size[case["x"]]
        if op == "products":
            made = b * n * size[case["out"]]
        else:
            made = b * case["k"] * 12 + (4 * n if case["metric"] == "l2" else 0)
        return {"bytes": held + made, "flops": 2.0 * b * n * dim}
    if op == "append":
        rows = sum(_ragged(case["count"], case["seqs"]))
        held = rows * (dim / 2 + _ceil(dim, case["group"]) * (3 if case["zeros"] else 2))
        return {"bytes": rows * dim * size[case["x"]] + 2 * held + 4 * rows + 4 * rows * dim, "flops": 4.0 * rows * dim}
    row = 2 * dim + 4
    if op == "copy":
        return {"bytes": 2.0 * case["pages"] * (case["page_rows"] * row + 4), "flops": 0.0}
    if op == "fork":
        lengths = _ragged(case["count"], case["parents"])
        moved = 0
        for i in range(case["children"]):
            n = lengths[i % case["parents"]]
            moved += 2 * (n % case["page_rows"]) * row + 5 * 4 * _ceil(n, case["page_rows"])
        return {"bytes": float(moved), "flops": 0.0}
    rows = sum(_ragged(case["count"], case["seqs"]))
    return {"bytes": rows * (1 + 2 * case["keep"] * row), "flops": 0.0}


# ------------------------------------------------------------------ inputs
def _rand(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _held(n, case, g):
    """n rows in 4 bits: bell-shaped codes, as quantised embeddings have, scales that
    make the rows' lengths about 1, zero points near the middle."""
    dim, group = case["dim"], case["group"]
    groups, padded = _ceil(dim, group), 32 * _ceil(dim, 32)
    c = torch.randn(n, padded, device=DEVICE, generator=g, dtype=torch.float16).mul_(2.6).add_(8).round_().clamp_(0, 15)
    c[:, dim:] = 0
    c = c.to(torch.uint8)
    codes = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = (torch.randn(n, groups, device=DEVICE, generator=g).mul_(0.2).exp_() * (0.38 / dim ** 0.5)).half()
    zeros = torch.randint(6, 11, (n, groups), device=DEVICE, generator=g, dtype=torch.uint8) if case["zeros"] else None
    return codes, scales, zeros


def _paged(t, pages, page_rows, total):
    """Rows t on the given pages of a new pool of `total` pages."""
    if t is None:
        return None
    pool = torch.zeros(total * page_rows, *t.shape[1:], dtype=t.dtype, device=t.device)
    at = torch.arange(t.shape[0], device=t.device)
    pool[pages[at // page_rows] * page_rows + at % page_rows] = t
    return pool.view(total, page_rows, *t.shape[1:])


def _package():
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuvs-silicon_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import cuvs_b200

    return cuvs_b200


def _store(case, lengths, spare, others, g):
    """Table, lengths and counts of references of a store whose first sequences have the
    given lengths on pages in no order, `spare` empty sequences, and one more that holds
    `others` pages in among them."""
    page_rows = case["page_rows"]
    need = [_ceil(n, page_rows) for n in lengths]
    need.append(others)
    free = sum(need) + 64
    total = sum(need) + free
    order = torch.randperm(total, device=DEVICE, generator=g)
    count = len(lengths) + spare + 1
    table = torch.full((count, max(need) + 2), -1, dtype=torch.int32, device=DEVICE)
    rows = torch.zeros(count, dtype=torch.int32, device=DEVICE)
    refs = torch.zeros(total, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        s = i if i < len(lengths) else count - 1
        table[s, :n] = order[at:at + n].int()
        rows[s] = lengths[i] if i < len(lengths) else n * page_rows
        at += n
    refs[order[:at]] = 1
    return {"table": table, "rows": rows, "refs": refs}


def _list(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = _rand(seed)
    op, dim, page_rows = case["op"], case["dim"], case["page_rows"]
    state = {"case": case}
    if op in ("products", "search"):
        n = case["n"]
        codes, scales, zeros = _held(n, case, g)
        x = torch.randn(case["batch"], dim, device=DEVICE, generator=g)
        if op == "search":
            x = x / dim ** 0.5  # about as long as the rows
        state["x"] = x.to(TYPES[case["x"]])
        norms = None
        if op == "search" and case["metric"] == "l2":
            norms = torch.cat([_values(codes[i:i + 65536], scales[i:i + 65536], None if zeros is None else zeros[i:i + 65536],
                                       dim, case["group"], torch.float32).square().sum(1) for i in range(0, n, 65536)])
        if page_rows:
            need = _ceil(n, page_rows)
            table = torch.full((2, need + 1), -1, dtype=torch.int32, device=DEVICE)
            pages = torch.randperm(need + 8, device=DEVICE, generator=g)[:need]
            table[1, :need] = pages.int()
            refs = torch.zeros(need + 8, dtype=torch.int32, device=DEVICE)
            refs[pages] = 1
            state |= {"table": table, "rows": _list([0, n]), "refs": refs}
            codes, scales, zeros, norms = (_paged(t, pages, page_rows, need + 8) for t in (codes, scales, zeros, norms))
        state |= {"codes": codes, "scales": scales, "zeros": zeros, "norms": norms}
    elif op == "append":
        counts = _ragged(case["count"], case["seqs"])
        need = sum(_ceil(n, page_rows) for n in counts)
        state |= _store(case, [], case["seqs"], need + 5, g)
        total, groups = state["refs"].numel(), _ceil(dim, case["group"])

        def pool(*tail, dtype):
            return torch.zeros(total, page_rows, *tail, dtype=dtype, device=DEVICE)

        state["codes"] = pool(16 * _ceil(dim, 32), dtype=torch.uint8)
        state["scales"] = pool(groups, dtype=torch.float16)
        state["zeros"] = pool(groups, dtype=torch.uint8) if case["zeros"] else None
        state["norms"] = pool(dtype=torch.float32)
        state["seqs"], state["counts"] = _list(list(range(case["seqs"]))), _list(counts)
        state["x"] = (torch.randn(sum(counts), dim, device=DEVICE, generator=g) / dim ** 0.5).to(TYPES[case["x"]])
    else:
        if op == "copy":
            n = case["pages"]
            total = 2 * n + 5
            order = torch.randperm(total, device=DEVICE, generator=g).int()
            state["sources"], state["targets"] = order[:n].clone(), order[n:2 * n].clone()
            state |= {"table": torch.full((1, 1), -1, dtype=torch.int32, device=DEVICE), "rows": _list([0]),
                      "refs": torch.zeros(total, dtype=torch.int32, device=DEVICE)}
        elif op == "fork":
            p, c = case["parents"], case["children"]
            lengths = _ragged(case["count"], p)
            state |= _store(case, lengths, c, c, g)
            state["parents"], state["children"] = _list([i % p for i in range(c)]), _list([p + i for i in range(c)])
        else:
            lengths = _ragged(case["count"], case["seqs"])
            state |= _store(case, lengths, case["seqs"], 5, g)
            state["sources"] = _list(list(range(case["seqs"])))
            state["targets"] = _list([case["seqs"] + i for i in range(case["seqs"])])
            state["keep"] = torch.rand(case["seqs"], case["count"], device=DEVICE, generator=g) < case["keep"]
        total = state["refs"].numel()
        state["pool"] = torch.randn(total, page_rows, dim, dtype=torch.float16, device=DEVICE, generator=g)
        state["norms"] = torch.rand(total, page_rows, device=DEVICE, generator=g)
    if own:
        # the handles that a program keeps: they hold the tensors above, nothing else
        package = _package()
        if "codes" not in state:
            state["pages"] = package.Pages(state["table"], state["rows"], state["refs"], [state["pool"], state["norms"]])
        else:
            held = [t for t in (state["codes"], state["scales"], state["zeros"], state["norms"]) if t is not None]
            pages = package.Pages(state["table"], state["rows"], state["refs"], held) if "table" in state else None
            state["held"] = package.Q4Rows(state["codes"], state["scales"], dim, case["group"], zeros=state["zeros"],
                                           norms=state["norms"], pages=pages)
            state["pages"] = pages
    return state


# ------------------------------------------------------------- plain forms
def _values(codes, scales, zeros, dim, group, dtype):
    """What rows in 4 bits stand for."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :dim].to(dtype)
    c = c - (8 if zeros is None else zeros.to(dtype).repeat_interleave(group, dim=-1)[..., :dim])
    return c * scales.to(dtype).repeat_interleave(group, dim=-1)[..., :dim]


def _rows_of(state, n):
    """The codes, scales and zero points of the n rows, out of their pages where they are in pages."""
    held = state["codes"], state["scales"], state["zeros"]
    r = state["case"]["page_rows"]
    if not r:
        return held
    pages = state["table"][1, :_ceil(n, r)].long()
    return tuple(None if t is None else t[pages].flatten(0, 1)[:n] for t in held)


def _free(state, seqs):
    seqs = seqs.long()
    pages = state["table"][seqs].flatten()
    held = (pages >= 0).int()
    state["refs"].index_add_(0, pages.clamp(min=0).long(), -held)
    state["table"][seqs] = -1
    state["rows"][seqs] = 0


def _fresh(state, wanted):
    """The lowest-numbered free pages, given out where `wanted` [sequences, columns] is true, in order."""
    pages = (state["refs"] == 0).nonzero().flatten()
    got = pages[(wanted.flatten().cumsum(0) - 1).clamp(min=0)].view(wanted.shape)
    state["refs"][got[wanted]] = 1
    return torch.where(wanted, got, -1)


def _take_pages(state, seqs, counts):
    """Pages for `counts` rows of each of the empty sequences."""
    r, seqs = state["case"]["page_rows"], seqs.long()
    wanted = torch.arange(state["table"].shape[1], device=DEVICE) < ((counts + r - 1) // r)[:, None]
    state["table"][seqs] = _fresh(state, wanted).int()
    state["rows"][seqs] = counts.int()


def _places(state, seqs, counts, total):
    """Where in the pools, counted in rows, the rows of the sequences lie, one after another."""
    r = state["case"]["page_rows"]
    which = torch.repeat_interleave(seqs.long(), counts.long(), output_size=total)
    first = torch.repeat_interleave(counts.cumsum(0) - counts, counts.long(), output_size=total)
    at = torch.arange(total, device=DEVICE) - first
    return state["table"][which, at // r].long() * r + at % r


def _nearest(q, t):
    """The quotient q / t to the nearest whole number, ties to even; 0 where t is 0 or not finite."""
    quotient = q.double() / t.double()
    return torch.where((t != 0) & torch.isfinite(t), quotient, 0.0).round()


def _quantised(v, group, with_zeros):
    """Codes (one to a value), scales and zero points of rows v."""
    rows, dim = v.shape
    groups = _ceil(dim, group)
    v = torch.nn.functional.pad(v.float(), (0, groups * group - dim)).view(rows, groups, group)
    divisor = torch.tensor(15.0 if with_zeros else 7.0, device=DEVICE)
    if with_zeros:
        low, high = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scales = ((high - low) / divisor).half()
        zeros = _nearest(-low, scales.float()).clamp(0, 15)
    else:
        scales = (v.abs().amax(-1) / divisor).half()
        zeros = torch.full_like(scales, 8.0, dtype=torch.float64)
    codes = (_nearest(v, scales.float()[..., None]) + zeros[..., None]).clamp(0, 15)
    return codes.to(torch.uint8).view(rows, -1)[:, :dim], scales, zeros.to(torch.uint8)


def _run_plain(state):
    case = state["case"]
    op, dim, r = case["op"], case["dim"], case["page_rows"]
    if op == "products":
        held = _values(*_rows_of(state, case["n"]), dim, case["group"], torch.float32)
        return (state["x"].float() @ held.T).to(TYPES[case["out"]])
    if op == "search":
        # in 64 bits: near neighbours lie close together, and their order is the result
        x = state["x"].double()
        held = _values(*_rows_of(state, case["n"]), dim, case["group"], torch.float64)
        key = x @ held.T
        if case["metric"] == "l2":
            key = x.square().sum(1)[:, None] - 2 * key + held.square().sum(1)
        else:
            key = -key
        key, order = key.sort(dim=1, stable=True)
        k = min(case["k"], case["n"])
        key = torch.nn.functional.pad(key[:, :k], (0, case["k"] - k), value=float("inf"))
        order = torch.nn.functional.pad(order[:, :k], (0, case["k"] - k), value=-1)
        return {"neighbors": order, "distances": (key if case["metric"] == "l2" else -key).float()}
    if op == "append":
        _free(state, state["seqs"])
        counts, total = state["counts"].long(), state["x"].shape[0]
        _take_pages(state, state["seqs"], counts)
        at = _places(state, state["seqs"], counts, total)
        c, scales, zeros = _quantised(state["x"], case["group"], case["zeros"])
        c = torch.nn.functional.pad(c, (0, 2 * state["codes"].shape[-1] - dim))
        state["codes"].flatten(0, 1)[at] = c[:, 0::2] | (c[:, 1::2] << 4)
        state["scales"].flatten(0, 1)[at] = scales
        if case["zeros"]:
            state["zeros"].flatten(0, 1)[at] = zeros
        kept = [None if t is None else t.flatten(0, 1)[at] for t in (state["codes"], state["scales"], state["zeros"])]
        values = _values(*kept, dim, case["group"], torch.float32)
        state["norms"].view(-1)[at] = values.square().sum(1)
        return _outputs(state, values)
    if op == "copy":
        s, t = state["sources"].long(), state["targets"].long()
        state["pool"][t] = state["pool"][s]
        state["norms"][t] = state["norms"][s]
    elif op == "fork":
        _free(state, state["children"])
        parents, children = state["parents"].long(), state["children"].long()
        lengths = state["rows"][parents].long()
        full, tail = lengths // r, lengths % r
        columns = torch.arange(state["table"].shape[1], device=DEVICE)
        theirs = state["table"][parents]
        shared = torch.where(columns < full[:, None], theirs, -1)
        state["refs"].index_add_(0, shared.clamp(min=0).flatten().long(), (shared >= 0).flatten().int())
        new = _fresh(state, (columns == full[:, None]) & (tail > 0)[:, None])
        state["table"][children] = torch.maximum(shared, new.int())
        state["rows"][children] = lengths.int()
        slot = torch.arange(r, device=DEVICE)
        child, slot = (slot < tail[:, None]).nonzero(as_tuple=True)
        source = theirs[child, full[child]].long()
        target = new[child, full[child]]
        state["pool"][target, slot] = state["pool"][source, slot]
        state["norms"][target, slot] = state["norms"][source, slot]
    else:
        _free(state, state["targets"])
        lengths = state["rows"][state["sources"].long()]
        keep = state["keep"] & (torch.arange(state["keep"].shape[1], device=DEVICE) < lengths[:, None])
        counts = keep.sum(1)
        _take_pages(state, state["targets"], counts)
        which, at = keep.nonzero(as_tuple=True)
        source = state["table"][state["sources"].long()[which], at // r].long() * r + at % r
        target = _places(state, state["targets"], counts, source.numel())
        state["pool"].flatten(0, 1)[target] = state["pool"].flatten(0, 1)[source]
        state["norms"].view(-1)[target] = state["norms"].view(-1)[source]
    return _outputs(state)


def _outputs(state, values=None):
    """The store as a pass leaves it."""
    if values is None:
        names = ("table", "rows", "refs", "pool", "norms")
    else:
        names = ("table", "rows", "refs", "scales", "norms") + (("zeros",) if state["zeros"] is not None else ())
    got = {name: state[name] for name in names}
    if values is not None:
        got["values"] = values
    return got


# --------------------------------------------------------- the framework's
def _run_own(state):
    case = state["case"]
    op, pages = case["op"], state["pages"]
    if op == "products":
        return state["held"].products(state["x"], seq=1 if pages else None, count=case["n"], dtype=TYPES[case["out"]])
    if op == "search":
        metric = 0 if case["metric"] == "l2" else 1  # METRIC_L2_EXPANDED, METRIC_INNER_PRODUCT
        neighbors, distances = state["held"].search(state["x"], case["k"], metric=metric, seq=1 if pages else None,
                                                    count=case["n"])
        return {"neighbors": neighbors, "distances": distances}
    if op == "append":
        pages.free(state["seqs"])
        state["held"].append(state["seqs"], state["counts"], state["x"])
        return _outputs(state, state["held"].read(state["seqs"], state["counts"], state["x"].shape[0]))
    if op == "copy":
        pages.copy(state["sources"], state["targets"])
    elif op == "fork":
        pages.free(state["children"])
        pages.fork(state["parents"], state["children"])
    else:
        pages.free(state["targets"])
        pages.compact(state["sources"], state["targets"], state["keep"])
    return _outputs(state)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------ in 64 bits
def _exact_rows(state, first, last):
    """Rows [first, last) as float64, looked up and taken apart one by one."""
    case = state["case"]
    dim, group, r = case["dim"], case["group"], case["page_rows"]
    at = torch.arange(first, last, device=DEVICE)
    if r:
        at = state["table"][1].long()[torch.div(at, r, rounding_mode="floor")] * r + at.remainder(r)
    codes = state["codes"].reshape(-1, state["codes"].shape[-1]).index_select(0, at).double()
    scales = state["scales"].reshape(-1, state["scales"].shape[-1]).index_select(0, at).double()
    column = torch.arange(dim, device=DEVICE)
    byte = codes.index_select(1, column // 2)
    high = torch.floor(byte / 16)
    code = torch.where((column % 2).bool(), high, byte - 16 * high)
    if state["zeros"] is None:
        code -= 8
    else:
        zeros = state["zeros"].reshape(-1, state["zeros"].shape[-1]).index_select(0, at).double()
        code -= zeros.index_select(1, column // group)
    return code * scales.index_select(1, column // group)


def _exact_quantised(v, group, with_zeros):
    """(values, scales, norms) of rows v (float64) after quantisation."""
    values, scales = torch.zeros_like(v), []
    for first in range(0, v.shape[1], group):
        part = v[:, first:first + group]
        if with_zeros:
            low = torch.minimum(part.min(1).values, torch.zeros_like(part[:, 0]))
            high = torch.maximum(part.max(1).values, torch.zeros_like(part[:, 0]))
            # the range is a 32-bit number, as the scale before its last rounding is
            s = ((high - low).float().double() / 15.0).float().half().double()
        else:
            s = (part.abs().max(1).values / 7.0).float().half().double()
        over = 1.0 / torch.where(s > 0, s, torch.ones_like(s))
        lowest, highest = torch.full_like(s, -8.0), torch.full_like(s, 7.0)
        if with_zeros:
            zero = torch.clamp(torch.round(-low / torch.where(s > 0, s, torch.ones_like(s))), 0, 15)
            lowest, highest = -zero, 15 - zero
        q = torch.round(part * over[:, None])
        # a product with the reciprocal may miss a tie: the remainder decides
        left = part - q * s[:, None]
        half = s[:, None] / 2
        odd = q.remainder(2) == 1
        q = q + ((left > half) | ((left == half) & odd)).double() - ((left < -half) | ((left == -half) & odd)).double()
        q = torch.minimum(torch.maximum(q, lowest[:, None]), highest[:, None])
        values[:, first:first + group] = torch.where(s[:, None] > 0, q * s[:, None], torch.zeros_like(q))
        scales.append(s)
    return values, torch.stack(scales, 1), values.square().sum(1)


def exact(case, seed):
    state = prepare(case, seed)
    op, r = case["op"], case["page_rows"]
    nothing = {"table": None, "rows": None, "refs": None}
    if op in ("products", "search"):
        n, x = case["n"], state["x"].double()
        keys = []
        for first in range(0, n, 50000):
            rows = _exact_rows(state, first, min(n, first + 50000))
            if op == "search" and case["metric"] == "l2":
                keys.append(torch.stack([-(rows - q).square().sum(1) for q in x]))
            else:
                keys.append(torch.stack([(rows * q).sum(1) for q in x]))
        key = torch.cat(keys, 1)
        if op == "products":
            return key
        best = torch.full((x.shape[0], case["k"]), -float("inf"), dtype=torch.float64, device=DEVICE)
        k = min(case["k"], n)
        best[:, :k] = key.topk(k, dim=1).values
        return {"neighbors": None, "distances": -best if case["metric"] == "l2" else best}
    free = [p for p, refs in enumerate(state["refs"].tolist()) if refs == 0]
    if op == "append":
        values, scales, norms = _exact_quantised(state["x"].double(), case["group"], case["zeros"])
        pool_scales, pool_norms = state["scales"].double(), state["norms"].double()
        first = 0
        for count in state["counts"].tolist():
            for at in range(0, count, r):
                page, m = free.pop(0), min(r, count - at)
                pool_scales[page, :m] = scales[first + at:first + at + m]
                pool_norms[page, :m] = norms[first + at:first + at + m]
            first += count
        return nothing | {"scales": pool_scales, "norms": pool_norms, "zeros": None, "values": values}
    pools = {"pool": state["pool"].double(), "norms": state["norms"].double()}
    table, lengths = state["table"].tolist(), state["rows"].tolist()
    for t in pools.values():
        before = t.clone()
        fresh = iter(free)
        if op == "copy":
            for s, d in zip(state["sources"].tolist(), state["targets"].tolist()):
                t[d] = before[s]
        elif op == "fork":
            for s in state["parents"].tolist():
                tail = lengths[s] % r
                if tail:
                    t[next(fresh), :tail] = before[table[s][lengths[s] // r], :tail]
        else:
            for i, s in enumerate(state["sources"].tolist()):
                flat = before[table[s][:_ceil(lengths[s], r)]].flatten(0, 1)[:lengths[s]]
                flat = flat[state["keep"][i, :lengths[s]]]
                for at in range(0, flat.shape[0], r):
                    t[next(fresh), :min(r, flat.shape[0] - at)] = flat[at:at + r]
    return nothing | pools
