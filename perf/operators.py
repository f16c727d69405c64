"""Cases of the adapter, top-logit and distillation operators: what is computed, on which sizes, and how a program calls it.

`own = False` computes the operators by elementary torch operations in 32 bits; `own = True` calls the entry points of
libkaldi_hip.so (include/kaldi_hip.h) on the same tensors, on torch's current stream.
"""
import ctypes
import math
import random

import torch

own = False

# Sizes: the 1320 -> 7 x 2048 -> 9000 and 440 -> 4 x 1024 -> 1483 networks, bunches of 256 frames, forward batches of
# about 4096 frames, and the 70001-output layer that the tests of extreme shapes hold.


def listed():
    return [
        # one frame of a live stream through a hidden layer with its speaker's adapter
        {"name": "adapt one frame", "op": "adapt", "rows": 1, "I": 2048, "O": 2048, "num": 8, "rank": 16, "ragged": False,
         "mix": "segments", "none": 0.0, "act": True},
        # one frame of each of 64 live streams, every one with another speaker's adapter, some without; odd output width
        {"name": "adapt 64 streams", "op": "adapt", "rows": 64, "I": 1024, "O": 1483, "num": 200, "rank": 32, "ragged": True,
         "mix": "each", "none": 0.05, "act": False},
        # a frame-shuffled training bunch of 40 speakers; the bunch's grouping is part of the pass
        {"name": "adapt bunch", "op": "adapt", "rows": 256, "I": 2048, "O": 2048, "num": 40, "rank": 16, "ragged": False,
         "mix": "shuffled", "none": 0.0, "act": True},
        # a forward batch of whole utterances
        {"name": "adapt batch", "op": "adapt", "rows": 4096, "I": 2048, "O": 2048, "num": 24, "rank": 16, "ragged": False,
         "mix": "segments", "none": 0.1, "act": True},
        # the training bunch's backward pass: error of the layer below and both gradients
        {"name": "adapt-backward bunch", "op": "adapt-backward", "rows": 256, "I": 2048, "O": 2048, "num": 40, "rank": 16,
         "ragged": False, "mix": "shuffled", "none": 0.0, "eout": True},
        # adaptation on whole utterances, a quarter of the frame cache at once, larger and uneven ranks
        {"name": "adapt-backward utterances", "op": "adapt-backward", "rows": 8192, "I": 2048, "O": 2048, "num": 16, "rank": 32,
         "ragged": True, "mix": "segments", "none": 0.05, "eout": True},
        # the teacher's largest logits of one live frame
        {"name": "top one frame", "op": "top", "rows": 1, "C": 9000, "K": 8, "masked": 0.0},
        # a forward batch of the teacher, as it is stored for training
        {"name": "top batch", "op": "top", "rows": 4096, "C": 9000, "K": 32, "masked": 0.0},
        # a bunch of the widest output layer, odd rows, a part of the outputs masked out
        {"name": "top wide", "op": "top", "rows": 256, "C": 70001, "K": 64, "masked": 0.3},
        # the loss and its gradient on a training bunch, soft and hard targets mixed
        {"name": "distill bunch", "op": "distill", "rows": 256, "C": 1483, "K": 8, "temperature": 2.0, "hard": 0.5, "diff": True},
        # the same towards the stored table of a forward batch, soft targets only
        {"name": "distill batch", "op": "distill", "rows": 4096, "C": 9000, "K": 32, "temperature": 2.0, "hard": 0.0, "diff": True},
        # cross-validation: the loss alone
        {"name": "distill validation", "op": "distill", "rows": 1999, "C": 9000, "K": 20, "temperature": 1.0, "hard": 0.3,
         "diff": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adapt", "adapt-backward", "top", "distill"])
    if op in ("adapt", "adapt-backward"):
        back = op == "adapt-backward"
        rows = _log_int(rng, 1, 8192 if back else 4096)
        case = {"op": op, "rows": rows, "I": _log_int(rng, 40, 2048), "O": _log_int(rng, 40, 2048), "num": _log_int(rng, 1, 200),
                "rank": _log_int(rng, 1, 32 if back else 64), "ragged": rng.random() < 0.5,
                "mix": rng.choice(["segments", "shuffled", "each"]), "none": rng.choice([0.0, 0.05, 0.5])}
        if case["mix"] == "each" and rows > 256:
            case["mix"] = "shuffled"
        if back:
            case["eout"] = rng.random() < 0.8
        else:
            case["act"] = rng.random() < 0.5
        return case
    C = _log_int(rng, 100, 70001)
    rows = _log_int(rng, 1, max(1, min(4096, 36864000 // (C + C // 4))))
    if op == "top":
        return {"op": op, "rows": rows, "C": C, "K": _log_int(rng, 1, min(64, C)), "masked": rng.choice([0.0, 0.3, 0.9])}
    return {"op": op, "rows": rows, "C": C, "K": _log_int(rng, 1, min(64, C)), "temperature": rng.choice([1.0, 2.0, 3.5]),
            "hard": rng.choice([0.0, 0.3, 0.5, 1.0]), "diff": rng.random() < 0.7}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _pitched(rows, cols, dtype=torch.float32):
    """rows x cols with rows that start on 256-byte boundaries, as hipK_malloc_pitch lays matrices out."""
    return torch.zeros((max(rows, 1), (cols + 63) // 64 * 64), dtype=dtype, device="cuda")[:rows, :cols]


def _put(a):
    m = _pitched(a.shape[0], a.shape[1], a.dtype)
    m.copy_(a)
    return m


def _inputs(case, seed):
    """The inputs of a case, the same for every side: from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    def randint(lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

    R, s = case["rows"], {}
    if case["op"] in ("adapt", "adapt-backward"):
        I, O, num, rank = case["I"], case["O"], case["num"], case["rank"]
        # a hidden layer's input: activations of the sigmoid layer below
        s["in"] = _put(torch.sigmoid(2.0 * randn(R, I)))
        s["W"] = _put(0.1 * randn(O, I))
        s["bias"] = -4.1 + 0.2 * rand(O)
        # the adapters' ranks belong to the case: outputs of every seed have the same shapes
        sizes = random.Random(num * 131 + rank)
        ranks = torch.tensor([sizes.randint(1, rank) if case["ragged"] else rank for _ in range(num)], device="cuda")
        s["begin"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), ranks.cumsum(0)]).to(torch.int32)
        total = int(s["begin"][-1])
        s["down"], s["up"] = _put(randn(total, I) / math.sqrt(I)), _put(0.3 * randn(total, O))
        s["scale"] = 0.5 + 1.5 * rand(num)
        if case["mix"] == "each":  # another adapter for every row as far as there are any
            ids = torch.randperm(num, generator=gen, device="cuda").repeat((R + num - 1) // num)[:R]
        elif case["mix"] == "segments":  # utterances, each of one speaker
            cuts = (rand(R) < 1.0 / 170).cumsum(0)
            ids = randint(0, num, (R + 1,))[cuts]
        else:
            ids = randint(0, num, (R,))
        ids = torch.where(rand(R) < case["none"], torch.full_like(ids, -1), ids) if case["mix"] != "segments" else \
            torch.where((rand(num) < case["none"])[ids], torch.full_like(ids, -1), ids)
        s["ids"] = ids.to(torch.int32)
        if case["op"] == "adapt-backward":
            # what the forward pass of the same bunch left behind: the grouping and the narrow products
            key = torch.where(ids < 0, torch.full_like(ids, num), ids)
            s["order"] = torch.argsort(key, stable=True).to(torch.int32)
            s["row_begin"] = torch.searchsorted(key.sort().values, torch.arange(num + 1, device="cuda")).to(torch.int32)
            s["e"] = _put(0.05 * randn(R, O))
            col = torch.arange(rank, device="cuda")
            have = (ids >= 0)[:, None] & (col < ranks[ids.clamp(min=0)][:, None])
            s["t"] = _put(torch.where(have, randn(R, rank), torch.zeros((), device="cuda")))
        return s
    C, K = case["C"], case["K"]
    if case["op"] == "top":
        z = 3.0 * randn(R, C)
        if case["masked"]:
            z = torch.where(rand(R, C) < case["masked"], torch.full((), -math.inf, device="cuda"), z)
        # values as they come out of a half-precision table: ties occur
        s["z"] = _put(z.half().float() if K % 2 or case["masked"] else z)
        return s
    teacher = 3.0 * randn(R, C)
    s["z"] = _put(teacher + randn(R, C))
    val, idx = teacher.topk(K, dim=1)
    kept = randint(max(1, K // 2), K + 1, (R, 1))
    kept = torch.where(rand(R, 1) < 0.03, torch.zeros_like(kept), kept)  # rows that the teacher has nothing for
    gone = torch.arange(K, device="cuda")[None, :] >= kept
    s["idx"] = _put(torch.where(gone, torch.full_like(idx, -1), idx).to(torch.int32))
    s["val"] = _put(val)
    s["label"] = torch.where(rand(R) < 0.7, teacher.argmax(1), randint(-1, C, (R,))).to(torch.int32)
    s["weight"] = torch.where(rand(R) < 0.05, torch.zeros((), device="cuda"), 0.5 + rand(R))
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    from kaldi_amd import hip
    hip.init(torch.cuda.current_device())
    s["call"], s["MatrixDim"] = hip.call, hip.MatrixDim
    R = case["rows"]
    if case["op"] in ("adapt", "adapt-backward"):
        s["adapters"] = hip.Adapters(case["num"], case["rank"], s["down"].shape[0], s["begin"].data_ptr(), s["scale"].data_ptr(),
                                     s["down"].data_ptr(), s["down"].stride(0), s["up"].data_ptr(), s["up"].stride(0))
        if case["op"] == "adapt":
            s["t"], s["out"] = _pitched(R, case["rank"]), _pitched(R, case["O"])
            s["order"] = torch.zeros(R, dtype=torch.int32, device="cuda")
            s["row_begin"] = torch.zeros(case["num"] + 1, dtype=torch.int32, device="cuda")
        else:
            s["u"], s["eout"] = _pitched(R, case["rank"]), _pitched(R, case["I"])
            s["gdown"], s["gup"] = _pitched(*s["down"].shape), _pitched(*s["up"].shape)
    elif case["op"] == "top":
        s["idx"], s["val"] = _pitched(R, case["K"], torch.int32), _pitched(R, case["K"])
        s["lse"] = torch.zeros(R, device="cuda")
    else:
        s["row_loss"] = torch.zeros(R, device="cuda")
        s["diff"] = _pitched(R, case["C"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(s):
    op = s["case"]["op"].replace("-", "_")
    return globals()[("_own_" if own else "_plain_") + op](s)


def _stream():
    # torch's default stream is the null stream, whose handle is 1 (hipStreamLegacy) for callers that must name it
    return torch.cuda.current_stream().cuda_stream or 1


def _own_adapt(s):
    c, p, st = s["case"], torch.Tensor.data_ptr, _stream()
    order = None
    if c["mix"] == "shuffled":
        order = p(s["order"])
        s["call"]("hipI32_adapter_plan", st, p(s["ids"]), c["rows"], c["num"], order, p(s["row_begin"]))
    s["call"]("hipF_adapter_forward", st, 1 if c["act"] else 0, c["rows"], c["O"], c["I"], p(s["in"]), s["in"].stride(0),
              p(s["W"]), s["W"].stride(0), p(s["bias"]), ctypes.byref(s["adapters"]), p(s["ids"]), order,
              p(s["t"]), s["t"].stride(0), p(s["out"]), s["out"].stride(0))
    return {"out": s["out"], "t": s["t"], **({"order": s["order"], "row_begin": s["row_begin"]} if order else {})}


def _own_adapt_backward(s):
    c, p = s["case"], torch.Tensor.data_ptr
    y = s["in"] if c["eout"] else None
    s["call"]("hipF_adapter_backward", _stream(), c["rows"], c["O"], c["I"], p(s["e"]), s["e"].stride(0), p(s["in"]),
              s["in"].stride(0), p(s["W"]), s["W"].stride(0), ctypes.byref(s["adapters"]), p(s["ids"]), p(s["order"]),
              p(s["row_begin"]), p(s["t"]), s["t"].stride(0), p(s["u"]), s["u"].stride(0), p(y) if c["eout"] else None,
              s["in"].stride(0), p(s["eout"]) if c["eout"] else None, s["eout"].stride(0), p(s["gdown"]), s["gdown"].stride(0),
              p(s["gup"]), s["gup"].stride(0))
    return {"u": s["u"], "gdown": s["gdown"], "gup": s["gup"], **({"eout": s["eout"]} if c["eout"] else {})}


def _own_top(s):
    c, p, z = s["case"], torch.Tensor.data_ptr, s["z"]
    s["call"]("hipF_row_top", _stream(), p(z), s["MatrixDim"](c["rows"], c["C"], z.stride(0)), c["K"], p(s["idx"]),
              s["idx"].stride(0), p(s["val"]), s["val"].stride(0), p(s["lse"]))
    return {"idx": s["idx"], "val": s["val"], "lse": s["lse"]}


def _own_distill(s):
    c, p, z = s["case"], torch.Tensor.data_ptr, s["z"]
    s["call"]("hipF_distill_eval", _stream(), p(z), s["MatrixDim"](c["rows"], c["C"], z.stride(0)), p(s["idx"]),
              s["idx"].stride(0), p(s["val"]), s["val"].stride(0), c["K"], p(s["label"]), p(s["weight"]), c["temperature"],
              c["hard"], p(s["diff"]) if c["diff"] else None, s["diff"].stride(0), p(s["row_loss"]), None)
    return {"row_loss": s["row_loss"], **({"diff": s["diff"]} if c["diff"] else {})}


# The plain forms.


def _columns(s):
    """Which rows of the stacks a row's adapter holds, and which of `rank` places are there."""
    c = s["case"]
    on = (s["ids"] >= 0) & (s["ids"] < c["num"])
    g = torch.where(on, s["ids"], torch.zeros_like(s["ids"])).long()
    k = torch.arange(c["rank"], device="cuda")
    there = on[:, None] & (k < (s["begin"][g + 1] - s["begin"][g])[:, None])
    return torch.where(there, s["begin"][g][:, None] + k, torch.zeros_like(k)), there, s["scale"][g][:, None]


def _narrow(x, side, at, there, scale):
    # the products with all adapters' rows at once, then each row's own
    return torch.where(there, scale * (x @ side.t()).gather(1, at), torch.zeros((), device="cuda"))


def _spread(t, total, at):
    # each row's narrow product at its adapter's columns, zero elsewhere: the sums over one adapter become one product
    return torch.zeros((t.shape[0], total), device="cuda").scatter_add_(1, at, t)


def _plain_adapt(s):
    c, (at, there, scale) = s["case"], _columns(s)
    t = _narrow(s["in"], s["down"], at, there, scale)
    out = s["in"] @ s["W"].t() + s["bias"] + _spread(t, s["up"].shape[0], at) @ s["up"]
    out = torch.sigmoid(out) if c["act"] else out
    if c["mix"] != "shuffled":
        return {"out": out, "t": t}
    key = torch.where(s["ids"] < 0, torch.full_like(s["ids"], c["num"]), s["ids"])
    key, order = torch.sort(key, stable=True)
    begin = torch.searchsorted(key, torch.arange(c["num"] + 1, device="cuda", dtype=key.dtype))
    return {"out": out, "t": t, "order": order.to(torch.int32), "row_begin": begin.to(torch.int32)}


def _plain_adapt_backward(s):
    c, (at, there, scale), total = s["case"], _columns(s), s["up"].shape[0]
    u = _narrow(s["e"], s["up"], at, there, scale)
    wide = _spread(u, total, at)
    answer = {"u": u, "gdown": wide.t() @ s["in"], "gup": _spread(s["t"], total, at).t() @ s["e"]}
    if c["eout"]:
        answer["eout"] = (s["e"] @ s["W"] + wide @ s["down"]) * (s["in"] * (1.0 - s["in"]))
    return answer


def _plain_top(s):
    c, z = s["case"], s["z"]
    # unique keys that order by value, then by column: the 32 bits of the value made comparable above the column's
    bits = (z + 0.0).view(torch.int32).to(torch.int64)
    key = (torch.where(bits < 0, -2147483649 - bits, bits) << 32) + (c["C"] - 1 - torch.arange(c["C"], device="cuda"))
    top = key.topk(c["K"], dim=1).values
    idx = c["C"] - 1 - (top & 0xFFFFFFFF)
    peak = z.max(1, keepdim=True).values
    peak = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)  # (a row with nothing left: log 0)
    return {"idx": idx.to(torch.int32), "val": z.gather(1, idx), "lse": peak[:, 0] + torch.exp(z - peak).sum(1).log()}


def _log_softmax(z):
    z = z - z.max(1, keepdim=True).values
    return z - torch.exp(z).sum(1, keepdim=True).log()


def _plain_distill(s):
    c, z = s["case"], s["z"]
    T, hard, C = c["temperature"], c["hard"], c["C"]
    there = (s["idx"] >= 0) & (s["idx"] < C)
    at = torch.where(there, s["idx"], torch.zeros_like(s["idx"])).long()
    some = there.any(1, keepdim=True)
    v = torch.where(there, s["val"] / T, torch.full((), -math.inf, device="cuda"))
    logq = torch.where(there, _log_softmax(torch.where(some, v, torch.zeros_like(v))), torch.zeros_like(v))
    q = torch.where(there, torch.exp(logq), torch.zeros_like(v))
    logp = _log_softmax(z / T)
    soft = T * T * (q * (logq - logp.gather(1, at))).sum(1)
    labelled = (s["label"] >= 0) & (s["label"] < C)
    label = torch.where(labelled, s["label"], torch.zeros_like(s["label"])).long()[:, None]
    logp1 = _log_softmax(z)
    w = s["weight"]
    ce = torch.where(labelled, -logp1.gather(1, label)[:, 0], torch.zeros_like(w))
    row_loss = w * ((1.0 - hard) * soft + hard * ce)
    answer = {"row_loss": row_loss}
    if c["diff"]:
        diff = ((1.0 - hard) * T * w)[:, None] * (torch.exp(logp) * some)
        diff.scatter_add_(1, at, ((hard - 1.0) * T * w)[:, None] * q)
        if hard:
            hw = hard * w * labelled
            diff += hw[:, None] * torch.exp(logp1)
            diff.scatter_add_(1, label, -hw[:, None])
        answer["diff"] = diff
    return answer


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    s = {k: v.double() if v.dtype == torch.float32 else v for k, v in s.items()}
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    if case["op"] in ("adapt", "adapt-backward"):
        ids, begin, scale, rank = s["ids"].long(), s["begin"].long(), s["scale"], case["rank"]
        back = case["op"] == "adapt-backward"
        x, side_in, side_out = (s["e"], s["up"], s["down"]) if back else (s["in"], s["down"], s["up"])
        narrow = torch.zeros((case["rows"], rank), dtype=torch.float64, device="cuda")
        wide = x @ (s["W"] if back else s["W"].t())
        g_out, g_in = torch.zeros_like(side_out), torch.zeros_like(side_in)
        for g in ids.unique().tolist():
            if g < 0:
                continue
            member = (ids == g).double()[:, None]
            a, b = int(begin[g]), int(begin[g + 1])
            part = member * (x @ side_in[a:b].t()) * scale[g]
            narrow[:, :b - a] += part
            wide += part @ side_out[a:b]
            if back:
                g_out[a:b] = (part.t() @ s["in"])
                g_in[a:b] = ((member * s["t"][:, :b - a]).t() @ x)
        if back:
            answer = {"u": narrow, "gdown": g_out, "gup": g_in}
            return {**answer, "eout": wide * s["in"] * (1.0 - s["in"])} if case["eout"] else answer
        wide = wide + s["bias"]
        answer = {"out": 1.0 / (1.0 + torch.exp(-wide)) if case["act"] else wide, "t": narrow}
        if case["mix"] == "shuffled":
            none = ids < 0
            place = torch.where(none, torch.full_like(ids, case["num"]), ids) * case["rows"] + torch.arange(case["rows"], device="cuda")
            answer["order"] = (place.sort().values % case["rows"]).to(torch.int32)
            answer["row_begin"] = (ids[None, :] < torch.arange(case["num"] + 1, device="cuda")[:, None]).logical_and(~none[None, :]) \
                .sum(1).to(torch.int32)
        return answer
    z, K = s["z"], case["K"]
    if case["op"] == "top":
        val, idx = torch.sort(z, dim=1, descending=True, stable=True)
        return {"idx": idx[:, :K].to(torch.int32), "val": val[:, :K], "lse": torch.logsumexp(z, 1)}
    T, hard, w = case["temperature"], case["hard"], s["weight"]
    R, C = z.shape
    kept = (s["idx"] >= 0).sum(1)
    q = torch.zeros_like(z)
    entropy = torch.zeros(R, dtype=torch.float64, device="cuda")
    for k in range(K):  # the kept entries stand first in a row
        mass = torch.where(k < kept, torch.exp((s["val"][:, k] - s["val"][:, 0]) / T), zero)
        q[torch.arange(R, device="cuda"), s["idx"][:, k].clamp(min=0).long()] += mass
    q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
    entropy = torch.where(q > 0, q * torch.log(q.clamp(min=1e-300)), zero).sum(1)
    lp, lp1 = torch.log_softmax(z / T, 1), torch.log_softmax(z, 1)
    soft = T * T * (entropy - (q * lp).sum(1))
    has = (s["label"] >= 0).double()
    lab = s["label"].clamp(min=0).long()[:, None]
    row_loss = w * ((1 - hard) * soft - hard * has * lp1.gather(1, lab)[:, 0])
    answer = {"row_loss": row_loss}
    if case["diff"]:
        onehot = torch.zeros_like(z).scatter_(1, lab, 1.0)
        answer["diff"] = w[:, None] * ((1 - hard) * T * (q.sum(1, keepdim=True) * lp.exp() - q)
                                       + hard * has[:, None] * (lp1.exp() - onehot))
    return answer


def work(case):
    R = case["rows"]
    if case["op"] in ("adapt", "adapt-backward"):
        I, O, rank = case["I"], case["O"], case["rank"] * (0.5 if case["ragged"] else 1.0)
        used = min(case["num"], R)
        if case["op"] == "adapt":
            return {"bytes": 4.0 * (R * (I + O + rank + 1) + O * I + O + used * rank * (I + O)),
                    "flops": 2.0 * R * I * O + 2.0 * R * rank * (I + O)}
        return {"bytes": 4.0 * (R * (I + O + 2 * rank + 2 + (I if case["eout"] else 0)) + (O * I if case["eout"] else 0)
                                + used * rank * (I + O) + case["num"] * rank * (I + O)),
                "flops": (2.0 * R * I * O + 2.0 * R * rank * I if case["eout"] else 0.0) + 2.0 * R * rank * (I + 2 * O)}
    C, K = case["C"], case["K"]
    if case["op"] == "top":
        return {"bytes": 4.0 * R * (C + 2 * K + 1), "flops": 4.0 * R * C}
    return {"bytes": 4.0 * R * (C * (2 if case["diff"] else 1) + 2 * K + 3) + 8.0, "flops": 8.0 * R * C}
