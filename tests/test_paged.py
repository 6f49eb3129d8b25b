"""The paged operators against their definitions: block tables and slot maps,
page release, the append into slots and the attention behind a shared prompt.

Table outputs are whole numbers and must be equal.  The attention's tolerance
is derived per element from the 64-bit result: with h = finfo(dtype).eps / 2,
A = sum p |v| / sum p and |s| the largest sum of |q k| products of a row,
  * the output is rounded once: h |o|;
  * every probability is rounded once on its way to the matrix product: each
    moves the numerator by at most h p |v|, and the normaliser, summed from
    rounded or unrounded probabilities, by at most h of itself: 2 h A (fp32
    products take them unrounded);
  * a logit is a dot product of D terms in fp32 and its scale: it is off by at
    most (D + 4) 2^-24 |s|, the exponential by 2^-22 of itself, and sums of n
    terms by n 2^-24: numerator and normaliser, so twice that times A.
"""

import math

import pytest
import torch

from hotcold_kv import _native as N
from hotcold_kv import ops

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# The definitions
# ---------------------------------------------------------------------------
def ref_extend(lens, new, tables, free, count, P, n):
    lens, new, tables = list(lens), list(new), [list(t) for t in tables]
    B, T = len(lens), len(tables[0])
    cu, out, need_sum, used, taken = [0], list(lens), 0, 0, []
    slots, pos = [-1] * n, [-1] * n
    total = 0
    for b in range(B):
        total += max(new[b], 0)
        cu.append(min(total, n))
        have, want = -(-lens[b] // P), -(-(lens[b] + new[b]) // P)
        if lens[b] < 0 or new[b] < 0 or want > T or total > n:
            continue
        need = want - have
        first = need_sum
        need_sum += need
        if need and need_sum > count:
            continue
        used = max(used, need_sum) if need else used
        for k in range(need):
            tables[b][have + k] = free[count - 1 - first - k]
        out[b] = lens[b] + new[b]
        for i in range(new[b]):
            r = lens[b] + i
            pos[cu[b] + i] = r
            slots[cu[b] + i] = tables[b][r // P] * P + r % P if tables[b][r // P] >= 0 else -1
    return out, count - used, cu, slots, pos, tables


def ref_release(lens, keep, tables, free, count, P):
    out, free = list(lens), list(free)
    T = len(tables[0])
    for b, n in enumerate(lens):
        if n < 0 or -(-n // P) > T:
            continue
        k = min(n, max(keep[b], 0))
        for i in range(-(-k // P), -(-n // P)):
            if count < len(free):
                free[count] = tables[b][i]
                count += 1
        out[b] = k
    return out, count, free


def ref_attention(q, kp, vp, k_pages, v_pages, tables, lens, scaling, cu=None, prefix_lens=None):
    """(out, lse, bound of |o| weights A, largest |s|) in fp64 on the CPU; rows no request owns are NaN."""
    q, k_pages, v_pages = (x.detach().cpu().double() for x in (q, k_pages, v_pages))
    n, Hq, D = q.shape
    pages, Hk, P, _ = k_pages.shape
    G = Hq // Hk
    lens = lens.tolist()
    starts = cu.tolist() if cu is not None else list(range(len(lens) + 1))
    out = torch.full((n, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((n, Hq), math.nan, dtype=torch.float64)
    A = torch.zeros((n, Hq, D), dtype=torch.float64)
    top = torch.zeros((n, Hq), dtype=torch.float64)
    count = torch.zeros((n, 1, 1), dtype=torch.float64)
    for b, total in enumerate(lens):
        S = 0 if kp is None else kp.shape[-2]
        if prefix_lens is not None:
            S = min(max(int(prefix_lens[b]), 0), S)
        c0, c1 = starts[b], starts[b + 1]
        for i in range(c0, c1):
            own = max(0, total - (c1 - 1 - i))
            rows = [(int(tables[b, r // P]), r % P) for r in range(own)]
            rows = [(p, r) for p, r in rows if 0 <= p < pages]
            pg, rw = torch.tensor([p for p, _ in rows], dtype=torch.long), torch.tensor([r for _, r in rows], dtype=torch.long)
            k, v = k_pages[pg, :, rw].transpose(0, 1), v_pages[pg, :, rw].transpose(0, 1)
            if S:
                k = torch.cat([kp.detach().cpu().double().reshape(Hk, -1, D)[:, :S], k], 1)
                v = torch.cat([vp.detach().cpu().double().reshape(Hk, -1, D)[:, :S], v], 1)
            count[i] = k.shape[1]
            if k.shape[1] == 0:
                out[i], lse[i] = 0, -math.inf
                continue
            x = q[i].view(Hk, G, D) @ k.transpose(1, 2) * scaling
            p = torch.softmax(x, -1)
            out[i] = (p @ v).reshape(Hq, D)
            lse[i] = torch.logsumexp(x, -1).reshape(Hq)
            A[i] = (p @ v.abs()).reshape(Hq, D)
            top[i] = (q[i].view(Hk, G, D).abs() @ k.abs().transpose(1, 2) * abs(scaling)).amax(-1).reshape(Hq)
    return out, lse, A, top, count


def check_attention(got, want, dtype, lse=None):
    out, lw, A, top, count = want
    D = out.shape[-1]
    h = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    logit = (D + 4) * 2.0 ** -24 * top
    tol = (h or 2.0 ** -24) * out.abs() + 2 * h * A + 2 * A * (logit[..., None] + 2.0 ** -22 + count * 2.0 ** -24)
    tol = tol + torch.finfo(dtype).tiny
    mine = ~torch.isnan(out[:, :1, :1]).expand_as(out)
    err = (got.detach().cpu().double() - out).abs()
    bad = mine & ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {int(mine.sum())} off, worst {float((err / tol)[mine].max()):.3g} times the bound"
    if lse is not None:
        e = (lse.detach().cpu().double() - lw).abs()
        both = lse.detach().cpu().double() == lw
        # the sum's own error, and of the fp32 result of magnitude |lse|
        t = logit + 2.0 ** -22 + count[:, 0] * 2.0 ** -24 + 2 * h + 2.0 ** -22 * lw.abs().nan_to_num(posinf=0, neginf=0)
        bad = mine[..., 0] & ~both & ~(e <= t)
        assert not bad.any(), f"lse off by up to {float(e[mine[..., 0] & ~both].max()):.3g}"


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def paged_case(dtype, lens, new=None, prefix=64, Hq=8, Hk=2, D=64, P=16, seed=0, kscale=1.0, spare=3, stale=math.nan):
    """CPU tensors of one attention call; rows nobody holds are `stale`."""
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    new = new if new is not None else [1] * len(lens)
    have = [-(-max(n, 0) // P) for n in lens]
    width = max(1, max(have))
    pages = sum(have) + spare
    perm = torch.randperm(pages, generator=g).int()
    tables = torch.zeros((len(lens), width), dtype=torch.int32)
    k_pages = torch.randn((pages, Hk, P, D), generator=g).mul(kscale).to(dt)
    v_pages = torch.randn((pages, Hk, P, D), generator=g).to(dt)
    used = torch.zeros((pages, P), dtype=torch.bool)
    o = 0
    for b, n in enumerate(have):
        tables[b, :n] = perm[o:o + n]
        o += n
        for r in range(max(lens[b], 0)):
            used[tables[b, r // P], r % P] = True
    for t in (k_pages, v_pages):
        t.transpose(1, 2)[~used] = stale
    return dict(q=torch.randn((sum(new), Hq, D), generator=g).to(dt),
                kp=torch.randn((1, Hk, prefix, D), generator=g).mul(kscale).to(dt) if prefix is not None else None,
                vp=torch.randn((1, Hk, prefix, D), generator=g).to(dt) if prefix is not None else None,
                k_pages=k_pages, v_pages=v_pages, tables=tables, lens=torch.tensor(lens, dtype=torch.int32),
                cu=torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32) if max(new) != 1 or min(new) != 1 else None,
                max_new=max(new), scaling=1.0 / math.sqrt(D))


def to_dev(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def attend(c, prefix_lens=None, out=None, return_lse=False):
    return ops.prefix_attention(c["q"], c["kp"], c["vp"], c["k_pages"], c["v_pages"], c["tables"], c["lens"], c["scaling"],
                                cu_new=c["cu"], max_new=c["max_new"], prefix_lens=prefix_lens, out=out,
                                return_lse=return_lse)


def want_attention(c, prefix_lens=None):
    return ref_attention(c["q"], c["kp"], c["vp"], c["k_pages"], c["v_pages"], c["tables"], c["lens"], c["scaling"], c["cu"],
                         prefix_lens)


# ---------------------------------------------------------------------------
# Refusals (no GPU: the checks come before the devices', the library's before any launch)
# ---------------------------------------------------------------------------
def test_paged_operators_refuse_host_tensors():
    c = paged_case("f32", [5, 9], stale=0.0)
    with pytest.raises(RuntimeError, match="ROCm device tensors only"):
        attend(c)
    i = torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device tensors only"):
        ops.extend_pages(i, i, c["tables"], i, i[:1], 16, 2)
    with pytest.raises(RuntimeError, match="ROCm device tensors only"):
        ops.release_pages(i, i, c["tables"], i, i[:1], 16)
    with pytest.raises(RuntimeError, match="ROCm device tensors only"):
        ops.append_paged(torch.zeros(2, dtype=torch.int64), c["k_pages"][:2, :, 0], c["v_pages"][:2, :, 0], c["k_pages"],
                         c["v_pages"])


@pytest.mark.parametrize("change,message", [
    (dict(lens=torch.ones(2)), "lens must be a contiguous int32 vector"),
    (dict(lens=torch.ones(4, dtype=torch.int32)[::2]), "lens must be a contiguous int32 vector"),
    (dict(tables=torch.zeros((3, 2), dtype=torch.int32)), "tables must be"),
    (dict(tables=torch.zeros((2, 2), dtype=torch.int64)), "tables must be"),
    (dict(k_pages=torch.zeros((4, 2, 16, 32))), "k_pages, v_pages must be"),
    (dict(kp=torch.zeros((2, 2, 8, 64))), "k_prefix, v_prefix must be"),
    (dict(vp=None), "go together"),
    (dict(q=torch.zeros((3, 8, 64))), "one token"),
    (dict(cu=torch.zeros(2, dtype=torch.int32)), "cu_new must be"),
    (dict(cu=torch.zeros(3, dtype=torch.int32), max_new=None), "needs max_new"),
    (dict(prefix_lens=torch.ones(3, dtype=torch.int32)), "prefix_lens must be"),
    (dict(out=torch.zeros((2, 8, 64), dtype=torch.float16)), "out must be"),
    (dict(q=torch.zeros((2, 8, 64), dtype=torch.float64)), "unsupported dtype"),
])
def test_prefix_attention_refuses(change, message):
    c = paged_case("f32", [5, 9], stale=0.0)
    extra = {k: change.pop(k) for k in ("prefix_lens", "out") if k in change}
    c.update(change)
    with pytest.raises((RuntimeError, TypeError), match=message):
        attend(c, **extra)


def test_table_operators_refuse():
    i = torch.ones(2, dtype=torch.int32)
    t = torch.zeros((2, 4), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="new_lens"):
        ops.extend_pages(i, i[:1], t, i, i[:1], 16, 2)
    with pytest.raises(RuntimeError, match="lens_out"):
        ops.extend_pages(i, i, t, i, i[:1], 16, 2, lens_out=torch.ones(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="free_count"):
        ops.release_pages(i, i, t, i, i, 16)
    with pytest.raises(RuntimeError, match="keep_lens"):
        ops.release_pages(i, i.long(), t, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="slots"):
        ops.append_paged(torch.zeros(3, dtype=torch.int64), torch.zeros((2, 2, 8)), torch.zeros((2, 2, 8)),
                         torch.zeros((4, 2, 4, 8)), torch.zeros((4, 2, 4, 8)))
    with pytest.raises(RuntimeError, match="must match"):
        ops.append_paged(torch.zeros(2, dtype=torch.int64), torch.zeros((2, 2, 8)), torch.zeros((2, 2, 16)),
                         torch.zeros((4, 2, 4, 8)), torch.zeros((4, 2, 4, 8)))


def _attn_args(**change):
    """Arguments of a valid call over addresses that are never read."""
    a = N.PrefixAttnArgs(dtype=N.HC_DTYPE_F16, N=2, B=2, Hq=8, Hk=2, D=64, q=4096, q_sn=512, q_sh=64, k_prefix=4096,
                         kp_sh=4096, kp_ss=64, v_prefix=4096, vp_sh=4096, vp_ss=64, prefix_rows=64, k_pages=4096,
                         kg_sp=2048, kg_sh=1024, kg_ss=64, v_pages=4096, vg_sp=2048, vg_sh=1024, vg_ss=64, num_pages=4,
                         page_size=16, tables=4096, t_sb=2, table_width=2, lens=4096, max_new=1, scaling=0.125, out=4096,
                         o_sn=512, o_sh=64)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), N.HC_ERR_INVALID), (dict(Hq=9), N.HC_ERR_GROUP), (dict(D=48), N.HC_ERR_UNSUPPORTED),
    (dict(D=256), N.HC_ERR_UNSUPPORTED), (dict(page_size=24), N.HC_ERR_INVALID), (dict(page_size=0), N.HC_ERR_INVALID),
    (dict(num_pages=0), N.HC_ERR_INVALID), (dict(table_width=0), N.HC_ERR_INVALID), (dict(t_sb=1), N.HC_ERR_INVALID),
    (dict(N=3), N.HC_ERR_INVALID), (dict(max_new=2), N.HC_ERR_INVALID), (dict(max_new=0, cu_new=4096), N.HC_ERR_INVALID),
    (dict(q=None), N.HC_ERR_INVALID), (dict(q=4104), N.HC_ERR_INVALID), (dict(kg_ss=68), N.HC_ERR_INVALID),
    (dict(k_prefix=None), N.HC_ERR_INVALID), (dict(prefix_rows=-1), N.HC_ERR_INVALID), (dict(B=0), N.HC_ERR_INVALID),
])
def test_library_refuses_attention_arguments(change, code):
    import ctypes
    a = _attn_args(**change)
    assert N.lib().hc_prefix_attn(ctypes.addressof(a), None) == code
    assert b"prefix_attention" in N.lib().hc_last_error()
    assert N.lib().hc_prefix_attn_workspace_size(ctypes.addressof(a)) < 0


def test_library_refuses_table_arguments():
    lib = N.lib()
    p = 4096
    extend = [2, p, p, p, 4, 4, p, 8, p, 16, 4, p, p, p, p, p, None]
    release = [2, p, p, p, 4, 4, p, 8, p, 16, p, p, None]
    for at, value in ((0, 0), (0, 4097), (1, None), (4, 3), (5, 0), (5, 1 << 28), (7, 0), (9, 3), (10, -1), (10, (1 << 20) + 1)):
        assert lib.hc_extend_pages(*[value if i == at else x for i, x in enumerate(extend)]) == N.HC_ERR_INVALID, (at, value)
    for at, value in ((0, 0), (0, 4097), (1, None), (4, 3), (5, 0), (7, 0), (9, 3), (9, 1 << 17)):
        assert lib.hc_release_pages(*[value if i == at else x for i, x in enumerate(release)]) == N.HC_ERR_INVALID, (at, value)
    append = [N.HC_DTYPE_F16, 2, 2, 64, p, p, 128, 64, p, 128, 64, p, 2048, 1024, 64, p, 2048, 1024, 64, 4, 16, None]
    for at, value in ((0, 9), (1, -1), (2, 0), (3, 12), (4, None), (5, p + 8), (6, 3), (14, 4), (19, 0), (20, 12)):
        assert lib.hc_append_paged(*[value if i == at else x for i, x in enumerate(append)]) == N.HC_ERR_INVALID, (at, value)


# ---------------------------------------------------------------------------
# Tables
# ---------------------------------------------------------------------------
def _tables(g, lens, T, P, spare):
    have = [min(T, -(-max(n, 0) // P)) for n in lens]
    perm = torch.randperm(sum(have) + spare, generator=g).tolist()
    t = [[1000000 + b * T + j for j in range(T)] for b in range(len(lens))]      # entries nobody holds
    o = 0
    for b, n in enumerate(have):
        t[b][:n] = perm[o:o + n]
        o += n
    return t, perm[o:] + [0] * o, spare


EXTENDS = [
    # lens, new, table width, page size, free pages, rows of the token batch
    ([0], [1], 1, 16, 1, 1),
    ([0], [0], 1, 16, 0, 0),
    ([15, 16, 17, 0], [1, 1, 1, 1], 4, 16, 4, 4),
    ([15, 16, 17, 0], [1, 1, 1, 1], 4, 16, 1, 6),           # the second page is missing
    ([3, 5, 9, 60, 2], [40, 0, 7, 4, 70], 8, 8, 9, 130),     # an exact fit, and one that does not
    ([0, 0, 0], [33, 64, 1], 2, 32, 2, 98),                  # the second takes none, the third is behind it
    ([-1, 4, 4, 4], [1, -1, 1, 200], 4, 16, 9, 50),          # bad lengths, a table too short
    ([4, 4, 4], [8, 8, 8], 4, 4, 20, 17),                    # tokens past the batch
    ([7, 8, 9], [1, 1, 1], 12, 1, 3, 3),                     # pages of one row
    ([2 ** 31 - 1, 5], [2 ** 31 - 1, 1], 4, 16, 3, 3),       # sums past 32 bits
]


def _rand_extend(seed, B, P, most_len, most_new, spare_share, pad):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, most_len + 1, (B,), generator=g).tolist()
    new = torch.randint(0, most_new + 1, (B,), generator=g).tolist()
    need = sum(-(-(a + b) // P) - -(-a // P) for a, b in zip(lens, new))
    return lens, new, -(-(most_len + most_new) // P), P, int(need * spare_share), sum(new) + pad


RANDOM = [_rand_extend(1, 64, 16, 100, 3, 1.0, 5), _rand_extend(2, 257, 16, 500, 1, 0.5, 0),
          _rand_extend(3, 300, 8, 90, 40, 0.9, 77), _rand_extend(4, 1000, 32, 64, 9, 1.0, 1),
          _rand_extend(5, 4096, 16, 40, 2, 0.99, 0), _rand_extend(6, 3, 64, 5000, 3000, 1.0, 11)]


def run_extend(lens, new, T, P, spare, n, inplace=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    tables, free, count = _tables(g, lens, T, P, spare)
    free = free or [0]
    want = ref_extend(lens, new, tables, free, count, P, n)
    i32 = dict(dtype=torch.int32, device="cuda")
    dl, dn, dt, df, dc = (torch.tensor(x, **i32) for x in (lens, new, tables, free, [count]))
    if inplace:
        got = ops.extend_pages(dl, dn, dt, df, dc, P, n, lens_out=dl, count_out=dc)
        assert got[0] is dl or got[0].data_ptr() == dl.data_ptr()
    else:
        got = ops.extend_pages(dl, dn, dt, df, dc, P, n)
        assert dl.tolist() == list(lens) and dc.tolist() == [count]
    out, c, cu, slots, pos, t = want
    assert got[0].tolist() == out and got[1].tolist() == [c] and got[2].tolist() == cu
    assert got[4].tolist() == pos and got[3].tolist() == slots and dt.tolist() == t
    assert df.tolist() == list(free)


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", EXTENDS + RANDOM, ids=lambda c: f"B{len(c[0])}_P{c[3]}_N{c[5]}_free{c[4]}")
def test_extend_pages_equals_the_definition(case, inplace):
    run_extend(*case, inplace=inplace)


@pytest.mark.gpu
def test_extend_pages_clamps_the_free_count():
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, new, free = torch.zeros(2, **i32), torch.ones(2, **i32), torch.tensor([5, 6, 7], **i32)
    for count, left, want in ((-4, 0, [0, 0]), (9, 1, [1, 1])):
        t = torch.full((2, 2), -1, **i32)
        lo, co, cu, slots, pos = ops.extend_pages(lens, new, t, free, torch.tensor([count], **i32), 8, 2)
        assert lo.tolist() == want and co.tolist() == [left] and cu.tolist() == [0, 1, 2]
        assert slots.tolist() == ([-1, -1] if count < 0 else [7 * 8, 6 * 8])


@pytest.mark.gpu
def test_extend_pages_gives_no_slot_in_a_page_below_zero():
    i32 = dict(dtype=torch.int32, device="cuda")
    t = torch.tensor([[-3, 0]], **i32)
    lo, _, _, slots, pos = ops.extend_pages(torch.tensor([2], **i32), torch.tensor([3], **i32), t, torch.tensor([9], **i32),
                                            torch.tensor([1], **i32), 4, 3)
    assert lo.tolist() == [5] and slots.tolist() == [-1, -1, 36] and pos.tolist() == [2, 3, 4] and t.tolist() == [[-3, 9]]


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens,keep,T,P,cap", [
    ([40], [0], 3, 16, None), ([40], [33], 3, 16, None), ([40], [32], 3, 16, None), ([0, 5], [0, 9], 2, 8, None),
    ([33, 64, 1, 17], [0, 64, -5, 16], 4, 16, None), ([-2, 99, 7], [0, 0, 0], 4, 16, None), ([64, 64], [0, 0], 8, 8, 10),
    (list(range(0, 300)), [i % 7 * 20 for i in range(300)], 40, 8, None), ([2000] * 40, [0] * 40, 125, 16, None),
    ([3] * 4096, [0, 3] * 2048, 1, 4, None),
])
def test_release_pages_equals_the_definition(lens, keep, T, P, cap, inplace):
    g = torch.Generator().manual_seed(len(lens))
    tables, free, count = _tables(g, lens, T, P, 3)
    free = (free + [0] * 8)[:cap]
    want = ref_release(lens, keep, tables, free, count, P)
    i32 = dict(dtype=torch.int32, device="cuda")
    dl, dk, dt, df, dc = (torch.tensor(x, **i32) for x in (lens, keep, tables, free, [count]))
    kw = dict(lens_out=dl, count_out=dc) if inplace else {}
    lo, co = ops.release_pages(dl, dk, dt, df, dc, P, **kw)
    assert lo.tolist() == want[0] and co.tolist() == [want[1]] and df.tolist() == want[2] and dt.tolist() == tables


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,Hk,D,P", [("f16", 1, 1, 16, 16), ("bf16", 7, 3, 32, 8), ("f32", 33, 2, 64, 1),
                                            ("f16", 300, 8, 128, 32), ("bf16", 65, 5, 128, 64), ("f32", 9, 1, 4, 16)])
@pytest.mark.parametrize("layout", ["plain", "strided"])
def test_append_paged_writes_its_slots_only(dtype, n, Hk, D, P, layout):
    g = torch.Generator().manual_seed(n)
    dt = DTYPES[dtype]
    pages = -(-n // P) + 3
    new = torch.randn((n, 2 * Hk, D), generator=g).to(dt).cuda()
    k, v = new[:, :Hk], new[:, Hk:]
    if layout == "strided":                       # keys beside values, and a head-first token batch
        kv = torch.zeros((pages, P, Hk, 2, D), dtype=dt, device="cuda")
        kp, vp = kv[..., 0, :].transpose(1, 2), kv[..., 1, :].transpose(1, 2)
        k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    else:
        kp, vp = (torch.zeros((pages, Hk, P, D), dtype=dt, device="cuda") for _ in range(2))
    slots = torch.randperm(pages * P, generator=g)[:n].cuda()
    slots[::5] = torch.tensor([-1, pages * P, -2 ** 40, 2 ** 40]).repeat(n)[:len(slots[::5])].cuda()
    want_k, want_v = kp.clone(), vp.clone()
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages * P:
            want_k[s // P, :, s % P], want_v[s // P, :, s % P] = k[i], v[i]
    ops.append_paged(slots, k, v, kp, vp)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    ops.append_paged(slots[:0], k[:0], v[:0], kp, vp)
    assert torch.equal(kp, want_k)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
CASES = [
    # one token a request
    dict(lens=[1]), dict(lens=[1], prefix=None), dict(lens=[1], prefix=0), dict(lens=[5, 17, 64, 1], prefix=1),
    dict(lens=[31, 32, 33, 16], prefix=33), dict(lens=[300, 2, 129], prefix=257, P=8), dict(lens=[40, 7], prefix=1000, Hq=2, Hk=2),
    dict(lens=[65, 1, 250, 33, 90], prefix=95, Hq=12, Hk=4, D=32), dict(lens=[9, 70], prefix=130, Hq=3, Hk=1, D=16),
    dict(lens=[513, 77, 300], prefix=700, Hq=16, Hk=2, D=128, P=32), dict(lens=[50] * 9, prefix=64, Hq=16, Hk=1, D=128, P=1),
    dict(lens=[20 + i for i in range(17)], prefix=321, Hq=8, Hk=2, D=128), dict(lens=[3] * 40, prefix=129, Hq=20, Hk=4, D=64),
    dict(lens=[100 + i for i in range(70)], prefix=600, Hq=4, Hk=1, D=64, P=64),
    # several, among them none
    dict(lens=[5, 40], new=[2, 3], prefix=50), dict(lens=[70, 3, 9, 33], new=[64, 0, 1, 33], prefix=77),
    dict(lens=[200, 10, 300], new=[130, 10, 7], prefix=100, Hq=4, Hk=2, D=128, P=32), dict(lens=[90, 1], new=[90, 1], prefix=None, Hq=6, Hk=2, D=32),
    dict(lens=[257, 31, 600], new=[257, 31, 1], prefix=65, Hq=8, Hk=1, D=16, P=8), dict(lens=[4], new=[4], prefix=0, Hq=1, Hk=1, D=128),
    dict(lens=[150, 90], new=[100, 90], prefix=515, Hq=10, Hk=2, D=64), dict(lens=[2, 0, 1], new=[5, 1, 1], prefix=40),   # more tokens than rows
]


def _id(c):
    return "_".join(f"{k}{v if not isinstance(v, list) else 'x'.join(map(str, v[:3]))}" for k, v in c.items())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_prefix_attention_equals_the_definition(dtype, case):
    c = paged_case(dtype, **case)
    want = want_attention(c)
    out, lse = attend(to_dev(c), return_lse=True)
    check_attention(out, want, DTYPES[dtype], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_requests_share_a_part_of_the_prompt(dtype):
    lens, new = [30, 4, 0, 61, 9, 12], [5, 1, 2, 40, 3, 1]
    shared = torch.tensor([0, 150, 0, 37, -3, 10 ** 6], dtype=torch.int32)
    c = paged_case(dtype, lens, new, prefix=150, Hq=8, Hk=2, D=128)
    want = want_attention(c, shared)
    assert (want[4] == 0).sum() == 2                        # two tokens attend nothing
    out, lse = attend(to_dev(c), shared.cuda(), return_lse=True)
    check_attention(out, want, DTYPES[dtype], lse)
    assert (out[6:8] == 0).all() and (lse[6:8] == -math.inf).all()
    one = paged_case(dtype, [30, 4, 0, 61, 9, 12], prefix=150, Hq=8, Hk=2, D=128)
    out, lse = attend(to_dev(one), shared.cuda(), return_lse=True)
    check_attention(out, want_attention(one, shared), DTYPES[dtype], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_rows_that_are_not_attended_may_hold_anything(dtype, value):
    """Stale rows of pages, the prompt past prefix_lens, and later tokens of the same request."""
    c = paged_case(dtype, [40, 77], [20, 60], prefix=90, Hq=4, Hk=2, D=64, stale=value)
    shared = torch.tensor([70, 33], dtype=torch.int32)
    c["kp"][:, :, 70:], c["vp"][:, :, 70:] = value, value
    want = want_attention(c, shared)
    out, lse = attend(to_dev(c), shared.cuda(), return_lse=True)
    check_attention(out, want, DTYPES[dtype], lse)
    # the last token's own row: every earlier token's sum has the same terms, added in another order in the tile that
    # holds the row (n terms in any order: n 2^-24 of A, in the bound already)
    page, row = int(c["tables"][1, 76 // 16]), 76 % 16
    c["k_pages"][page, :, row], c["v_pages"][page, :, row] = value, value
    again, lse2 = attend(to_dev(c), shared.cuda(), return_lse=True)
    check_attention(again[:79], [x[:79] for x in want], DTYPES[dtype], lse2[:79])
    # the prompt's rows between the two requests' shares
    c = paged_case(dtype, [40, 77], prefix=90, Hq=4, Hk=2, D=64)
    out = attend(to_dev(c), shared.cuda())
    c["kp"][:, :, 33:], c["vp"][:, :, 33:] = value, value
    assert torch.equal(attend(to_dev(c), shared.cuda())[1], out[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_values_that_are_attended_reach_the_output(dtype):
    """An infinity or NaN in an attended row shows where the definition has it."""
    c = paged_case(dtype, [40, 77], [20, 60], prefix=90, Hq=4, Hk=2, D=64)
    page, row = int(c["tables"][1, 30 // 16]), 30 % 16            # seen by request 1's tokens from row 30 on
    c["v_pages"][page, 0, row, 5], c["v_pages"][page, 1, row, 9] = math.inf, math.nan
    out = attend(to_dev(c)).cpu()
    want = want_attention(c)[0]
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    assert torch.isinf(out).sum() == 47 * 2 and torch.isnan(out).sum() == 47 * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_large_logits(dtype):
    c = paged_case(dtype, [40, 77, 300], [3, 60, 1], prefix=290, Hq=4, Hk=2, D=64, kscale=30.0)
    out, lse = attend(to_dev(c), return_lse=True)
    check_attention(out, want_attention(c), DTYPES[dtype], lse)
    for scaling in (0.0, -0.05):                                   # a plain mean; the least similar keys
        c["scaling"] = scaling
        check_attention(attend(to_dev(c)), want_attention(c), DTYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_pages_outside_the_pool_hide_their_rows(dtype):
    c = paged_case(dtype, [100, 77, 60], [1, 40, 1], prefix=20, Hq=4, Hk=2, D=64)
    pages = c["k_pages"].shape[0]
    c["tables"][0, 2], c["tables"][1, 0], c["tables"][2, :4] = -1, pages, torch.tensor([2 ** 31 - 1, -2 ** 31, pages + 5, -7])
    out, lse = attend(to_dev(c), return_lse=True)
    check_attention(out, want_attention(c), DTYPES[dtype], lse)


@pytest.mark.gpu
def test_lengths_past_the_table_are_cut():
    c = paged_case("f16", [64, 48], prefix=20, P=16)
    want = want_attention(c)
    c["lens"] = torch.tensor([10 ** 9, 48], dtype=torch.int32)
    out = attend(to_dev(c))
    check_attention(out, want, torch.float16)
    c["lens"] = torch.tensor([-5, 48], dtype=torch.int32)
    check_attention(attend(to_dev(c)), want_attention(c), torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_behind_the_last_request_stay(dtype):
    host = paged_case(dtype, [40, 20], [7, 3], prefix=33)
    c = to_dev(host)
    q = torch.full((25, 8, 64), math.nan, dtype=DTYPES[dtype], device="cuda")
    q[:10] = c["q"]
    out = torch.full((25, 2, 8, 64), 7.0, dtype=DTYPES[dtype], device="cuda")[:, 1]
    c["q"] = q
    got = attend(c, out=out)
    # (a larger token batch may be split otherwise: the same sums in another order, within the bound)
    check_attention(out[:10], want_attention(host), DTYPES[dtype])
    assert got.data_ptr() == out.data_ptr() and (out[10:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts(dtype):
    """Views: q of a fused projection, a hot buffer's prompt, pools with keys beside values or token-major rows."""
    c = to_dev(paged_case(dtype, [70, 33, 5], [40, 1, 5], prefix=100, Hq=8, Hk=2, D=64))
    want = attend(c)
    n = c["q"].shape[0]
    c["q"] = torch.cat([c["q"], torch.zeros((n, 4, 64), device="cuda").to(c["q"].dtype)], 1)[:, :8]
    c["kp"], c["vp"] = torch.stack([c["kp"], c["vp"]], 3).unbind(3)
    pools = torch.stack([c["k_pages"], c["v_pages"]], 3)
    c["k_pages"], c["v_pages"] = pools.unbind(3)
    assert torch.equal(attend(c), want)
    c["k_pages"], c["v_pages"] = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c["k_pages"], c["v_pages"]))
    c["q"], c["kp"], c["vp"] = c["q"][:, :, None], c["kp"][0], c["vp"][0]
    assert torch.equal(attend(c), want)
    c["q"] = c["q"][:, :, 0].transpose(1, 2).contiguous().transpose(1, 2)      # a strided head dimension is copied
    assert torch.equal(attend(c), want)


@pytest.mark.gpu
def test_long_pool_offsets_pass_32_bits():
    """Pages past 4 GiB (and 2^31 elements) of the pool, and a prompt whose heads lie that far apart."""
    P, D = 16, 128
    pages = (1 << 32) // (P * D * 2) + 4096
    pool = torch.zeros((2, pages, 1, P, D), dtype=torch.float16, device="cuda")
    c = paged_case("f16", [100, 45], [3, 1], prefix=70, Hq=4, Hk=1, D=D, P=P, stale=0.0)
    want = want_attention(c)
    d = to_dev(c)
    used = c["k_pages"].shape[0]
    pool[0, pages - used:], pool[1, pages - used:] = d["k_pages"], d["v_pages"]
    d["k_pages"], d["v_pages"], d["tables"] = pool[0], pool[1], d["tables"] + (pages - used)
    check_attention(attend(d), want, torch.float16)
    slots = torch.tensor([pages * P - 1], device="cuda")
    row = torch.ones((1, 1, D), dtype=torch.float16, device="cuda")
    ops.append_paged(slots, row, 2 * row, pool[0], pool[1])
    assert (pool[0, -1, 0, -1] == 1).all() and (pool[1, -1, 0, -1] == 2).all()
    two = paged_case("f16", [9], prefix=70, Hq=4, Hk=2, D=D, P=P)
    far = pool.view(-1)[:(1 << 32) + 70 * D].as_strided((1, 2, 70, D), (0, 1 << 32, D, 1))
    far.copy_(two["kp"])
    t = to_dev(two)
    t["kp"] = far
    check_attention(attend(t), want_attention(two), torch.float16)


@pytest.mark.gpu
def test_two_streams_at_once():
    cs = [to_dev(paged_case("bf16", [300 + 40 * s, 77], [90, 1], prefix=900, Hq=8, Hk=2, D=128, seed=s)) for s in range(2)]
    want = [attend(c) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(3):
        got = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                got.append([attend(c) for _ in range(4)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, w) for x in g)


@pytest.mark.gpu
def test_same_call_gives_the_same_bits():
    c = to_dev(paged_case("f16", [700, 64, 333], prefix=3000, Hq=16, Hk=2, D=128))
    want = attend(c)
    assert all(torch.equal(attend(c), want) for _ in range(5))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", ["one", "several"])
def test_a_captured_step_replays_over_new_lengths(tokens):
    """Tables, append and attention of a serving step in a graph, replayed as the requests grow, against the eager
    calls; two graphs over the same pool, their replays interleaved with eager work."""
    P, Hq, Hk, D, B, most = 8, 8, 2, 64, 5, 6
    g = torch.Generator().manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = B if tokens == "one" else B * most

    def state():
        return dict(lens=torch.zeros(B, **i32), new=torch.zeros(B, **i32), tables=torch.zeros((B, 20), **i32),
                    free=torch.arange(100, **i32), count=torch.tensor([100], **i32),
                    k_pages=torch.zeros((100, Hk, P, D), dtype=torch.float16, device="cuda"),
                    v_pages=torch.zeros((100, Hk, P, D), dtype=torch.float16, device="cuda"),
                    q=torch.zeros((rows, Hq, D), dtype=torch.float16, device="cuda"),
                    kv=torch.zeros((rows, 2, Hk, D), dtype=torch.float16, device="cuda"),
                    out=torch.zeros((rows, Hq, D), dtype=torch.float16, device="cuda"))

    kp, vp = (torch.randn((1, Hk, 77, D), generator=g).half().cuda() for _ in range(2))

    def step(s):
        _, _, cu, slots, _ = ops.extend_pages(s["lens"], s["new"], s["tables"], s["free"], s["count"], P, rows,
                                              lens_out=s["lens"], count_out=s["count"])
        ops.append_paged(slots, s["kv"][:, 0], s["kv"][:, 1], s["k_pages"], s["v_pages"])
        ops.prefix_attention(s["q"], kp, vp, s["k_pages"], s["v_pages"], s["tables"], s["lens"], 0.125,
                             cu_new=None if tokens == "one" else cu, max_new=None if tokens == "one" else most,
                             out=s["out"])

    eager, sides = state(), [state(), state()]
    graphs = []
    for s in sides:
        step(s)                                                     # no tokens yet
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(s)
        graphs.append(graph)
    for it in range(8):
        new = torch.ones(B) if tokens == "one" else torch.randint(0, most + 1, (B,), generator=g)
        q, kv = torch.randn((rows, Hq, D), generator=g).half(), torch.randn((rows, 2, Hk, D), generator=g).half()
        for s in [eager] + sides:
            s["new"].copy_(new), s["q"].copy_(q), s["kv"].copy_(kv)
        step(eager)
        for graph in graphs:
            graph.replay()
        if it % 3 == 2:                                             # the eager side's program goes on between replays
            ops.release_pages(eager["lens"], eager["lens"], eager["tables"], eager["free"], eager["count"], P)
            torch.cuda.synchronize()
        for s in sides:
            for name in ("lens", "count", "tables", "out", "k_pages", "v_pages"):
                assert torch.equal(s[name], eager[name]), (it, name)


# ---------------------------------------------------------------------------
# The operators as a serving loop uses them
# ---------------------------------------------------------------------------
def test_argument_struct_has_the_headers_fields():
    import os
    import re
    path = os.path.join(os.path.dirname(__file__), "..", "include", "hotcold_hip.h")
    with open(path) as f:
        body = re.search(r"typedef struct hc_prefix_attn_args \{(.*?)\}", f.read(), re.S).group(1)
    want = []
    for decl in filter(None, (d.strip() for d in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"))):
        kind = "p" if "*" in decl else "d" if decl.startswith("double") else "i"
        names = re.sub(r"^(const )?(void|float|int32_t|int64_t|double)\s*\*?\s*", "", decl)
        want += [(n.strip(), kind) for n in names.split(",")]
    kinds = {N._vp: "p", N._dbl: "d", N._i64: "i"}
    assert [(n, kinds[t]) for n, t in N.PrefixAttnArgs._fields_] == want


def test_batch_refuses():
    from hotcold_kv import SharedPromptBatch
    from hotcold_kv.hot_buffer import HotBuffer
    with pytest.raises(ValueError, match="at least 1"):
        SharedPromptBatch(1, 0, 2, 64, torch.float16, "cpu", 8, 16, 64)
    b = SharedPromptBatch(1, 2, 2, 64, torch.float16, "cpu", 8, 16, 64)
    with pytest.raises(ValueError, match="batch 2"):
        b.set_prompt(0, HotBuffer(2, 2, 64, torch.float16, "cpu", 4))
    with pytest.raises(RuntimeError, match="before extend"):
        b.attend(0, None, None, None, 1.0)
    with pytest.raises(RuntimeError, match="device"):
        b.extend(torch.ones(2, dtype=torch.int32), 2, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,requests,Hq,Hk,D,P", [("f16", 5, 8, 2, 128, 16), ("bf16", 40, 6, 3, 64, 4), ("f32", 3, 4, 4, 16, 32)])
def test_a_batch_behind_a_compacted_prompt(dtype, requests, Hq, Hk, D, P):
    """Prompts, decode steps, rejected tokens, requests that end and others that take their rows, over two layers
    whose prompts were compacted to different rows: every token against the 64-bit attention over a dense copy of
    what its request holds."""
    from hotcold_kv import SharedPromptBatch
    from hotcold_kv.hot_buffer import HotBuffer
    g = torch.Generator().manual_seed(11)
    dt, layers, S, longest, most = DTYPES[dtype], 2, 200, 60, 20
    pages = requests * -(-longest // P)
    batch = SharedPromptBatch(layers, requests, Hk, D, dt, "cuda", pages, P, longest)
    prompts = []
    for layer in range(layers):
        buf = HotBuffer(1, Hk, D, dt, "cuda", S)
        k, v = (torch.randn((1, Hk, S, D), generator=g).to(dt) for _ in range(2))
        buf.append(k.cuda(), v.cuda())
        keep = torch.stack([torch.randperm(S, generator=g)[:90 + 40 * layer].sort().values for _ in range(Hk)])[None]
        buf.compact(keep.cuda())
        at = keep[..., None].expand(-1, -1, -1, D)
        prompts.append((k.gather(2, at), v.gather(2, at)))
        batch.set_prompt(layer, buf)
    held = [0] * requests
    dense = [[torch.zeros((requests, Hk, longest, D), dtype=dt) for _ in range(2)] for _ in range(layers)]
    own = torch.arange(requests, dtype=torch.int32)[:, None]            # the dense copy is a pool of one page a request
    for it in range(9):
        new = [int(x) for x in torch.randint(1, most + 1, (requests,), generator=g)] if it % 4 == 0 else [1] * requests
        new = [min(n, longest - h) for n, h in zip(new, held)]
        if it == 5:
            new[1] = 0                                                  # idle in this step
        n = sum(new) + it % 3
        pos = batch.extend(torch.tensor(new, dtype=torch.int32).cuda(), n, max(new))
        held = [h + x for h, x in zip(held, new)]
        assert batch.lens.tolist() == held
        rows = [(b, held[b] - new[b] + i) for b in range(requests) for i in range(new[b])]
        assert pos.tolist() == [r for _, r in rows] + [-1] * (n - len(rows))
        cu = torch.tensor([0] + new).cumsum(0).int()
        for layer in range(layers):
            q = torch.randn((n, Hq, D), generator=g).to(dt)
            k, v = (torch.randn((n, Hk, D), generator=g).to(dt) for _ in range(2))
            for i, (b, r) in enumerate(rows):
                dense[layer][0][b, :, r], dense[layer][1][b, :, r] = k[i], v[i]
            out = torch.full((n, Hq, D), 7.0, dtype=dt, device="cuda")
            batch.attend(layer, q.cuda(), k.cuda(), v.cuda(), D ** -0.5, out=out)
            want = ref_attention(q, *prompts[layer], *dense[layer], own, torch.tensor(held), D ** -0.5, cu)
            check_attention(out, want, dt)
            assert bool((out[len(rows):] == 7).all())
        if it % 2 == 1:                                                 # reject up to two tokens, end every fifth request
            keep = [0 if (b + it) % 5 == 0 else max(h - b % 3, 0) for b, h in enumerate(held)]
            batch.release(torch.tensor(keep, dtype=torch.int32).cuda())
            held = keep
            with pytest.raises(RuntimeError, match="before extend"):
                batch.attend(0, q, k, v, 1.0)
    batch.release(torch.zeros(requests, dtype=torch.int32).cuda())
    assert batch.lens.tolist() == [0] * requests and batch.free_count.tolist() == [pages]
    assert sorted(batch.free_pages.tolist()) == list(range(pages))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 2500])
@pytest.mark.parametrize("overlap", ["none", "lens", "count", "crossed"])
def test_outputs_may_be_any_of_the_inputs(tokens, overlap):
    """Lengths and count written over any input they replace, with one workgroup and with several."""
    B, P, F = 40, 16, 400
    lens, new = [3 * b % 50 for b in range(B)], [1 + (tokens // B if b % 2 else 0) for b in range(B)]
    keep = [max(0, n - b % 30) for b, n in enumerate(lens)]
    g = torch.Generator().manual_seed(tokens)
    T = -(-(max(lens) + max(new)) // P)
    tables, _, _ = _tables(g, lens, T, P, 0)
    free = list(range(1000, 1000 + F))
    i32 = dict(dtype=torch.int32, device="cuda")
    for op in ("extend", "release"):
        count = 300
        dl, dn, dk, dt, df, dc = (torch.tensor(x, **i32) for x in (lens, new, keep, tables, free, [count]))
        lo, co = torch.zeros(B, **i32), torch.zeros(1, **i32)
        more = dn if op == "extend" else dk
        if overlap == "lens":
            lo = dl
        elif overlap == "count":
            co = dc
        elif overlap == "crossed":
            lo, co = more, dc
        if op == "extend":
            n = sum(new)
            want = ref_extend(lens, new, tables, free, count, P, n)
            got = ops.extend_pages(dl, dn, dt, df, dc, P, n, lens_out=lo, count_out=co)
            assert got[3].tolist() == want[3] and got[4].tolist() == want[4] and dt.tolist() == want[5]
        else:
            want = ref_release(lens, keep, tables, free, count, P)
            ops.release_pages(dl, dk, dt, df, dc, P, lens_out=lo, count_out=co)
            assert df.tolist() == want[2]
        assert lo.tolist() == want[0] and co.tolist() == [want[1]]


def test_library_refuses_grids_past_32_bits():
    import ctypes
    a = _attn_args(N=65536, B=65536, Hq=1024, Hk=1024, D=16, workspace=4096, workspace_bytes=1 << 60)
    assert N.lib().hc_prefix_attn(ctypes.addressof(a), None) == N.HC_ERR_INVALID
    assert b"workgroups" in N.lib().hc_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("requests,new,D,share", [(33, 1, 64, False), (70, 1, 128, True), (29, 3, 32, True), (9, 16, 128, False)])
def test_query_rows_that_do_not_fill_a_tile(dtype, requests, new, D, share):
    """Batches whose query rows leave waves of a tile, or of the last one, without any."""
    g = torch.Generator().manual_seed(requests)
    lens = [int(x) for x in torch.randint(new, 40, (requests,), generator=g)]
    c = paged_case(dtype, lens, [new] * requests, prefix=1500, Hq=8, Hk=2, D=D, P=8, seed=requests)
    if new == 1:
        c["cu"] = None
    limits = torch.randint(0, 1501, (requests,), generator=g).int() if share else None
    d = to_dev(c)
    got, lse = attend(d, prefix_lens=None if limits is None else limits.cuda(), return_lse=True)
    check_attention(got, want_attention(c, limits), DTYPES[dtype], lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("prefix", [None, 0])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([300, 0, 7, 64] * 40, [1] * 160), ([500, 3, 129] * 24, [200, 3, 1] * 24)])
def test_requests_without_a_prompt(dtype, prefix, lens, new):
    c = paged_case(dtype, lens, new, prefix=prefix, Hq=4, Hk=2, D=64, P=16, seed=len(lens))
    got, lse = attend(to_dev(c), return_lse=True)
    check_attention(got, want_attention(c), DTYPES[dtype], lse)


@pytest.mark.gpu
def test_a_step_of_no_tokens():
    from hotcold_kv import SharedPromptBatch
    b = SharedPromptBatch(1, 3, 2, 64, torch.float16, "cuda", 4, 16, 32)
    assert b.extend(torch.zeros(3, dtype=torch.int32, device="cuda"), 0, 0).shape == (0,)
    z = torch.zeros((0, 2, 64), dtype=torch.float16, device="cuda")
    assert b.attend(0, torch.zeros((0, 8, 64), dtype=torch.float16, device="cuda"), z, z, 1.0).shape == (0, 8, 64)
    assert b.lens.tolist() == [0, 0, 0] and b.free_count.tolist() == [4]
