"""Calls of ops.dropout, ops.layer_norm and ops.linear_cross_entropy at the ends of what their documentation allows: masks that leave
nothing, values that are not finite, sizes that no launch fits, forms and tiles that a rule on sizes chooses. Tolerances as in
test_dense_tail.py: one rounding of the result, plus the fp32 roundings on the way, counted."""
import pytest
import torch

from test_dense_tail import BF16, F16, F32, Tail, check_xent, gen, gpu, head, mask_of, spec_of, tail_reference

TYPES = pytest.mark.parametrize("t", [F32, BF16, F16])


# ---- rows do not meet --------------------------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("n,K,C", [(700, 64, 5000), (700, 128, 5000), (700, 190, 5000), (700, 250, 5000)])
def test_rows_in_another_order_give_the_same_values(dev, hiplib, n, K, C, t):
    """a row's loss and gradient do not depend on which lane or workgroup has it, nor on the tiles its workgroup walks beside others:
    to the bit, in any order of the rows and each time (K up to 128, 192, 256: the narrow form)"""
    from pagraph_amd import ops
    g = gen(61 + K, dev)
    lin = head(dev, K, C, t, g)
    h = torch.randn(n, K, generator=g, device=dev).to(t)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    up = torch.randn(n, generator=g, device=dev)

    def values(order):
        x = h[order].requires_grad_()
        loss = ops.linear_cross_entropy(x, lin, lab[order], reduction="none")
        return [loss.detach()] + list(torch.autograd.grad(loss, [x], up[order]))
    want = values(torch.arange(n, device=dev))
    for k in range(4):
        order = torch.randperm(n, generator=g, device=dev)
        assert all(torch.equal(a, b[order]) for a, b in zip(values(order), want)), k


# ---- masks of the type's lowest value ----------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("K,n,C", [(24, 70, 520), (300, 70, 520), (300, 2100, 7000)])
def test_a_head_of_nothing_but_masked_classes_is_uniform(dev, hiplib, K, n, C, t):
    """every class masked by the type's lowest value: no logit is larger than another, so each class has one C-th (beside the lowest
    value of fp32 and bf16 any h W is lost, in fp16 it is not: its weight is 0)"""
    from pagraph_amd import ops
    g = gen(71, dev)
    lin = head(dev, K, C, t, g)
    with torch.no_grad():
        lin.bias.fill_(torch.finfo(t).min)
        if t == F16:
            lin.weight.zero_()
    h = torch.randn(n, K, generator=g, device=dev).to(t).requires_grad_()
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    each = ops.linear_cross_entropy(h, lin, lab, reduction="none")
    want = torch.full((n,), float(C), dtype=torch.float64, device=dev).log()
    # log2 of a whole number times ln 2: three roundings
    assert ((each.double() - want).abs() <= 4 * 2.0 ** -24 * want).all()
    dh, dw, db = torch.autograd.grad(each.sum(), [h, lin.weight, lin.bias])
    G = torch.full((n, C), 1.0 / C, dtype=torch.float64, device=dev)
    G.scatter_add_(1, lab.view(-1, 1), torch.full((n, 1), -1.0, dtype=torch.float64, device=dev))
    W, H = lin.weight.detach().double(), h.detach().double()
    # an element of G is off by its rounding to t (fp32: a few roundings), a sum by one rounding an addition, a result by half a step
    eg = torch.finfo(t).eps / 2 + 8 * 2.0 ** -24
    half, least = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal
    for got, ref, size, adds in ((dh, G @ W, G.abs() @ W.abs(), C), (dw, G.t() @ H, G.abs().t() @ H.abs(), n), (db, G.sum(0), G.abs().sum(0), n)):
        bound = size * (eg + (adds + 32) * 2.0 ** -24) + half * ref.abs() * 1.01 + least
        assert ((got.double() - ref).abs() <= bound).all()


@gpu
@TYPES
@pytest.mark.parametrize("K", [24, 300])
def test_a_label_whose_class_is_masked_by_the_lowest_value(dev, hiplib, K, t):
    """its loss is the mask's size, finite as in natural units, and its row pulls the masked class alone"""
    from pagraph_amd import ops
    g = gen(72, dev)
    n, C = 60, 400
    lin = head(dev, K, C, t, g)
    low = torch.finfo(t).min
    with torch.no_grad():
        lin.bias[100:130] = low
    h = torch.randn(n, K, generator=g, device=dev).to(t).requires_grad_()
    lab = torch.randint(130, C, (n,), generator=g, device=dev)
    lab[::4] = 107
    each = ops.linear_cross_entropy(h, lin, lab, reduction="none")
    z = h.detach().double() @ lin.weight.detach().double().t() + lin.bias.detach().double()
    want = torch.logsumexp(z, 1) - z.gather(1, lab.view(-1, 1)).view(-1)
    # logits of some 2 sqrt(K) at most beside the mask: (K + 16) roundings of a sum of absolute products, some of the mask's own size
    mag = (h.detach().double().abs() @ lin.weight.detach().double().abs().t()).amax(1) + 2.0
    bound = (2 * (K + 16) * mag + 400) * 2.0 ** -24 + torch.where(lab == 107, 16 * 2.0 ** -24 * abs(low), 0.0)
    assert ((each.double() - want).abs() <= bound).all()
    db, = torch.autograd.grad(each.sum(), lin.bias)
    assert db[107] == -15 and (db[100:107] == 0).all() and (db[108:130] == 0).all()


@gpu
@pytest.mark.parametrize("bias", [True, False])
def test_a_logit_at_the_lowest_value_in_base_2_that_is_no_mask(dev, hiplib, bias):
    """h W and the bias together can be what a masked class's bias alone is held as, and there may be no bias at all"""
    from pagraph_amd import ops
    product, b = float.fromhex("-0x1.04p+126"), float.fromhex("-0x1.c1c85ep+126")
    log2e = torch.tensor(1.4426950408889634).double()
    # one fused multiply-add of the logit times log2(e), as the kernel has it, is the lowest fp32 value
    assert (product * log2e + (b * log2e).float().double()).float().item() == torch.finfo(F32).min
    lin = torch.nn.Linear(1, 2, bias=bias, device=dev)
    with torch.no_grad():
        lin.weight.copy_(torch.tensor([[1.0], [0.0]]))
        if bias:
            lin.bias.copy_(torch.tensor([b, 0.0]))
    h = torch.full((5, 1), product, device=dev)
    each = ops.linear_cross_entropy(h, lin, torch.zeros(5, dtype=torch.int64, device=dev), reduction="none")
    want = -(product + (b if bias else 0.0))
    assert ((each.double() - want).abs() <= 8 * 2.0 ** -24 * want).all()


# ---- infinite weights ----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("K,n,C", [(40, 67, 400), (64, 128, 400), (300, 67, 400), (256, 1100, 9000)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_class_taken_out_by_infinite_weights(dev, hiplib, reduction, K, n, C, t):
    """a class whose weights are -inf where h is positive has the logit -inf: the rest of the head is as without it, and rows that do
    not count (ignored ones, and those a tile has behind the last row) bring no NaN into the head's gradients"""
    from pagraph_amd import ops
    g = gen(73, dev)
    lin = head(dev, K, C, t, g)
    h = (torch.rand(n, K, generator=g, device=dev) + 0.5).to(t)
    lab = torch.randint(10, C, (n,), generator=g, device=dev)
    lab[::5] = -100
    h[::5] = 0.0
    up = torch.randn(n, generator=g, device=dev) if reduction == "none" else torch.ones((), device=dev)
    out = []
    for by_weight in (True, False):
        with torch.no_grad():
            lin.bias[3] = 0.5 if by_weight else float("-inf")
            lin.weight[3] = float("-inf") if by_weight else 0.0
        loss = ops.linear_cross_entropy(h, lin, lab, reduction=reduction)
        out.append([loss.detach()] + list(torch.autograd.grad(loss, [lin.weight, lin.bias], up)))
    assert all(torch.isfinite(v).all() for v in out[0])
    assert all(torch.equal(a, b) for a, b in zip(*out))


# ---- gradients of single rows far apart ----------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("n,K,C", [(61, 40, 512), (61, 300, 512), (2100, 300, 7000), (2100, 800, 7000)])
def test_rows_whose_gradients_are_far_below_the_largest(dev, hiplib, n, K, C, t):
    """a row's gradient is as exact however large another row's is. h is orthogonal to every class: all probabilities are 1 / C, a
    rounding of them that is the same for all would show in dh = up * (mean of W's rows - W[label])"""
    from pagraph_amd import ops
    g = gen(74, dev)
    lin = head(dev, K, C, t, g)
    with torch.no_grad():
        lin.weight.copy_(1.0 + (torch.arange(C, device=dev) % 2).to(t).view(C, 1) * torch.ones(K, device=dev, dtype=t))        # rows of 1, of 2
        lin.bias.zero_()
    h = torch.tensor([1.0, -1.0], device=dev).repeat(n, K // 2).to(t).requires_grad_()
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    # (exponents that leave dh, of fp16 too, its normal range: 2^13 to 2^-13 times 1/2)
    up = torch.exp2(13.0 - 26.0 * torch.rand(n, generator=g, device=dev))
    up[0] = 2.0 ** 13
    dh, db = torch.autograd.grad(ops.linear_cross_entropy(h, lin, lab, reduction="none"), [h, lin.bias], up)
    own = lin.weight.detach().double()[lab, 0]
    want = up.double() * (1.5 - own)
    # an element of G is off by half a step of its type (fp32: a few roundings): C of 1 / C with weights of 1.5 on average, and the
    # label's 1 / C - 1 with its weight, that is 1.5 + own in all; C additions; the result's own half step
    half = torch.finfo(t).eps / 2
    bound = up.double() * (1.5 + own) * ((half if t != F32 else 8 * 2.0 ** -24) + (C + 32) * 2.0 ** -24) + half * want.abs() * 1.01 + 2.0 ** -25
    assert ((dh.double() - want.view(n, 1)).abs() <= bound.view(n, 1)).all()
    G = (up.double() / C).sum() - torch.zeros(C, dtype=torch.float64, device=dev).index_add_(0, lab, up.double())
    # (a sum over the rows: half a step of G's type of each, fp16 G's smallest step 2^-24 of the largest row times 2^14)
    eb = (up.double().sum() + up.double().sum() / C) * (half + (n + 40) * 2.0 ** -24) + n * 2.0 ** 13 * 2.0 ** -38
    assert ((db.double() - G).abs() <= eb + half * G.abs() * 1.01).all()


# ---- the ends of fp32 ----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("K", [8, 300])
@pytest.mark.parametrize("big", [3.4e38, -3.4028234e38, 3.3895e38, 3.392e38])
def test_fp32_values_above_the_largest_of_bf16(dev, hiplib, K, big):
    """fp32 is multiplied in three bf16 parts; a finite value whose rounding to bf16 is infinite is finite all the same, in h and in
    the head. Weights of whole numbers times 2^-124 have one part, logits are some 16 times those numbers"""
    from pagraph_amd import ops
    g = gen(75, dev)
    n, C = 50, 200
    lin = head(dev, K, C, F32, g, bias=False)
    h = torch.zeros(n, K, device=dev)
    h[:, 0] = big
    with torch.no_grad():
        lin.weight.zero_()
        lin.weight[:, 0] = torch.randint(-8, 9, (C,), generator=g, device=dev).float() * 2.0 ** -124
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    for x, m in ((h, lin), (lin.weight.detach()[:n] * 1.0, torch.nn.Linear(K, C, bias=False, device=dev))):
        if m is not lin:
            with torch.no_grad():
                m.weight.zero_()
                m.weight[:, 0] = big
                m.weight[::2, 0] *= 0.5
        x = x.detach().requires_grad_()
        each = ops.linear_cross_entropy(x, m, lab, reduction="none")
        z = x.detach().double() @ m.weight.detach().double().t()
        want = torch.logsumexp(z, 1) - z.gather(1, lab.view(-1, 1)).view(-1)
        # |z| <= 128: one product of three parts, the logit's rounding in base 2, the sum's; 400 as everywhere for the exponentials
        assert ((each.double() - want).abs() <= (8 * 128 + 400) * 2.0 ** -24).all()
        dx, = torch.autograd.grad(each.sum(), x)
        assert torch.isfinite(dx).all()


@gpu
@pytest.mark.parametrize("K", [40, 300])
def test_fp32_infinities_stay_with_their_rows(dev, hiplib, K):
    """an infinite element of a row makes that row's loss NaN and no other's"""
    from pagraph_amd import ops
    g = gen(76, dev)
    lin = head(dev, K, 500, F32, g)
    h = torch.randn(90, K, generator=g, device=dev)
    lab = torch.randint(0, 500, (90,), generator=g, device=dev)
    bad = h.clone()
    bad[11, 3], bad[64, K - 1] = float("inf"), float("-inf")
    rest = torch.ones(90, dtype=torch.bool, device=dev)
    rest[11], rest[64] = False, False
    out = []
    for x in (h, bad):
        x = x.requires_grad_()
        each = ops.linear_cross_entropy(x, lin, lab, reduction="none")
        out.append((each.detach(), torch.autograd.grad(each.sum(), x)[0]))
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(*out))
    assert torch.isnan(out[1][0][~rest]).all() and torch.isnan(out[1][1][~rest]).all()


# ---- sizes that no launch fits, and those that need more than one round of it -----------------------------------------------------
def test_sizes_beyond_a_launch_are_refused_before_anything_is_allocated(hiplib):
    """a launch has fewer than 2^32 threads: what needs more is refused by the call that sizes the workspace"""
    from pagraph_amd import _lib as L
    scratch = hiplib.pg_linear_xent_scratch
    for back in (0, 1):
        # logits: tiles of 256 x 128 and 256 threads, of 256 x 256 and 512 threads; a piece of the classes at a time for gradients
        assert scratch(1 << 20, 512, 1 << 18, L.PG_DTYPE_BF16, back) > 0
        assert scratch(1 << 18, 1024, 1 << 20, L.PG_DTYPE_BF16, back) > 0
        assert (scratch(1 << 20, 512, 1 << 20, L.PG_DTYPE_BF16, back) < 0) == (back == 0)
        assert (scratch(1 << 22, 1024, 1 << 17, L.PG_DTYPE_BF16, back) < 0) == (back == 0)
        # narrow: 128 rows and 256 threads a workgroup
        assert scratch((1 << 31) - 128, 64, 61, L.PG_DTYPE_F32, back) > 0
        assert scratch(1 << 31, 64, 61, L.PG_DTYPE_F32, back) < 0
    # dh's tiles: 4 to each 256 rows, of 512 threads
    assert scratch(1 << 28, 1024, 128, L.PG_DTYPE_BF16, 1) > 0 and scratch(1 << 30, 1024, 128, L.PG_DTYPE_BF16, 1) < 0


def test_a_workspace_that_is_not_aligned_is_refused(hiplib):
    import ctypes
    from pagraph_amd import _lib as L
    x = L.PgLinearXentDesc()
    for name in ("h", "W", "labels", "top", "sum", "row_loss", "loss", "meta", "grad", "dh", "dW", "db"):
        setattr(x, name, 4096)                       # (never looked at)
    x.n, x.K, x.C, x.h_stride, x.w_stride = 4, 8, 8, 8, 8
    for scratch in (4100, 4104, 4097):
        x.scratch = scratch
        assert hiplib.pg_linear_xent_fwd(ctypes.addressof(x), None) == hiplib.pg_linear_xent_bwd(ctypes.addressof(x), None) == -1


@gpu
@pytest.mark.parametrize("t", [F32, F16])
def test_more_rows_than_workgroups_of_a_launch(dev, hiplib, t):
    """the joining of the rows' statistics goes round its grid: 262144 rows at a time"""
    from pagraph_amd import ops
    g = gen(77, dev)
    n, K, C = 600001, 16, 61
    lin = head(dev, K, C, t, g)
    h = torch.randn(n, K, generator=g, device=dev).to(t)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    with torch.no_grad():
        each = ops.linear_cross_entropy(h, lin, lab, reduction="none")
        parts = [ops.linear_cross_entropy(h[i:i + 200000], lin, lab[i:i + 200000], reduction="none") for i in range(0, n, 200000)]
    assert (each - torch.cat(parts)).abs().max() <= 64 * 2.0 ** -24 * each.abs().max()


# ---- graphs that live beside a capture -------------------------------------------------------------------------------------------
@pytest.fixture
def watched(monkeypatch):
    """an operator that ops._watch_graph watches, without a GPU: whether its stream captures, and which it is, are made up"""
    from pagraph_amd import ops
    state = {"capturing": False, "stream": 1}
    monkeypatch.setattr(ops, "_capture_state", lambda device: (state["capturing"], state["stream"]))
    monkeypatch.setattr(ops, "_EAGER_GRAPHS", type(ops._EAGER_GRAPHS)())

    class F(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ops._watch_graph("f", ctx, x.device, x, w)
            return x * w

        @staticmethod
        def backward(ctx, g):
            return g, g
    return F, state


def test_a_capture_meets_no_living_graph_of_leaves_behind_its_inputs(watched):
    from pagraph_amd import _lib
    F, state = watched
    x, w, u, v = (torch.ones(3, requires_grad=True) for _ in range(4))
    fixed = torch.ones(3)
    kept = F.apply(torch.relu(x * w), fixed) + 1.0
    state.update(capturing=True, stream=2)
    F.apply(torch.tanh(u) * v, v)                            # other leaves
    F.apply(fixed, u)
    for f in (lambda: F.apply(torch.tanh(u * w), v), lambda: F.apply(u, (x + v) * 2.0), lambda: F.apply(w, fixed)):
        with pytest.raises(_lib.PgError, match="still alive"):
            f()
    state.update(stream=1)
    F.apply(torch.tanh(u * w), v)                            # the stream the graph was recorded on
    state.update(stream=2)
    del kept
    F.apply(torch.tanh(u * w), v)


def test_graphs_are_recorded_by_other_threads_during_a_capture(watched, monkeypatch):
    """another thread's eager graph comes in while a capture goes through those that live"""
    import threading
    from pagraph_amd import ops
    F, state = watched
    kept, others = [], []

    def record():
        kept.append(F.apply(torch.ones(3, requires_grad=True), torch.ones(3)))

    class Interrupted(type(ops._EAGER_GRAPHS)):
        def __iter__(self):
            graphs = super().__iter__()
            for graph in graphs:
                yield graph
                others.append(threading.Thread(target=record))
                others[-1].start()
                others[-1].join(0.3)                 # (comes in now, or waits until the capture is through them)
    monkeypatch.setattr(ops, "_EAGER_GRAPHS", Interrupted())
    here = threading.get_ident()
    monkeypatch.setattr(ops, "_capture_state", lambda device: (state["capturing"] and threading.get_ident() == here, state["stream"]))
    for _ in range(3):
        record()
    state.update(capturing=True, stream=2)
    u = torch.ones(3, requires_grad=True)
    F.apply(u, u)
    for other in others:
        other.join()
    assert len(kept) == 6


# ---- dropout where it reads ---------------------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("n,d", [(1, 3), (50, 64), (333, 602), (7, 2048), (2, 9001)])
def test_dropout_in_place(dev, hiplib, n, d, t):
    """pg_dropout_apply may write where it reads"""
    import ctypes
    from pagraph_amd import _lib as L
    from pagraph_amd import ops
    spec = spec_of(dev, 0.4)
    x = torch.randn(n, d, generator=gen(78, dev), device=dev).to(t)
    want = ops.dropout(x, spec)
    drop = L.PgDropout(spec.threshold, spec.tag, spec.seed, spec.step.data_ptr(), 0)
    L.check(hiplib.pg_dropout_apply(x.data_ptr(), d, x.data_ptr(), d, n, d, ops._DTYPES[t], ctypes.addressof(drop), None, L.stream_ptr()),
            "pg_dropout_apply")
    assert torch.equal(x, want)


# ---- the parts of fp32 products ----------------------------------------------------------------------------------------------------
# values whose bf16 parts are (1, 0, 0), (1, 2^-8, 0) and (1, 2^-9, 2^-17)
PARTS = (1.0, 1.0 + 2.0 ** -8, 1.0 + 2.0 ** -9 + 2.0 ** -17)


def three_parts(x):
    parts = []
    for _ in range(3):
        parts.append(torch.tensor(x, dtype=torch.float64).to(BF16).double().item())
        x -= parts[-1]
    return parts, x


def test_the_parts_are_what_they_are_taken_for():
    assert [three_parts(x) for x in PARTS] == [([1.0, 0.0, 0.0], 0.0), ([1.0, 2.0 ** -8, 0.0], 0.0), ([1.0, 2.0 ** -9, 2.0 ** -17], 0.0)]


@gpu
@pytest.mark.parametrize("n,K,C", [(2, 1, 2), (2, 100, 2), (300, 128, 3000), (2, 300, 2), (2100, 300, 7000), (5000, 1030, 9000), (300, 1030, 70000)])
def test_fp32_products_keep_every_part_that_is_not_below_2_to_the_minus_23(dev, hiplib, n, K, C):
    """logits of +-1024 in one row and two classes (the others masked, the other rows not counted, but one with a gradient of its own),
    so that loss, dh and dW are single products of values whose parts are known. A product that lacked one of its six would be off
    by 2^-16 (middle times middle) or 2^-17 (lowest times first, either way round)"""
    from pagraph_amd import ops
    lin = torch.nn.Linear(K, C, device=dev)
    h = torch.zeros(n, K, device=dev, requires_grad=True)
    lab = torch.full((n,), -100, dtype=torch.int64, device=dev)
    up = torch.zeros(n, device=dev)
    row, other, one, two, col = n - 1, 0, 0, C - 1, K - 1
    lab[other], lab[row] = one, two
    with torch.no_grad():
        lin.weight.zero_()
        lin.bias.fill_(float("-inf"))
        lin.bias[one], lin.bias[two] = 0.0, 0.0
    for x in PARTS:
        for y in PARTS:
            for f in PARTS:
                with torch.no_grad():
                    h[row, col] = 32.0 * x
                    lin.weight[one, col], lin.weight[two, col] = 32.0 * y, -32.0 * y
                up[other], up[row] = 1.0, 0.5 * f
                each = ops.linear_cross_entropy(h, lin, lab, reduction="none")
                dh, dw, db = torch.autograd.grad(each, [h, lin.weight, lin.bias], up)
                # the three products left out are below 2^-22.9; six partial sums, into base 2 and out of it: 2^-24 each. (the gradients:
                # the factors' quotient and product, G's own roundings)
                off = 2.0 ** -22.9 + 12 * 2.0 ** -24
                for got, want in ((each[row], 2048.0 * x * y), (dh[row, col], 32.0 * y * f), (dw[one, col], 16.0 * x * f), (dw[two, col], -16.0 * x * f)):
                    assert abs(got.item() - want) <= off * abs(want), (x, y, f, got.item(), want)
                # (the other row: two equal logits)
                assert abs(db[one].item() - (0.5 * f - 0.5)) <= off and abs(db[two].item() - (0.5 - 0.5 * f)) <= off
                assert abs(each[other].item() - 0.6931471805599453) <= off


# ---- forms that a rule on sizes chooses ---------------------------------------------------------------------------------------------
@gpu
@TYPES
@pytest.mark.parametrize("n,K,C", [(2100, 300, 7000), (4099, 1030, 8200)])
@pytest.mark.parametrize("bias,reduction", [(True, "none"), (False, "none"), (False, "mean"), (False, "sum")])
def test_large_tiles_with_row_gradients_and_without_a_bias(dev, hiplib, bias, reduction, n, K, C, t):
    check_xent(dev, n, K, C, t, ignored=0.1, reduction=reduction, bias=bias)


@gpu
def test_gradients_of_the_tail_against_differences_along_them(dev, hiplib, oracle):
    """the losses' own differences along each gradient, where they are largest. In 64 bits, how far a difference is from the derivative;
    the kernels' losses are off by some 300 roundings one behind the other (two layers of depth <= 64, the row sums of 230 and 90), on
    either side. Both together are well below the gradient: zeros, or the wrong sign, would not pass"""
    g = gen(79, dev)
    n, d, C = 90, 60, 230
    m = Tail(d, C, dev)
    x = torch.randn(n, d, generator=g, device=dev, requires_grad=True)
    lab = torch.randint(0, C, (n,), generator=g, device=dev)
    lab[::11] = -100
    s1, s2 = spec_of(dev, 0.2, tag=1), spec_of(dev, 0.4, tag=2)
    k1, k2 = [(lambda km: km[0].to(dev).double() * km[1])(mask_of(oracle, n, d, s, 5)) for s in (s1, s2)]
    leaves = [x] + list(m.parameters())
    grads = torch.autograd.grad(m(x, lab, s1, s2), leaves)
    loss, exact = tail_reference(m, x, lab, k1, k2)
    with torch.no_grad():
        for p, gp, ge in zip(leaves, grads, exact):
            size = ge.norm().item()
            v, old, e, both = (ge / size).float(), p.detach().clone(), 5e-2, []
            for sign in (e, -e):
                p.copy_(old + sign * v)
                with torch.enable_grad():
                    both.append((m(x, lab, s1, s2).item(), tail_reference(m, x, lab, k1, k2)[0].item()))
            p.copy_(old)
            here, there = [(a - b) / (2 * e) for a, b in zip(*both)]
            along = (gp.double() * v.double()).sum().item()
            bound = abs(there - size) + 300 * 2.0 ** -24 * loss.item() / e
            assert bound < 0.25 * size, (p.shape, bound, size)
            assert abs(here - along) <= bound, (p.shape, here, along, bound)
