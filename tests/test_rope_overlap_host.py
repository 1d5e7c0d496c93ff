"""Which rows of rotary positions share memory, on the CPU: calls that are refused, and calls that come as far as a later refusal."""
import ctypes as C
import random

from tests.test_rope_host import FAKE, _refused


def _places(at, strides, sizes, head):
    out = [at]
    for stride, n in zip(strides, sizes):
        out = [x + stride * i for x in out for i in range(n)]
    return [x + d for x in out for d in range(head)]


def test_overlap_is_found_exactly_where_it_is(abi):
    """x_out in any place and layout beside x, against the sets of their elements. (y is missing: a call whose x and x_out are accepted is refused for that, in front of any launch.)"""
    rng, seen, err = random.Random(5), {}, C.create_string_buffer(256)
    for _ in range(6000):
        B, S, heads, head = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3), 2 * rng.randint(1, 6)
        layout = lambda: rng.choice([(S * heads * head, heads * head, head), (heads * S * head, head, S * head), (S * 3 * heads * head, 3 * heads * head, head), (3 * heads * S * head, head, S * head),
                                     tuple(rng.randint(0, 6 * head) for _ in range(3)), (rng.randint(0, 100), rng.randint(0, 50), head)])
        x, out = layout(), layout()
        if rng.random() < 0.6:
            out = x
        at = rng.choice([0, 1, head, head * heads, head * S, heads * S * head, rng.randint(0, 80)]) * rng.choice([-1, 1])
        places, others = (_places(p, strides, (B, S, heads), head) for p, strides in ((0, x), (at, out)))
        strides = lambda s: [a if n > 1 else 0 for a, n in zip(s, (B, S, heads))]
        want = "share memory" if len(set(others)) < len(others) else "y must be given" if (at == 0 and strides(x) == strides(out)) or not set(places) & set(others) else "x_out must be x"
        a = abi.RopeArgs(x=abi.Kv4Rows(FAKE, *x), x_out=abi.Kv4Rows(FAKE + 2 * at, *out), turns=FAKE, positions=FAKE, B=B, S=S, heads_x=heads, heads_y=1, head_dim=head, rotary=2, factor=1.0)
        assert abi.load().fmha_rope_rotate(a, None, err, 256) == 6
        assert want in err.value.decode(), (B, S, heads, head, x, out, at, err.value)
        seen[want] = seen.get(want, 0) + 1
    assert all(n > 300 for n in seen.values()) and len(seen) == 3, seen


def test_heads_in_front_of_tokens(abi):
    """One projection [B, heads, S, D]: heads that both have are found, x_out in heads behind x's is no overlap."""
    B, S, D, H, HK = 2, 5, 64, 4, 2
    part = lambda first: abi.Kv4Rows(FAKE + 2 * first * S * D, (2 * H + 2 * HK) * S * D, D, S * D)
    more = dict(B=B, S=S, heads_x=H, heads_y=HK)
    _refused(abi, "other input or output", x=part(0), x_out=part(0), y=part(H - 1), y_out=part(H - 1), **more)
    _refused(abi, "x_out must be x", x=part(0), x_out=part(H - 1), **more)
    _refused(abi, "y must be given", x=part(0), x_out=part(H), y=abi.Kv4Rows(), **more)


def test_rows_of_one_batch_between_the_rows_of_another(abi):
    """Strides of 150 and 100 elements: heads of 40 at 0 and at 50 meet at 150, where one's second sequence begins and the other's first sequence has its second token."""
    rows = lambda first: abi.Kv4Rows(FAKE + 2 * first, 150, 100, 40)
    more = dict(B=2, S=2, heads_x=1, heads_y=1, head_dim=40, rotary=40)
    _refused(abi, "other input or output", x=rows(0), x_out=rows(0), y=rows(50), y_out=rows(50), **more)
    _refused(abi, "x_out must be x", x=rows(0), x_out=rows(50), **more)
