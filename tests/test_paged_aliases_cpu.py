"""Which operands of the paged-cache operators may share memory: what a launch writes over rows that other blocks of it still read
is refused, and in place means at the same pitch."""
from __future__ import annotations

import pytest

from aginfer_b200.recipes import Arena, PagedCache, RecipeBuilder, Tensor, io

HEADS, KV, DIM, ROWS = 8, 2, 128, 5
QKV, Q, KEYS = (HEADS + 2 * KV) * DIM, HEADS * DIM, KV * DIM
AT = Arena(1 << 20)


def builder() -> RecipeBuilder:
    r = RecipeBuilder({"w": ("BF16", (8,))})
    pool = [9, KV, DIM // 64, 16, 64]
    r.begin_profile("default", [io("q", "BF16", [ROWS, Q]), io("table", "I32", [3, 4]), io("lengths", "I32", [3]), io("starts", "I32", [4])],
                    [io("x", "BF16", [ROWS, QKV]), io("flat", "BF16", [ROWS * QKV]), io("key", "BF16", [ROWS, Q]), io("o", "BF16", [ROWS, Q]), io("k", "BF16", pool),
                     io("v", "BF16", pool)])
    return r


def cache() -> PagedCache:
    return PagedCache(k=Tensor("k"), v=Tensor("v"), table=Tensor("table"), lengths=Tensor("lengths"), starts=Tensor("starts"), sequences=3, pages=9,
                      page=16, pages_per_sequence=4, kv_heads=KV, head_dim=DIM)


def append(q, out, **kw):
    """Row and output pitch of the launch."""
    r = builder()
    r.kv_append(q, out, cache(), rows=ROWS, q_heads=HEADS, theta=1e6, **kw)
    (launch,) = [l for l in r._profile.launches if l["kernel"] == "agi_kv_append_bf16"]
    values = [a.get("scalar_u32") for a in launch["arguments"]]
    return values[22], values[24]


@pytest.mark.parametrize("x", [Tensor("x"), AT], ids=["tensor", "arena"])
def test_queries_turned_in_place_keep_their_pitch(x):
    assert append(x, x) == (QKV, QKV)
    assert append(x, x, out_stride=QKV) == (QKV, QKV)
    assert append(x, Tensor("o")) == (QKV, Q)


@pytest.mark.parametrize("q,out,kw", [
    (Tensor("flat"), Tensor("flat"), dict(out_stride=Q)),
    (AT, AT, dict(out_stride=QKV + 8)),
    (AT, AT + 2 * Q, {}),                                     # over the keys
    (AT, AT + 2 * KEYS, dict(out_stride=QKV)),                # over queries of the same row that other threads read
    (AT + 2 * Q, AT, dict(out_stride=Q)),                     # a block of outputs that ends inside what is read
    (AT, AT + 2 * (QKV * (ROWS - 1) + QKV - 8), {}),          # the last row's last values
    (Tensor("q"), Tensor("key"), dict(k=Tensor("key"), v=Tensor("o"), kv_stride=Q)),
    (Tensor("q"), Tensor("key"), dict(k=Tensor("o"), v=Tensor("key"), kv_stride=Q)),
    (AT, AT, dict(row_stride=QKV, k=AT + 2 * (Q - 8), v=AT + 2 * (Q + KEYS), kv_stride=QKV)),
], ids=str)
def test_outputs_over_what_is_still_read_are_refused(q, out, kw):
    with pytest.raises(ValueError, match="still read"):
        append(q, out, **kw)


@pytest.mark.parametrize("q,out,kw", [
    (AT, AT + 2 * QKV * ROWS, {}), (AT + 2 * Q * ROWS, AT, {}),                                                # behind, in front
    (AT, AT, dict(row_stride=QKV, k=AT + 2 * Q, v=AT + 2 * (Q + KEYS), kv_stride=QKV)),                        # fused rows given apart
    (AT, AT + 2 * QKV, dict(row_stride=QKV + Q, out_stride=QKV + Q)),                                          # columns of the same rows
], ids=str)
def test_outputs_beside_what_is_read_are_taken(q, out, kw):
    append(q, out, **kw)


@pytest.mark.parametrize("longest", [1, ROWS])
@pytest.mark.parametrize("prefix", [False, True])
def test_attention_in_place_is_at_the_same_pitch(longest, prefix):
    def attend(q, o, **kw):
        common = dict(rows=ROWS, q_heads=HEADS, longest=longest) | kw
        if prefix:
            builder().prefix_attention(q, o, cache(), AT + (1 << 20), AT + (1 << 20) + 64, prefix_pages=2, **common)
        else:
            builder().paged_attention(q, o, cache(), **common)

    attend(AT, AT)
    for x in (Tensor("x"), AT):
        attend(x, x, q_stride=QKV, o_stride=QKV)
    for strides in (dict(q_stride=QKV), dict(o_stride=QKV)):
        with pytest.raises(ValueError, match="still read"):
            attend(AT, AT, **strides)
    with pytest.raises(ValueError, match="still read"):
        attend(AT, AT + 16)
    attend(AT, AT + 2 * Q * ROWS)
    attend(AT, AT + 2 * Q, q_stride=QKV + Q, o_stride=QKV + Q)
