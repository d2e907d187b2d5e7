"""CPU: arguments of the attention operators at the edges of their ranges."""
ARGS = -2
P = 0x10000  # an address that nothing looks at


def test_documents_without_keys():
    """With no keys their ids, like the keys themselves, are not looked at (an empty tensor has no address)."""
    import ajib
    op = lambda lk: ajib.attn_op(ajib.F16, 0, 5, lk, 4, 2, 64, 0.125, q_doc=P, doc_rows=1)  # a batch of none: checked alone
    q = ajib.heads(P, 1280, 256, 64)
    assert ajib.attention(op(0), q, None, None, q) == 0
    assert ajib.attention(op(3), q, q, q, q) == ARGS
