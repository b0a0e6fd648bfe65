"""What a status word says: the fault's text names what can have caused it."""

from wayfinder_attention_b200._lib import describe_status


def test_texts():
    assert "attention index" in describe_status(1) and "token" in describe_status(1)
    assert "out of range" in describe_status(1) and "timed out" not in describe_status(1)
    assert "timed out" in describe_status(2 | 32) and "0x2" in describe_status(2 | 32)
    assert "out of range" in describe_status(3) and "timed out" in describe_status(3)
    assert "unknown" in describe_status(1 << 20)
