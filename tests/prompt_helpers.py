"""What the tests of prompt attention share."""


def form(rows, requests, heads, kv_heads):
    """The rows (tokens x heads of a group) of the library's row tiles for a call of these sizes: 64 with keys split
    among waves, 128 in workgroups of four waves, 256 of eight."""
    if rows * heads <= 256 * 64 and requests * kv_heads <= 256:
        return 64
    return 256 if rows * heads >= 200 * 256 and rows // 512 >= requests else 128
