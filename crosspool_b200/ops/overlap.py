"""Whether the rows of a result lie over those of an input."""


def rows_meet(rows: int, at_a: int, pitch_a: int, width_a: int, at_b: int, pitch_b: int, width_b: int) -> bool:
    """Whether ``rows`` rows of ``width_a`` bytes, ``pitch_a`` bytes apart from address ``at_a`` on, and the rows ``b`` share memory.
    Rows of one pitch may stand side by side in a wider buffer; of rows of different pitches the whole ranges must not meet."""
    if rows == 0 or at_b >= at_a + (rows - 1) * pitch_a + width_a or at_a >= at_b + (rows - 1) * pitch_b + width_b:
        return False
    if rows == 1 or pitch_a != pitch_b or pitch_a == 0:
        return True
    d = (at_b - at_a) % pitch_a          # where in the pitch b's rows begin, seen from a's
    return d < width_a or d + width_b > pitch_a
