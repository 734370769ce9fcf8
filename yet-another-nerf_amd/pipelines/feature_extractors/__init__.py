from .builder import FEATURE_EXTRACTORS  # noqa: F401
from . import code_table, identity_mapper  # noqa: F401
