"""nn.Module surface of the bloom retrieval path, mirroring the reference's
silvertorch.modules (bloom_index_search_module.py, filter_query_parser_module.py
and their builders) over this build's torch.ops.st operators, and the
retrieval head and the query tower on them, which have no counterpart there."""

from silvertorch_amd.modules.bloom_index_search_module import BloomIndexSearchModule  # noqa: F401
from silvertorch_amd.modules.bloom_index_search_module_builder import (  # noqa: F401
    BloomIndexSearchModuleBuilder,
)
from silvertorch_amd.modules.filter_query_parser_module import FilterQueryParserModule  # noqa: F401
from silvertorch_amd.modules.filter_query_parser_module_builder import (  # noqa: F401
    FilterQueryParserModuleBuilder,
)
from silvertorch_amd.modules.query_tower_module import (  # noqa: F401
    Int8Linear,
    PackedQueryTowerModule,
    QueryTowerModule,
)
from silvertorch_amd.modules.retrieval_head_module import RetrievalHeadModule  # noqa: F401

__all__ = [
    "BloomIndexSearchModule",
    "BloomIndexSearchModuleBuilder",
    "FilterQueryParserModule",
    "FilterQueryParserModuleBuilder",
    "Int8Linear",
    "PackedQueryTowerModule",
    "QueryTowerModule",
    "RetrievalHeadModule",
]
