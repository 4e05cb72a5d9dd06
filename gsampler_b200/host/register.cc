// Registration of the custom class and operator library under the names the
// gSampler Python layer binds to (src/pybind.cc:9-78 in the gSampler tree).
#include <torch/custom_class.h>
#include <torch/script.h>

#include "graph.h"
#include "learn.h"
#include "ops.h"

using gsb_host::Graph;

TORCH_LIBRARY(gs_classes, m) {
  m.class_<Graph>("Graph")
      .def(torch::init<int64_t, int64_t>())
      .def("_CAPI_LoadCSC", &Graph::LoadCSC)
      .def("_CAPI_LoadCOO", &Graph::LoadCOO)
      .def("_CAPI_LoadCSR", &Graph::LoadCSR)
      .def("_CAPI_GetNumRows", &Graph::GetNumRows)
      .def("_CAPI_GetNumCols", &Graph::GetNumCols)
      .def("_CAPI_GetNumEdges", &Graph::GetNumEdges)
      .def("_CAPI_GetCSCIndptr", &Graph::GetCSCIndptr)
      .def("_CAPI_GetCSCIndices", &Graph::GetCSCIndices)
      .def("_CAPI_GetCSCEids", &Graph::GetCSCEids)
      .def("_CAPI_GetCOORows", &Graph::GetCOORows)
      .def("_CAPI_GetCOOCols", &Graph::GetCOOCols)
      .def("_CAPI_GetCOOEids", &Graph::GetCOOEids)
      .def("_CAPI_GetCSRIndptr", &Graph::GetCSRIndptr)
      .def("_CAPI_GetCSRIndices", &Graph::GetCSRIndices)
      .def("_CAPI_GetCSREids", &Graph::GetCSREids)
      .def("_CAPI_Slicing", &Graph::Slicing)
      .def("_CAPI_Sampling", &Graph::Sampling)
      .def("_CAPI_SamplingProbs", &Graph::SamplingProbs)
      .def("_CAPI_RandomWalk", &Graph::RandomWalk)
      .def("_CAPI_Node2Vec", &Graph::Node2Vec)
      .def("_CAPI_SDDMM", &Graph::SDDMM)
      .def("_CAPI_SpMM", &Graph::SpMM)
      .def("_CAPI_Compact", &Graph::Compact)
      .def("_CAPI_GraphRelabel", &Graph::GraphRelabel)
      .def("_CAPI_GetValidNodes", &Graph::GetValidNodes)
      .def("_CAPI_SlicingSampling", &Graph::FusedSlicingSampling)
      .def("_CAPI_FusedUOPV", &Graph::FusedUOPV)
      .def("_CAPI_FusedESquareSum", &Graph::FusedESquareSum)
      .def("_CAPI_FusedEDivUSum", &Graph::FusedEDivUSum)
      .def("_CAPI_SortCSCIndices", &Graph::SortCSCIndices)
      .def("_CAPI_BatchColSlicing", &Graph::BatchColSlicing)
      .def("_CAPI_BatchRowSlicing", &Graph::BatchRowSlicing)
      .def("_CAPI_BatchColRowSlcing", &Graph::BatchColRowSlcing)
      .def("_CAPI_BatchRowSampling", &Graph::BatchRowSampling)
      .def("_CAPI_BatchRowSamplingProbs", &Graph::BatchRowSamplingProbs)
      .def("_CAPI_BatchGraphRelabel", &Graph::BatchGraphRelabel)
      .def("_CAPI_BatchFusedSlicingSampling", &Graph::BatchFusedSlicingSampling)
      .def("_CAPI_GetEdgeBptr", &Graph::GetEdgeBptr)
      .def("_CAPI_GetColBptr", &Graph::GetColBptr)
      .def("_CAPI_GetRowBptr", &Graph::GetRowBptr)
      .def("_CAPI_SetEdgeBptr", &Graph::SetEdgeBptr)
      .def("_CAPI_SetColBptr", &Graph::SetColBptr)
      .def("_CAPI_SetRowBptr", &Graph::SetRowBptr)
      .def("_CAPI_BatchSetRows", &Graph::SetOrigRowIds)
      .def("_CAPI_BatchSetCols", &Graph::SetOrigColIds)
      .def("_CAPI_BatchGetRows", &Graph::BatchGetRows)
      .def("_CAPI_BatchGetCols", &Graph::BatchGetCols)
      .def("_CAPI_BatchGetCSCIndptr", &Graph::BatchGetCSCIndptr)
      .def("_CAPI_BatchGetCSCIndices", &Graph::BatchGetCSCIndices)
      .def("_CAPI_BatchGetCSCEids", &Graph::BatchGetCSCEids)
      .def("_CAPI_BatchGetCOORows", &Graph::BatchGetCOORows)
      // the reference binds this name to BatchGetCOORows (src/pybind.cc:62-63);
      // here it returns the columns its name promises
      .def("_CAPI_BatchGetCOOCols", &Graph::BatchGetCOOCols)
      .def("_CAPI_BatchGetCOOEids", &Graph::BatchGetCOOEids)
      .def("_CAPI_BatchGetColCounts", &Graph::BatchGetColCounts)
      .def("_CAPI_BatchGetValidNodes", &Graph::BatchGetValidNodes)
      // additions (no counterpart in the reference): random stream control and
      // the whole-sampler entry point
      .def("_CAPI_SetSeed", &Graph::SetSeed)
      .def("_CAPI_GetStreamCounter", &Graph::GetStreamCounter)
      .def("_CAPI_SetStreamCounter", &Graph::SetStreamCounter)
      .def("_CAPI_GetSeed", &Graph::GetSeed)
      .def("_CAPI_BatchGraphSAGE", &Graph::BatchGraphSAGE)
      .def("_CAPI_BatchGraphSAGEAsync", &Graph::BatchGraphSAGEAsync)
      .def("_CAPI_LadiesLayer", &Graph::LadiesLayer);
}

TORCH_LIBRARY(gs_ops, m) {
  m.def("_CAPI_ListSampling", &gsb_host::ListSampling);
  m.def("_CAPI_ListSamplingWithProbs", &gsb_host::ListSamplingProbs);
  m.def("_CAPI_BatchListSamplingWithProbs", &gsb_host::BatchListSamplingProbs);
  m.def("_CAPI_BatchListSampling", &gsb_host::BatchListSampling);
  m.def("_CAPI_BatchSplitByOffset", &gsb_host::SplitByOffset);
  m.def("_CAPI_BatchIndptrSplitByOffset", &gsb_host::SplitIndptrByOffset);
  m.def("_CAPI_IndexSearch", &gsb_host::IndexSearch);
  m.def("_CAPI_SetListSamplingSeed", &gsb_host::SetListSamplingSeed);
  m.def("_CAPI_GatherRows", &gsb_host::GatherRows);
  m.def("_CAPI_CheckAsyncErrors", &gsb_host::CheckAsyncErrors);
  // operators on learned node values (no counterpart in the reference)
  m.def("_CAPI_Embedding", &gsb_host::Embedding);
  m.def("_CAPI_EmbeddingGrad", &gsb_host::EmbeddingGrad);
  m.def("_CAPI_EmbeddingSparseGrad", &gsb_host::EmbeddingSparseGrad);
  m.def("_CAPI_Dropout", &gsb_host::Dropout);
  m.def("_CAPI_SetDropoutSeed", &gsb_host::SetDropoutSeed);
  m.def("_CAPI_NextDropoutStream", &gsb_host::NextDropoutStream);
  m.def("_CAPI_LinearCrossEntropy", &gsb_host::LinearCrossEntropy);
  m.def("_CAPI_LinearCrossEntropyTotal", &gsb_host::LinearCrossEntropyTotal);
  m.def("_CAPI_LinearCrossEntropyGrad", &gsb_host::LinearCrossEntropyGrad);
  // the same, differentiable
  m.def("_CAPI_EmbeddingLookup", &gsb_host::EmbeddingLookup);
  m.def("_CAPI_DropoutApply", &gsb_host::DropoutApply);
  m.def("_CAPI_LinearCrossEntropyLoss", &gsb_host::LinearCrossEntropyLoss);
}
