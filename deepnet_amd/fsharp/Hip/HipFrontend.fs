namespace Tensor

// The HipTensor module: creation functions on the HIP device, mirroring Tensor/Tensor/Cuda/CudaFrontend.fs:30-149.
// Source only (no .NET SDK on this repository's build machine).

open System
open System.Runtime.InteropServices
open Tensor.Backend
open Tensor.Hip

module HipTensor =
    /// the HIP tensor device
    let Dev = TensorHipDevice.Instance :> ITensorDevice

    /// copies a tensor (normally a HostTensor) to the HIP device
    let transfer x = Tensor.transfer Dev x

    let empty<'T> = Tensor<'T>.empty Dev
    let zeros<'T> = Tensor<'T>.zeros Dev
    let ones<'T> = Tensor<'T>.ones Dev
    let falses = Tensor.falses Dev
    let trues = Tensor.trues Dev
    let scalar<'T> = Tensor<'T>.scalar Dev
    let filled<'T> = Tensor<'T>.filled Dev
    let identity<'T> = Tensor<'T>.identity Dev
    let counting = Tensor.counting Dev
    let arange<'T> = Tensor<'T>.arange Dev
    let linspace<'T> = Tensor<'T>.linspace Dev

    /// <summary>Creates a tensor from the given device pointer, allocation size in bytes, type and layout
    /// (the counterpart of CudaTensor.usingPtrAndType, Tensor/Tensor/Cuda/CudaFrontend.fs:129-137).</summary>
    /// <remarks>The data is referenced, not copied, and is never freed by the tensor: changing values within the tensor changes
    /// the original data, and the memory must outlive the tensor.</remarks>
    let usingPtrAndType (ptr: nativeint) (sizeInBytes: int64) (typ: Type) (layout: TensorLayout) =
        let elemSize = int64 (System.Runtime.InteropServices.Marshal.SizeOf typ)
        let storType = typedefof<TensorHipStorage<_>>.MakeGenericType [|typ|]
        let ofPointer = storType.GetMethod "OfPointer"
        let stor = ofPointer.Invoke (null, [|box ptr; box (sizeInBytes / elemSize)|])
        let tensorType = typedefof<Tensor<_>>.MakeGenericType [|typ|]
        Activator.CreateInstance (tensorType, [|box layout; stor|]) :?> ITensor

    /// <summary>Creates a tensor from the given device pointer, allocation size in bytes and layout
    /// (the counterpart of CudaTensor.usingPtr, Tensor/Tensor/Cuda/CudaFrontend.fs:139-149).</summary>
    let usingPtr<'T> (ptr: nativeint) (sizeInBytes: int64) (layout: TensorLayout) =
        usingPtrAndType ptr sizeInBytes typeof<'T> layout :?> Tensor<'T>

/// Operators of language models on tensors of the HIP device (no counterpart in ITensorBackend): token embedding, token log
/// probabilities, cross attention, each with its gradient.  include/tensor_hip.h states shapes and semantics; 'T is single or double.
module HipModel =
    let private desc (t: Tensor<'A>) =
        let st = (t :> ITensorFrontend<'A>).Storage :?> TensorHipStorage<'A>
        box t, Desc.make st.Ptr typeof<'A> t.Layout
    let private opt (t: Tensor<'A> option) = t |> Option.map desc
    let private some t = Some (desc t)

    /// Calls f with the addresses of the descriptors (IntPtr.Zero for None), which the library copies before it returns.
    let private call (ts: (obj * DnhTensor) option list) (f: nativeint[] -> int) =
        let size = Marshal.SizeOf (typeof<DnhTensor>)
        let block = Marshal.AllocHGlobal (max 1 (size * List.length ts))
        try
            ts
            |> List.mapi (fun i t ->
                match t with
                | Some (_, d) ->
                    let p = block + nativeint (i * size)
                    Marshal.StructureToPtr (d, p, false)
                    p
                | None -> IntPtr.Zero)
            |> Array.ofList |> f |> Native.check
        finally
            Marshal.FreeHGlobal block
            ts |> List.iter (Option.iter (fun (t, _) -> GC.KeepAlive t))

    /// The same with the address of one host element, IntPtr.Zero for None.
    let private callScaled (scale: 'T option) ts (f: nativeint -> nativeint[] -> int) =
        match scale with
        | Some s -> Desc.withScalar s (fun p -> call ts (f p))
        | None -> call ts (f IntPtr.Zero)

    let private checkIndexError () =
        if Cfg.Stacktrace then
            let mutable code = 0
            Native.check (Native.dnh_async_error (Cfg.Stream, &code))
            Native.check code

    let private like (t: Tensor<'A>) shape : Tensor<'A> = Tensor<'A> (shape, HipTensor.Dev)

    /// scale * table.[tokens.[i], *]
    let embedding (scale: 'T option) (table: Tensor<'T>) (tokens: Tensor<int64>) : Tensor<'T> =
        let out = like table (tokens.Shape @ [table.Shape.[1]])
        callScaled scale [some out; some table; some tokens] (fun s p -> Native.embedding (p.[0], p.[1], p.[2], s, Cfg.Stream))
        checkIndexError ()
        out

    /// Gradient of embedding with respect to a table of `vocab` rows.
    let embeddingGrad (scale: 'T option) (vocab: int64) (tokens: Tensor<int64>) (dOut: Tensor<'T>) : Tensor<'T> =
        let dTable = like dOut [vocab; List.last dOut.Shape]
        callScaled scale [some dTable; some tokens; some dOut] (fun s p ->
            Native.embedding_grad (p.[0], p.[1], p.[2], s, 0, IntPtr.Zero, 0un, Cfg.Stream))
        checkIndexError ()
        dTable

    /// Adds the gradient of embedding to dTable.
    let addEmbeddingGrad (scale: 'T option) (dTable: Tensor<'T>) (tokens: Tensor<int64>) (dOut: Tensor<'T>) =
        callScaled scale [some dTable; some tokens; some dOut] (fun s p ->
            Native.embedding_grad (p.[0], p.[1], p.[2], s, 1, IntPtr.Zero, 0un, Cfg.Stream))
        checkIndexError ()

    /// (logProbs, lse, entropy, topLogProbs, topTokens) of logits [i_1 .. i_n; V]; top may be 0.
    let tokenLogProbs (top: int64) (logits: Tensor<'T>) (tokens: Tensor<int64>) =
        let row = logits.Shape |> List.take (logits.NDims - 1)
        let logProbs, lse, entropy = like logits row, like logits row, like logits row
        let topLogProbs, topTokens = like logits (row @ [top]), like tokens (row @ [top])
        let best, bestIdx = if top > 0L then some topLogProbs, some topTokens else None, None
        call [some logProbs; some lse; some entropy; best; bestIdx; some logits; some tokens] (fun p ->
            Native.token_log_probs (p.[0], p.[1], p.[2], p.[3], p.[4], p.[5], p.[6], IntPtr.Zero, 0un, Cfg.Stream))
        checkIndexError ()
        logProbs, lse, entropy, topLogProbs, topTokens

    /// Gradient of sum (dLogProbs * logProbs + dEntropy * entropy) with respect to the logits; entropy: (entropy, dEntropy).
    let tokenLogProbsGrad (logits: Tensor<'T>) (tokens: Tensor<int64>) (lse: Tensor<'T>) (dLogProbs: Tensor<'T>) (entropy: (Tensor<'T> * Tensor<'T>) option) =
        let dLogits = like logits logits.Shape
        call [some dLogits; some logits; some tokens; some lse; opt (Option.map fst entropy); some dLogProbs; opt (Option.map snd entropy)] (fun p ->
            Native.token_log_probs_grad (p.[0], p.[1], p.[2], p.[3], p.[4], p.[5], p.[6], Cfg.Stream))
        checkIndexError ()
        dLogits

    /// (out, lse) of softmax (scale q k^T) v over the keys that the mask [batch; position] leaves.
    let crossAttention (scale: 'T option) (mask: Tensor<bool> option) (q: Tensor<'T>) (k: Tensor<'T>) (v: Tensor<'T>) =
        let row = q.Shape |> List.take 3
        let out, lse = like q (row @ [v.Shape.[3]]), like q row
        callScaled scale [some out; some lse; some q; some k; some v; opt mask] (fun s p ->
            Native.cross_attention (p.[0], p.[1], p.[2], p.[3], p.[4], p.[5], s, IntPtr.Zero, 0un, Cfg.Stream))
        out, lse

    /// (dQ, dK, dV) of sum (dOut * out).
    let crossAttentionGrad (scale: 'T option) (mask: Tensor<bool> option) (dOut: Tensor<'T>) (q: Tensor<'T>) (k: Tensor<'T>) (v: Tensor<'T>) (out: Tensor<'T>) (lse: Tensor<'T>) =
        let dQ, dK, dV = like q q.Shape, like k k.Shape, like v v.Shape
        callScaled scale [some dQ; some dK; some dV; some dOut; some q; some k; some v; some out; some lse; opt mask] (fun s p ->
            Native.cross_attention_grad (p.[0], p.[1], p.[2], p.[3], p.[4], p.[5], p.[6], p.[7], p.[8], p.[9], s, IntPtr.Zero, 0un, Cfg.Stream))
        dQ, dK, dV
